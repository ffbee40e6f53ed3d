// Host side of linear / grouped_linear: argument checks and launches.  Included by
// moe_b200.cu, whose helpers it uses.
#pragma once

#include "few_sm100.cuh"
#include "linear.cuh"

namespace moe {

// When the few-row kernel takes a product over the row tiles of 128 x 256: up to 16 rows, and up to
// 192 rows of a dense product whose tiles would keep no more than an eighth of the SMs busy over
// a long contraction.  Measured, row tiles / few rows in us (bf16, dense unless said):
//   1 row   4096 -> 11008   41 / 25       64 rows  4096 -> 11008  39 / 46
//   37 rows 7168 -> 4096    49 / 27       64 rows  7168 -> 2048   48 / 25
//   64 rows 2048 -> 7168    23 / 35       192 rows 7168 -> 2048   49 / 40
//   64 rows 1024 -> 1024    16 / 29       256 rows 7168 -> 2048   49 / 60
//   16 rows, 8 groups, 4096 -> 2048  43 / 33;  64 rows 45 / 52
static bool few_linear_wins(int64_t m, int64_t n, int64_t k, bool dense) {
  if (m <= 16) return true;
  return dense && m <= 192 && k >= 4096 &&
         (m + 127) / 128 * ((n + 255) / 256) * 8 <= num_sms(current_device());
}

struct LinearArgs {
  const void* A;
  const void* B;
  const void* bias;
  const void* residual;
  void* out;
  void* preact;
  const int32_t* offsets;
  int plus_one;
  int64_t m, n, k;
  int E;
  bool b_mn;
  int act, dtype;
  cudaStream_t stream;
};

// A warp per weight row (linear_rows_kernel), or 64 x 64 tiles: the smaller of two estimates in us.
//   warps  6 + chunks of at most 8 rows x n x (k + the joining of a row's sums) x the time of a
//          weight, which grows with the rows of a chunk; no less than the loop's latency.
//   tiles  8 + K / 32 slices one after the other, each as long as the blocks that an SM holds ask.
// m rows are taken to pick their group at random.  Measured, tiles / warps in us, fp32 unless said:
//   1 x 7168 -> 11008 655 / 169    16: 661 / 476    32: 665 / 935     (rows x k -> n)
//   16 x 4096 -> 4096 254 / 94     32: 255 / 183    64: 256 / 351
//   8 x 4097 -> 4097  257 / 121    24: 257 / 267    48: 259 / 638
//   64 x 1024 -> 1024 71 / 38      128: 70 / 60     256: 70 / 108
//   8 x 300 -> 7168   29 / 19      32: 29 / 41      333 x 257 -> 130  25 / 12
//   256 x 7168 -> 300 442 / 256    bf16 4 x 4097 -> 4097  454 / 72    16: 460 / 178
//   grouped, 8 x 1999 -> 2001  64: 198 / 196    128: 269 / 388;  bf16  32: 277 / 132   128: 323 / 376
//   grouped, 64 x 999 -> 1001  16: 140 / 52     256: 326 / 232   1024: 370 / 683
static bool linear_warps_win(int64_t m, int64_t n, int64_t k, int E, int elem_size, bool vec) {
  const auto ceil_div = [](double a, double b) { return ceil(a / b); };
  const double live = E <= 1 ? 1.0 : E * (1.0 - pow(1.0 - 1.0 / E, (double)m));
  // pieces of up to `rows` rows that the groups' rows fall into
  const auto pieces = [&](double rows) {
    return E <= 1 ? ceil_div(m, rows) : std::max(live, m / rows + live / 2);
  };
  const double chunks = pieces(kWarpRows), q = std::min<double>(kWarpRows, m / chunks);
  const double weight = vec ? 2.0 + 0.1 * q : 2.4 + 0.3 * q;  // us per 10^6
  const double turns = k * elem_size / (32.0 * (vec ? 16 : elem_size));
  const double warps = 6 + std::max(chunks * n * (k + (vec ? 250.0 : 100.0)) * weight * 1e-6,
                                    turns * (0.3 + 0.08 * q));
  const double blocks = ceil_div(pieces(simt::TM) * ceil_div(n, simt::TN), num_sms(current_device()));
  const double slice = elem_size == 4 ? 0.7 + 1.3 * blocks : 1.5 + 1.8 * blocks;
  return warps < 8 + ceil_div(k, simt::TK) * slice;
}

template <typename T>
static int linear_simt(const LinearArgs& a) {
  const LinearEpilogue<T> epi{(T*)a.out, (T*)a.preact, (const T*)a.bias, (const T*)a.residual, a.act};
  const bool vec = (a.k * sizeof(T)) % 16 == 0 && aligned16(a.A) && aligned16(a.B);
  if (!a.b_mn && a.n < (1 << 30) && a.k < (1 << 30) &&
      linear_warps_win(a.m, a.n, a.k, a.E, sizeof(T), vec)) {
    const int64_t warps = ((a.m + kWarpRows - 1) / kWarpRows + (a.offsets ? a.E : 0)) * a.n;
    const unsigned grid = (unsigned)std::min<int64_t>((warps + 7) / 8, 8 * num_sms(current_device()));
    const size_t smem = (size_t)(a.E + 1) * 4;
    if (vec)
      linear_rows_kernel<T, true><<<grid, 256, smem, a.stream>>>(
          (const T*)a.A, (const T*)a.B, epi, a.offsets, a.plus_one, a.E, a.m, (int)a.n, (int)a.k);
    else
      linear_rows_kernel<T, false><<<grid, 256, smem, a.stream>>>(
          (const T*)a.A, (const T*)a.B, epi, a.offsets, a.plus_one, a.E, a.m, (int)a.n, (int)a.k);
    MOE_LAUNCH_CHECK();
    return MOE_OK;
  }
  const dim3 grid((unsigned)((a.m + simt::TM - 1) / simt::TM), (unsigned)((a.n + simt::TN - 1) / simt::TN),
                  (unsigned)a.E);
  MOE_REQUIRE(grid.y <= 65535, "linear: too large for the CUDA-core path");
  simt::gmm_rows_simt_kernel<T><<<grid, 256, 0, a.stream>>>(
      (const T*)a.A, (const T*)a.B, epi, a.offsets, a.plus_one, a.m, a.n, a.k, a.b_mn);
  MOE_LAUNCH_CHECK();
  return MOE_OK;
}

static bool linear_tc_ok(const LinearArgs& a) {
  return a.dtype != MOE_F32 && a.k > 0 && a.k % 8 == 0 && a.n % 8 == 0 &&
         aligned16(a.A) && aligned16(a.B) && aligned16(a.out) && aligned16(a.preact) &&
         aligned16(a.bias) && aligned16(a.residual) && a.m < (1ll << 31) && a.n < (1ll << 31) &&
         a.k < (1ll << 31);
}

static int linear_tiles(const LinearArgs& a) {
  const int cg = a.b_mn ? 1 : pick_cg(a.m >= 1024ll * a.E ? 2 : 1);
  CUtensorMap ma, mb, mc, mz;
  int rc;
  {
    const uint64_t dims[2] = {(uint64_t)a.k, (uint64_t)a.m};
    const uint32_t box[2] = {(uint32_t)gmm::BK, 64u};
    if ((rc = make_map(&ma, a.A, a.dtype, 2, dims, box))) return rc;
  }
  if (!a.b_mn) {
    const uint64_t dims[3] = {(uint64_t)a.k, (uint64_t)a.n, (uint64_t)a.E};
    const uint32_t box[3] = {(uint32_t)gmm::BK, (uint32_t)(gmm::BN / cg), 1};
    if ((rc = make_map(&mb, a.B, a.dtype, 3, dims, box))) return rc;
  } else {
    const uint64_t dims[3] = {(uint64_t)a.n, (uint64_t)a.k, (uint64_t)a.E};
    const uint32_t box[3] = {64, (uint32_t)gmm::BK, 1};
    if ((rc = make_map(&mb, a.B, a.dtype, 3, dims, box))) return rc;
  }
  {
    const uint64_t dims[2] = {(uint64_t)a.n, (uint64_t)a.m};
    const uint32_t box[2] = {32, 32};
    if ((rc = make_map(&mc, a.out, a.dtype, 2, dims, box, CU_TENSOR_MAP_SWIZZLE_64B))) return rc;
    mz = mc;
    if (a.preact && (rc = make_map(&mz, a.preact, a.dtype, 2, dims, box, CU_TENSOR_MAP_SWIZZLE_64B)))
      return rc;
  }
  gmm::Params p = {};
  p.offsets = a.offsets;
  p.offsets_plus_one = a.plus_one;
  p.num_groups = a.E;
  p.m_total = a.m;
  p.n_out = (int)a.n;
  p.k_red = (int)a.k;
  p.out = a.out;
  p.bias = a.bias;
  p.residual = a.residual;
  p.preact = a.preact;
  p.act = a.act;
  const CUtensorMap extra[3] = {mb, mz, mc};
  constexpr int ML = gmm::kModeLinear;
  if (a.dtype == MOE_BF16) {
    if (a.b_mn) return launch_sm100<ML, 1, 1, false, true, __nv_bfloat16>(ma, mb, mc, p, a.stream, extra);
    return cg == 2 ? launch_sm100<ML, 2, 1, false, false, __nv_bfloat16>(ma, mb, mc, p, a.stream, extra)
                   : launch_sm100<ML, 1, 1, false, false, __nv_bfloat16>(ma, mb, mc, p, a.stream, extra);
  }
  if (a.b_mn) return launch_sm100<ML, 1, 0, false, true, __half>(ma, mb, mc, p, a.stream, extra);
  return cg == 2 ? launch_sm100<ML, 2, 0, false, false, __half>(ma, mb, mc, p, a.stream, extra)
                 : launch_sm100<ML, 1, 0, false, false, __half>(ma, mb, mc, p, a.stream, extra);
}

// The few-row kernel's split, counters and partials.
struct FewLinear {
  int nb, max_units, grid;
  FewSplit split;
  size_t part, total;
};
static FewLinear few_linear_plan(int64_t m, int64_t n, int64_t k, int E, bool dense) {
  FewLinear f = {};
  f.nb = few_nb(m);
  f.max_units = fewtc::row_units_max(m, E, f.nb);
  // groups that are likely to have a row, when the rows pick groups at random
  const double live = E <= 1 ? 1.0 : E * (1.0 - pow(1.0 - 1.0 / E, (double)m));
  const double units = dense ? (double)((m + f.nb - 1) / f.nb) : std::max(live, (double)m / f.nb);
  f.split = few_split_linear(units, n, (k + fewtc::BK - 1) / fewtc::BK,
                             std::min<double>(f.nb, (double)m / units));
  f.part = 256;
  f.total = f.part + (f.split.parts > 1 ? (size_t)f.split.parts * m * n * 4 : 0);
  f.grid = num_sms(current_device());
  if (dense) f.grid = (int)std::min<int64_t>(f.grid, (int64_t)units * f.split.shape.tiles * f.split.parts);
  return f;
}

static bool few_linear_ok(const LinearArgs& a) {
  return linear_tc_ok(a) && !a.b_mn && few_linear_wins(a.m, a.n, a.k, a.offsets == nullptr);
}

static int few_linear(const LinearArgs& a, void* workspace, size_t workspace_bytes) {
  const FewLinear f = few_linear_plan(a.m, a.n, a.k, a.E, a.offsets == nullptr);
  if (!workspace || workspace_bytes < f.total)
    return set_error(MOE_ERR_WORKSPACE, "linear: workspace has %zu bytes, needs %zu",
                     workspace ? workspace_bytes : (size_t)0, f.total);
  MOE_REQUIRE(aligned16(workspace), "linear: workspace must be 16-byte aligned");
  CUtensorMap map;
  int rc;
  if ((rc = few_weight_map(&map, a.B, a.dtype, a.k, a.n, a.E, f.split.shape.rows))) return rc;
  uint8_t* ws = (uint8_t*)workspace;
  fewtc::Params p = {};
  p.offsets = a.offsets;
  p.plus_one = a.plus_one;
  p.E = a.E;
  p.m = a.m;
  p.N = (int)a.n;
  p.K = (int)a.k;
  p.bias = a.bias;
  p.residual = a.residual;
  p.preact = a.preact;
  p.act = a.act;
  p.x = a.A;
  p.y = a.out;
  p.counters = (int*)ws;
  p.part = (float*)(ws + f.part);
  p.parts = f.split.parts;
  p.max_units = f.max_units;
  p.shape[0] = f.split.shape;
  const int table = fewtc::row_units_bytes(f.max_units);
  if ((rc = few_ring(p, 1, f.nb, table))) return rc;
  if (f.split.parts > 1 && (rc = zero_counters(p.counters, 2, a.stream))) return rc;
  const CUtensorMap maps[3] = {map, map, map};
  if (a.dtype == MOE_BF16)
    return few_kernel_nb<fewtc::kLinear, 1, __nv_bfloat16>(f.nb, maps, p, (unsigned)f.grid, table, a.stream);
  return few_kernel_nb<fewtc::kLinear, 0, __half>(f.nb, maps, p, (unsigned)f.grid, table, a.stream);
}

static int tail_rows(void* out, const void* residual, const int32_t* offsets, int last, int64_t m,
                     int64_t n, int dtype, cudaStream_t s) {
  if (offsets == nullptr || m == 0 || n == 0) return MOE_OK;
  // A few blocks: the usual call has no such row.
  const unsigned grid = (unsigned)std::min<int64_t>((m * n + 255) / 256, 64);
  return MOE_DISPATCH_DTYPE(dtype, T, [&] {
    tail_rows_kernel<T><<<grid, 256, 0, s>>>((T*)out, (const T*)residual, offsets, last, m, n);
    MOE_LAUNCH_CHECK();
    return (int)MOE_OK;
  });
}

static int check_linear(const void* a, const void* b, const void* out, const int32_t* offsets,
                        int num_offsets, int64_t m, int64_t n, int64_t k, int E, int act, int dtype) {
  MOE_REQUIRE(act >= MOE_ACT_NONE && act <= MOE_ACT_SILU, "linear: bad activation %d", act);
  MOE_REQUIRE(E >= 1 || offsets != nullptr || m == 0, "linear: no groups");
  MOE_REQUIRE(E <= gmm::kMaxGroups, "linear: more than %d experts", gmm::kMaxGroups);
  // An operand with no elements may be NULL.
  if (m > 0 && n > 0)
    MOE_REQUIRE(out && ((a && b) || k == 0 || E == 0), "linear: NULL operand");
  return check_gmm_args(out, out, out, offsets, num_offsets, out ? m : 0, n, k, E, dtype, true);
}

// Workspace of the backward: dz [m, n] (unless there is no activation), then the bias gradient's
// partial sums.
struct BwdWorkspace {
  size_t partial, total;
};
static BwdWorkspace bwd_workspace(int64_t m, int64_t n, int E, int act, int dtype) {
  BwdWorkspace w;
  w.partial = act == MOE_ACT_NONE ? 0 : align256((size_t)m * n * dtype_size(dtype));
  w.total = w.partial + (size_t)((m + kDzRows - 1) / kDzRows + E) * n * 4 + 16;
  return w;
}

// dz = grad_out * act'(preact) (written unless act is none) and grad_bias (may be NULL).
static int act_bwd(const void* grad_out, const void* preact, void* dz, void* grad_bias,
                   const int32_t* offsets, int num_offsets, int64_t m, int64_t n, int E, int activation,
                   int dtype, float* partial, cudaStream_t s) {
  const bool act = activation != MOE_ACT_NONE;
  const int plus_one = num_offsets == E + 1;
  if (!grad_bias) partial = nullptr;
  const int64_t chunks = (m + kDzRows - 1) / kDzRows + (offsets ? E : 0);
  const size_t smem = (size_t)(E + 1) * 4;
  const bool vec = (n * dtype_size(dtype)) % 16 == 0 && aligned16(grad_out) &&
                   (!act || (aligned16(preact) && aligned16(dz)));
  int rc = MOE_DISPATCH_DTYPE(dtype, T, [&] {
    constexpr int V = 16 / (int)sizeof(T);
    const int cols = 32 * (vec ? V : 1);
    const dim3 grid((unsigned)((n + cols - 1) / cols), (unsigned)std::min<int64_t>(chunks, 32768));
    MOE_SWITCH_ACT(activation, ACT, {
      if (vec)
        dz_kernel<T, V, ACT><<<grid, kDzThreads, smem, s>>>(
            (const T*)grad_out, (const T*)preact, (T*)dz, partial, offsets, plus_one, E, m, n);
      else
        dz_kernel<T, 1, ACT><<<grid, kDzThreads, smem, s>>>(
            (const T*)grad_out, (const T*)preact, (T*)dz, partial, offsets, plus_one, E, m, n);
    })
    MOE_LAUNCH_CHECK();
    return (int)MOE_OK;
  });
  if (rc || !grad_bias) return rc;
  return MOE_DISPATCH_DTYPE(dtype, T, [&] {
    const dim3 grid((unsigned)((n + 31) / 32), (unsigned)std::min(E, 1024));
    MOE_CUDA_CHECK(launch_pdl(dbias_kernel<T>, grid, dim3(kDzThreads), smem, s, (const float*)partial,
                              (T*)grad_bias, offsets, plus_one, E, m, n));
    return (int)MOE_OK;
  });
}

}  // namespace moe

extern "C" {

size_t moe_linear_workspace_bytes(int64_t m_total, int64_t n, int64_t k, int32_t num_experts,
                                  int trans_b, int dtype) {
  if (m_total <= 0 || n <= 0 || k <= 0 || num_experts <= 0 || !trans_b || dtype == MOE_F32) return 0;
  size_t need = 0;  // of a grouped and, with one expert, of a dense product
  if (few_linear_wins(m_total, n, k, false))
    need = few_linear_plan(m_total, n, k, num_experts, false).total;
  if (num_experts == 1 && few_linear_wins(m_total, n, k, true))
    need = std::max(need, few_linear_plan(m_total, n, k, 1, true).total);
  return need;
}

int moe_linear_fwd(const void* A, const void* B, const void* bias, const void* residual, void* out,
                   void* preact, const int32_t* offsets, int32_t num_offsets, int64_t m_total,
                   int64_t n, int64_t k, int32_t num_experts, int trans_b, int activation, int dtype,
                   void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_linear(A, B, out, offsets, num_offsets, m_total, n, k, num_experts, activation, dtype);
  if (rc) return rc;
  if (m_total == 0 || n == 0) return MOE_OK;
  LinearArgs a = {A, B, bias, residual, out, preact, offsets, num_offsets == num_experts + 1,
                  m_total, n, k, num_experts, !trans_b, activation, dtype, (cudaStream_t)stream};
  if (num_experts > 0) {
    if (few_linear_ok(a)) {
      rc = few_linear(a, workspace, workspace_bytes);
    } else if (linear_tc_ok(a)) {
      rc = linear_tiles(a);
    } else {
      rc = MOE_DISPATCH_DTYPE(dtype, T, [&] { return linear_simt<T>(a); });
    }
    if (rc) return rc;
    return tail_rows(out, residual, offsets, num_offsets - 1, m_total, n, dtype, a.stream);
  }
  if (residual)
    MOE_CUDA_CHECK(cudaMemcpyAsync(out, residual, (size_t)m_total * n * dtype_size(dtype),
                                   cudaMemcpyDeviceToDevice, a.stream));
  else
    MOE_CUDA_CHECK(cudaMemsetAsync(out, 0, (size_t)m_total * n * dtype_size(dtype), a.stream));
  return MOE_OK;
}

size_t moe_linear_bwd_workspace_bytes(int64_t m_total, int64_t n, int32_t num_experts, int activation,
                                      int dtype) {
  if (m_total <= 0 || n <= 0 || num_experts <= 0 || !dtype_ok(dtype)) return 16;
  return bwd_workspace(m_total, n, num_experts, activation, dtype).total;
}

int moe_linear_bwd(const void* grad_out, const void* A, const void* B, const void* preact, void* grad_A,
                   void* grad_B, void* grad_bias, const int32_t* offsets, int32_t num_offsets,
                   int64_t m_total, int64_t n, int64_t k, int32_t num_experts, int trans_b,
                   int activation, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_linear(nullptr, nullptr, grad_out, offsets, num_offsets, m_total, n, 0, num_experts,
                        activation, dtype);
  if (rc) return rc;
  MOE_REQUIRE(k >= 0, "linear_bwd: negative size");
  const bool act = activation != MOE_ACT_NONE, any = m_total > 0 && n > 0 && num_experts > 0;
  MOE_REQUIRE(!any || !act || preact, "linear_bwd: preact is NULL");
  MOE_REQUIRE(!any || k == 0 || ((!grad_A || B) && (!grad_B || A)), "linear_bwd: NULL operand");
  cudaStream_t s = (cudaStream_t)stream;
  const int es = dtype_size(dtype);
  if (!any) {  // sums over nothing
    if (grad_A && m_total > 0 && k > 0) MOE_CUDA_CHECK(cudaMemsetAsync(grad_A, 0, (size_t)m_total * k * es, s));
    if (grad_B && num_experts * n * k > 0)
      MOE_CUDA_CHECK(cudaMemsetAsync(grad_B, 0, (size_t)num_experts * n * k * es, s));
    if (grad_bias && num_experts * n > 0)
      MOE_CUDA_CHECK(cudaMemsetAsync(grad_bias, 0, (size_t)num_experts * n * es, s));
    return MOE_OK;
  }
  const BwdWorkspace w = bwd_workspace(m_total, n, num_experts, activation, dtype);
  if ((act || grad_bias) && (!workspace || workspace_bytes < w.total))
    return set_error(MOE_ERR_WORKSPACE, "linear_bwd: workspace has %zu bytes, needs %zu",
                     workspace ? workspace_bytes : (size_t)0, w.total);
  MOE_REQUIRE(!(act || grad_bias) || aligned16(workspace), "linear_bwd: workspace must be 16-byte aligned");
  void* dz = act ? workspace : const_cast<void*>(grad_out);
  if (act || grad_bias) {
    rc = act_bwd(grad_out, preact, dz, grad_bias, offsets, num_offsets, m_total, n, num_experts,
                 activation, dtype, (float*)((uint8_t*)workspace + w.partial), s);
    if (rc) return rc;
  }
  if (grad_A && k > 0) {
    rc = moe_gmm_dgrad(dz, B, grad_A, offsets, num_offsets, m_total, n, k, num_experts, trans_b, dtype, stream);
    if (rc) return rc;
    rc = tail_rows(grad_A, nullptr, offsets, num_offsets - 1, m_total, k, dtype, s);
    if (rc) return rc;
  }
  if (grad_B && k > 0)
    return moe_gmm_wgrad(A, dz, grad_B, offsets, num_offsets, m_total, n, k, num_experts, trans_b, dtype, stream);
  return MOE_OK;
}

}  // extern "C"
