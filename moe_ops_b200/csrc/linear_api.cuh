// Host side of linear / grouped_linear: argument checks and launches.  Included by
// moe_b200.cu, whose helpers it uses.
#pragma once

#include "few_sm100.cuh"
#include "linear.cuh"

namespace moe {

// Rows up to which the few-row kernel takes a product.
static int64_t few_linear_max_rows(int E) { return E <= 1 ? 64 : 64; }

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

// Rows per group up to which a warp per weight row is taken over 64 x 64 tiles (which need at least
// a slice of 32 in K per step, and 64 rows to be full).
constexpr int kLinearWarpRows = 16;

template <typename T>
static int linear_simt(const LinearArgs& a) {
  const LinearEpilogue<T> epi{(T*)a.out, (T*)a.preact, (const T*)a.bias, (const T*)a.residual, a.act};
  if (!a.b_mn && a.E <= gmm::kMaxGroups && a.m <= (int64_t)kLinearWarpRows * a.E) {
    const int64_t warps = ((a.m + kWarpRows - 1) / kWarpRows + (a.offsets ? a.E : 0)) * a.n;
    const unsigned grid = (unsigned)std::min<int64_t>((warps + 7) / 8, 8 * num_sms(current_device()));
    linear_rows_kernel<T><<<grid, 256, (size_t)(a.E + 1) * 4, a.stream>>>(
        (const T*)a.A, (const T*)a.B, epi, a.offsets, a.plus_one, a.E, a.m, a.n, a.k);
    MOE_LAUNCH_CHECK();
    return MOE_OK;
  }
  const dim3 grid((unsigned)((a.m + simt::TM - 1) / simt::TM), (unsigned)((a.n + simt::TN - 1) / simt::TN),
                  (unsigned)a.E);
  MOE_REQUIRE(grid.y <= 65535 && grid.z <= 65535, "linear: too large for the CUDA-core path");
  simt::gmm_rows_simt_kernel<T><<<grid, 256, 0, a.stream>>>(
      (const T*)a.A, (const T*)a.B, epi, a.offsets, a.plus_one, a.m, a.n, a.k, a.b_mn);
  MOE_LAUNCH_CHECK();
  return MOE_OK;
}

static bool linear_tc_ok(const LinearArgs& a) {
  return a.dtype != MOE_F32 && a.k > 0 && a.k % 8 == 0 && a.n % 8 == 0 && a.E <= gmm::kMaxGroups &&
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
  return linear_tc_ok(a) && !a.b_mn && a.m <= few_linear_max_rows(a.E);
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
  // An operand with no elements may be NULL.
  if (m > 0 && n > 0)
    MOE_REQUIRE(out && ((a && b) || k == 0 || E == 0), "linear: NULL operand");
  return check_gmm_args(out, out, out, offsets, num_offsets, out ? m : 0, n, k, E, dtype);
}

}  // namespace moe

extern "C" {

size_t moe_linear_workspace_bytes(int64_t m_total, int64_t n, int64_t k, int32_t num_experts,
                                  int trans_b, int dtype) {
  if (m_total <= 0 || n <= 0 || k <= 0 || num_experts <= 0 || !trans_b || dtype == MOE_F32 ||
      m_total > few_linear_max_rows(num_experts))
    return 0;
  // whether the product is dense only changes the split: the larger of the two
  return std::max(few_linear_plan(m_total, n, k, num_experts, false).total,
                  few_linear_plan(m_total, n, k, num_experts, true).total);
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

size_t moe_linear_act_bwd_workspace_bytes(int64_t m_total, int64_t n, int32_t num_experts) {
  if (m_total <= 0 || n <= 0 || num_experts <= 0) return 16;
  return (size_t)((m_total + kDzRows - 1) / kDzRows + num_experts) * n * 4 + 16;
}

int moe_linear_act_bwd(const void* grad_out, const void* preact, void* grad_preact, void* grad_bias,
                       const int32_t* offsets, int32_t num_offsets, int64_t m_total, int64_t n,
                       int32_t num_experts, int activation, int dtype, void* workspace,
                       size_t workspace_bytes, void* stream) {
  int rc = check_linear(nullptr, nullptr, grad_out, offsets, num_offsets, m_total, n, 0, num_experts,
                        activation, dtype);
  if (rc) return rc;
  const bool act = activation != MOE_ACT_NONE;
  MOE_REQUIRE(!act || m_total == 0 || (preact && grad_preact), "linear_act_bwd: NULL operand");
  cudaStream_t s = (cudaStream_t)stream;
  if (n == 0 || num_experts == 0) return MOE_OK;
  if (m_total == 0) {
    if (grad_bias)
      MOE_CUDA_CHECK(cudaMemsetAsync(grad_bias, 0, (size_t)num_experts * n * dtype_size(dtype), s));
    return MOE_OK;
  }
  if (!act && !grad_bias) return MOE_OK;
  MOE_REQUIRE(num_experts <= gmm::kMaxGroups, "linear_act_bwd: more than %d experts", gmm::kMaxGroups);
  if (grad_bias && (!workspace || workspace_bytes <
                                      moe_linear_act_bwd_workspace_bytes(m_total, n, num_experts)))
    return set_error(MOE_ERR_WORKSPACE, "linear_act_bwd: workspace too small");
  const int plus_one = num_offsets == num_experts + 1;
  const int E = num_experts;
  float* partial = grad_bias ? (float*)workspace : nullptr;
  const int64_t chunks = (m_total + kDzRows - 1) / kDzRows + (offsets ? E : 0);
  const size_t smem = (size_t)(E + 1) * 4;
  const int es = dtype_size(dtype);
  const bool vec = (n * es) % 16 == 0 && aligned16(grad_out) && (!act || (aligned16(preact) && aligned16(grad_preact)));
  rc = MOE_DISPATCH_DTYPE(dtype, T, [&] {
    constexpr int V = 16 / (int)sizeof(T);
    const int cols = 32 * (vec ? V : 1);
    const dim3 grid((unsigned)((n + cols - 1) / cols), (unsigned)std::min<int64_t>(chunks, 32768));
    if (vec)
      dz_kernel<T, V><<<grid, kDzThreads, smem, s>>>((const T*)grad_out, (const T*)preact,
                                                     (T*)grad_preact, partial, offsets, plus_one, E,
                                                     m_total, n, activation);
    else
      dz_kernel<T, 1><<<grid, kDzThreads, smem, s>>>((const T*)grad_out, (const T*)preact,
                                                     (T*)grad_preact, partial, offsets, plus_one, E,
                                                     m_total, n, activation);
    MOE_LAUNCH_CHECK();
    return (int)MOE_OK;
  });
  if (rc || !grad_bias) return rc;
  return MOE_DISPATCH_DTYPE(dtype, T, [&] {
    const dim3 grid((unsigned)((n + 31) / 32), (unsigned)std::min(E, 1024));
    MOE_CUDA_CHECK(launch_pdl(dbias_kernel<T>, grid, dim3(kDzThreads), smem, s, (const float*)partial,
                              (T*)grad_bias, offsets, plus_one, E, m_total, n));
    return (int)MOE_OK;
  });
}

int moe_zero_tail_rows(void* out, const int32_t* offsets, int32_t num_offsets, int64_t m_total,
                       int64_t n, int dtype, void* stream) {
  MOE_REQUIRE(dtype_ok(dtype), "zero_tail_rows: bad dtype %d", dtype);
  MOE_REQUIRE(offsets && num_offsets > 0 && m_total >= 0 && n >= 0 && (out || m_total == 0 || n == 0),
              "zero_tail_rows: bad arguments");
  return tail_rows(out, nullptr, offsets, num_offsets - 1, m_total, n, dtype, (cudaStream_t)stream);
}

}  // extern "C"
