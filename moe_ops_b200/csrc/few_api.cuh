// Host side of the few-token mixture-of-experts layer (few_tokens.cuh): argument checks,
// workspace layout and launches.  Included by moe_b200.cu, whose helpers it uses.
#pragma once

#include "few_sm100.cuh"
#include "few_tokens.cuh"

namespace moe {

struct FewArgs {
  const void* x;
  const void* w_router;        // NULL: weights / indices are given
  const float* router_bias;
  const float* weights;
  const int32_t* indices;
  const void* w_gate;
  const void* w_up;
  const void* w_down;
  int64_t num_tokens, d, hidden;
  int32_t E, topk;
  int dtype;
  void* out;
  void* workspace;
  size_t workspace_bytes;
  cudaStream_t stream;
};

constexpr size_t kMaxSmem = 232448;  // dynamic shared memory a block may have on sm_100

static size_t align256(size_t v) { return (v + 255) / 256 * 256; }

// Rows of a unit of the tensor-core kernel, by the most rows that one expert (one group) can
// have unless an expert repeats: smaller units leave room for more stages, larger ones read a
// crowded expert's weights once.
static int few_nb(int64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

struct FewSplit {
  fewtc::Params::Shape shape;
  int parts;
};
static FewSplit few_tiles(int64_t rows, int64_t height, int64_t KB, int64_t parts, bool gate_up) {
  FewSplit f = {};
  const int64_t len = (KB + parts - 1) / parts;  // equal chunks, none empty
  f.parts = (int)((KB + len - 1) / len);
  f.shape.rows = (int)std::min(height, rows);
  f.shape.tiles = (int)((rows + f.shape.rows - 1) / f.shape.rows);
  const int h = (f.shape.rows + 7) / 8 * 8;  // boxes start at multiples of 1 KB
  f.shape.m_tiles = h > (gate_up ? 64 : 128) ? 2 : 1;
  f.shape.second = gate_up ? std::max(64, h) * 128 : h > 128 ? 16384 : 0;
  f.shape.block_bytes = gate_up ? f.shape.second + h * 128 : h * 128;
  return f;
}

// kMoe.  Full M tiles throughout.  Phase 0: 128 columns of h to a tile from 4 waves of tiles on,
// else 64 (measured, all of a call: 32 tokens d = 7168 E = 256 H = 2048, 17 waves, 2019 us against
// 2260; 1 token d = 4096 H = 11008, 1.2 waves, 122 against 109).  Phase 1: 256 rows from 2 waves
// on, else 128 rows, and the contraction cut into chunks of 8 blocks or more: SMs leave phase 0
// at different times and small chunks even that out (the 1-token call: 4 waves of chunks 106 us,
// one wave 123 us; 16 tokens: 256 rows cut in 5 961 us, 128 rows uncut 987 us).
static FewSplit few_split0(double units, int64_t H, int64_t d) {
  const int64_t KB = (d + fewtc::BK - 1) / fewtc::BK;
  const double waves = units * ((H + 127) / 128) / num_sms(current_device());
  return few_tiles(H, waves >= 4 ? 128 : 64, KB, 1, true);
}
static FewSplit few_split1(double units, int64_t d, int64_t H) {
  const int64_t KB = (H + fewtc::BK - 1) / fewtc::BK;
  const double sms = num_sms(current_device());
  const bool high = units * ((d + 255) / 256) >= 2 * sms;
  const int64_t height = high ? 256 : 128;
  const int64_t parts = (int64_t)((high ? 12 : 4) * sms / (units * ((d + height - 1) / height)));
  return few_tiles(d, height, KB, std::max<int64_t>(1, std::min(parts, KB / 8)), false);
}

// kLinear: `units` units of `n` rows, counted in SM cycles.  A 64-deep block of a tile takes the
// larger of its weights at an SM's share of HBM (26 bytes per cycle), weights and activations at
// the rate an SM reads L2 (50), and its MMAs (75 each, and up to 250 a stage); a chunk costs
// about 1000 more, and adding parts up at the end 6000 and a pass over them.  Heights that fill
// 1 to 4 waves of the SMs are compared, and whole ones.  (37 rows, K = 7168, N = 4096: picks 148
// chunks of 111 rows and a quarter of K, 26.7 us; 128 rows and a third 33 us, and a fifth 37 us.)
static FewSplit few_split_linear(double units, int64_t rows, int64_t KB, double n) {
  const double sms = num_sms(current_device());
  double best = 1e30;
  FewSplit f = {};
  for (const int64_t parts : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16}) {
    const int64_t len = (KB + parts - 1) / parts;
    if ((KB + len - 1) / len != parts) continue;
    if (parts > 1 && len < 4) break;
    for (int w = 1; w <= 5; ++w) {
      int64_t height = (int64_t)(units * parts * rows / (sms * w)) + 1;
      if (w == 5) height = 256;
      height = std::min<int64_t>(256, std::max<int64_t>(16, std::min(height, rows)));
      const int64_t tiles = (rows + height - 1) / height;
      const double weights = 128.0 * height;
      const double block = std::max({weights / 26, (weights + n * 128) / 50,
                                     300.0 * (height > 128 ? 2 : 1) + std::min(250.0, weights / 128)});
      double cost = ceil(units * tiles * parts / sms - 1e-6) * (len * block + 1000);
      if (parts > 1) cost += 6000 + parts * units * n * rows * 8 / (sms * 30);
      if (cost < best) {
        best = cost;
        f = few_tiles(rows, height, KB, parts, false);
      }
    }
  }
  return f;
}

// Ring geometry: as many 64-deep blocks per stage as about 36 KB hold, then as many stages as
// shared memory holds.
static int few_ring(fewtc::Params& p, int phases, int nb, int table_bytes) {
  int bytes = 0;
  for (int i = 0; i < phases; ++i) {
    auto& s = p.shape[i];
    const int block = s.block_bytes + nb * 128;
    s.blocks = std::max(1, std::min(fewtc::kMaxBlocksPerStage, 36864 / block));
    bytes = std::max(bytes, s.blocks * block);
  }
  p.stage_bytes = bytes;
  const size_t fixed = 1024 + fewtc::kCtlBytes + fewtc::kStagedBytes + (size_t)table_bytes;
  MOE_REQUIRE(fixed < kMaxSmem, "few rows: routing tables too large");
  p.stages = (int)std::min<size_t>(fewtc::kMaxStages, (kMaxSmem - fixed) / bytes);
  MOE_REQUIRE(p.stages >= 2, "few rows: routing tables too large");
  return MOE_OK;
}

// Workspace: logits [T, E] fp32; h [T*K, H] (fp32 for the CUDA cores, which also take 16-bit operands
// off a boundary, so 4 bytes an element; the tensor cores use half); the CUDA cores' slot weights and
// positions; the tensor-core kernel's counters; the experts' outputs, fp32
// [parts, T*K, d] (one part for the CUDA cores).
struct FewWorkspace {
  size_t logits, h, slots, counters, part, total;
  int num_counters, max_units;
  FewSplit split0, split1;
};
static FewWorkspace few_workspace(int64_t T, int64_t d, int64_t H, int64_t E, int64_t K, int dtype) {
  FewWorkspace w = {};
  const size_t S = (size_t)(T * K);
  w.logits = 0;
  w.h = align256((size_t)T * E * 4);
  w.slots = w.h + align256(S * H * 4);
  w.counters = w.slots + align256(S * 8);
  w.part = w.counters;
  int parts = 1;
  if (dtype != MOE_F32 && d > 0 && H > 0) {
    // experts that the tokens are expected to touch when each picks K of E
    const double touched = K >= E ? (double)E : E * (1.0 - pow(1.0 - (double)K / E, (double)T));
    w.split0 = few_split0(touched, H, d);
    w.split1 = few_split1(touched, d, H);
    parts = w.split1.parts;
    w.max_units = few::plan_max_units((int)S, (int)E, few_nb(T));
    w.num_counters = 2 + w.max_units;
    w.part = w.counters + align256((size_t)w.num_counters * 4);
  }
  w.total = w.part + align256((size_t)parts * S * d * 4);
  return w;
}

static int check_few(const FewArgs& a) {
  MOE_REQUIRE(dtype_ok(a.dtype), "few_tokens: bad dtype %d", a.dtype);
  MOE_REQUIRE(a.num_tokens >= 0 && a.num_tokens <= few::kMaxTokens,
              "few_tokens: num_tokens must be in [0, %d] (got %lld)", few::kMaxTokens,
              (long long)a.num_tokens);
  MOE_REQUIRE(a.E > 0 && a.E <= few::kMaxExperts, "few_tokens: need 0 < E <= %d (E=%d)",
              few::kMaxExperts, a.E);
  MOE_REQUIRE(a.topk > 0 && a.topk <= few::kMaxTopk && (a.topk <= a.E || !a.w_router),
              "few_tokens: need 0 < K <= min(E, %d) (E=%d, K=%d)", few::kMaxTopk, a.E, a.topk);
  MOE_REQUIRE(a.d >= 0 && a.hidden >= 0 && a.d < (1ll << 30) && a.hidden < (1ll << 30),
              "few_tokens: bad sizes d=%lld H=%lld", (long long)a.d, (long long)a.hidden);
  if (a.num_tokens == 0 || a.d == 0) return MOE_OK;
  MOE_REQUIRE(a.x && a.out && (a.hidden == 0 || (a.w_gate && a.w_up && a.w_down)),
              "few_tokens: NULL operand");
  MOE_REQUIRE(a.w_router || (a.weights && a.indices), "few_tokens: NULL routing");
  const FewWorkspace w = few_workspace(a.num_tokens, a.d, a.hidden, a.E, a.topk, a.dtype);
  if (!a.workspace || a.workspace_bytes < w.total)
    return set_error(MOE_ERR_WORKSPACE, "few_tokens: workspace has %zu bytes, needs %zu",
                     a.workspace ? a.workspace_bytes : (size_t)0, w.total);
  MOE_REQUIRE(aligned16(a.workspace), "few_tokens: workspace must be 16-byte aligned");
  return MOE_OK;
}

template <typename T>
static int few_router_launch(const FewArgs& a, float* logits, int* zero, int num_zero) {
  const bool vec = (a.d * sizeof(T)) % 16 == 0 && aligned16(a.x) && aligned16(a.w_router);
  const int64_t warps = (a.num_tokens + few::kRouterTokens - 1) / few::kRouterTokens * a.E;
  const unsigned grid = (unsigned)std::min<int64_t>((warps + 7) / 8, 4 * num_sms(current_device()));
  if (vec)
    few::router_kernel<T, true><<<grid, 256, 0, a.stream>>>(
        (const T*)a.x, (const T*)a.w_router, a.router_bias, logits, (int)a.num_tokens, (int)a.d,
        a.E, zero, num_zero);
  else
    few::router_kernel<T, false><<<grid, 256, 0, a.stream>>>(
        (const T*)a.x, (const T*)a.w_router, a.router_bias, logits, (int)a.num_tokens, (int)a.d,
        a.E, zero, num_zero);
  MOE_LAUNCH_CHECK();
  return MOE_OK;
}

template <typename T, bool VEC>
static int few_simt_launch(const FewArgs& a, const few::Routing& r, const FewWorkspace& w) {
  uint8_t* ws = (uint8_t*)a.workspace;
  float *h = (float*)(ws + w.h), *o = (float*)(ws + w.part), *slot_w = (float*)(ws + w.slots);
  int* slot_pos = (int*)(slot_w + r.num_tokens * r.K);
  const int S = r.num_tokens * r.K, plan = few::plan_bytes(S, r.E, few::kSimtRows);
  const int64_t units = few::plan_max_units(S, r.E, few::kSimtRows), most = 4 * num_sms(current_device());
  const auto grid = [&](int64_t warps) { return dim3((unsigned)std::max<int64_t>(1, std::min((warps + 7) / 8, most))); };
  const T *x = (const T*)a.x, *wg = (const T*)a.w_gate, *wu = (const T*)a.w_up, *wd = (const T*)a.w_down;
  const int d = (int)a.d, H = (int)a.hidden;
  MOE_CUDA_CHECK(launch_pdl(few::gate_up_simt_kernel<T, VEC>, grid(units * H), dim3(256), plan, a.stream, x,
                            wg, wu, h, slot_pos, slot_w, r, d, H));
  MOE_CUDA_CHECK(launch_pdl(few::down_simt_kernel<T, VEC>, grid(units * d), dim3(256), plan, a.stream,
                            (const float*)h, wd, o, r, d, H));
  MOE_CUDA_CHECK(launch_pdl(few::combine_simt_kernel<T>, grid((int64_t)r.num_tokens * d / 32 + 1), dim3(256), 0,
                            a.stream, (const float*)o, (const int*)slot_pos, (const float*)slot_w, (T*)a.out,
                            r.num_tokens, r.K, d));
  return MOE_OK;
}

// 16-bit operands whose rows are 16-byte multiples (TMA and 16-byte copies).
static bool few_tc_ok(const FewArgs& a) {
  return a.dtype != MOE_F32 && a.d % 8 == 0 && a.hidden % 8 == 0 && aligned16(a.x) &&
         aligned16(a.w_gate) && aligned16(a.w_up) && aligned16(a.w_down);
}

template <int MODE, int FMT, typename T, int NB>
static int few_kernel_launch(const CUtensorMap* maps, const fewtc::Params& p, unsigned grid, int table_bytes,
                             cudaStream_t stream) {
  auto kern = fewtc::few_kernel<MODE, FMT, T, NB>;
  const int dev = current_device();
  static unsigned long long attr_set = 0;  // per-device bitmask, one per instantiation
  {
    std::lock_guard<std::mutex> lock(g_cache_mu);
    if (dev >= 64 || !(attr_set & (1ull << dev))) {
      MOE_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem));
      if (dev < 64) attr_set |= 1ull << dev;
    }
  }
  const size_t smem = 1024 + (size_t)p.stages * p.stage_bytes + fewtc::kCtlBytes + fewtc::kStagedBytes + table_bytes;
  MOE_CUDA_CHECK(launch_pdl(kern, dim3(grid), dim3(fewtc::kThreads), smem, stream, maps[0], maps[1],
                            maps[2], p));
  return MOE_OK;
}

template <int MODE, int FMT, typename T>
static int few_kernel_nb(int nb, const CUtensorMap* maps, const fewtc::Params& p, unsigned grid,
                         int table_bytes, cudaStream_t stream) {
  if (nb == 16) return few_kernel_launch<MODE, FMT, T, 16>(maps, p, grid, table_bytes, stream);
  if (nb == 32) return few_kernel_launch<MODE, FMT, T, 32>(maps, p, grid, table_bytes, stream);
  return few_kernel_launch<MODE, FMT, T, 64>(maps, p, grid, table_bytes, stream);
}

static int zero_counters(int* counters, int n, cudaStream_t s) {
  fewtc::zero_counters_kernel<<<std::min(num_sms(current_device()), (n + 511) / 512), 256, 0, s>>>(counters, n);
  MOE_LAUNCH_CHECK();
  return MOE_OK;
}

static int few_weight_map(CUtensorMap* map, const void* w, int dtype, int64_t inner, int64_t rows, int64_t E,
                          int rows_of_box) {
  const uint64_t dims[3] = {(uint64_t)inner, (uint64_t)rows, (uint64_t)E};
  const uint32_t box[3] = {(uint32_t)fewtc::BK, (uint32_t)rows_of_box, 1};
  return make_map(map, w, dtype, 3, dims, box);
}

static int few_tc_launch(const FewArgs& a, const few::Routing& r, const FewWorkspace& w) {
  uint8_t* ws = (uint8_t*)a.workspace;
  const int nb = few_nb(a.num_tokens);
  const int table = few::plan_bytes(r.num_tokens * r.K, r.E, nb);
  fewtc::Params p = {};
  p.r = r;
  p.d = (int)a.d;
  p.H = (int)a.hidden;
  p.x = a.x;
  p.y = a.out;
  p.h = ws + w.h;
  p.parts = w.split1.parts;
  p.part = (float*)(ws + w.part);
  p.counters = (int*)(ws + w.counters);
  p.max_units = w.max_units;
  p.shape[0] = w.split0.shape;
  p.shape[1] = w.split1.shape;
  int rc;
  if ((rc = few_ring(p, 2, nb, table))) return rc;
  CUtensorMap maps[3];
  if ((rc = few_weight_map(&maps[0], a.w_gate, a.dtype, a.d, a.hidden, a.E, p.shape[0].rows))) return rc;
  if ((rc = few_weight_map(&maps[1], a.w_up, a.dtype, a.d, a.hidden, a.E, p.shape[0].rows))) return rc;
  if ((rc = few_weight_map(&maps[2], a.w_down, a.dtype, a.hidden, a.d, a.E, p.shape[1].rows))) return rc;
  const unsigned grid = (unsigned)num_sms(current_device());
  if (a.dtype == MOE_BF16)
    return few_kernel_nb<fewtc::kMoe, 1, __nv_bfloat16>(nb, maps, p, grid, table, a.stream);
  return few_kernel_nb<fewtc::kMoe, 0, __half>(nb, maps, p, grid, table, a.stream);
}

static int few_tokens_run(const FewArgs& a) {
  int rc = check_few(a);
  if (rc) return rc;
  if (a.num_tokens == 0 || a.d == 0) return MOE_OK;
  if (a.hidden == 0) {
    MOE_CUDA_CHECK(cudaMemsetAsync(a.out, 0, (size_t)a.num_tokens * a.d * dtype_size(a.dtype), a.stream));
    return MOE_OK;
  }
  const FewWorkspace w = few_workspace(a.num_tokens, a.d, a.hidden, a.E, a.topk, a.dtype);
  uint8_t* ws = (uint8_t*)a.workspace;
  float* logits = (float*)(ws + w.logits);
  const bool tc = few_tc_ok(a);
  int* counters = tc ? (int*)(ws + w.counters) : nullptr;
  const int num_counters = tc ? w.num_counters : 0;
  few::Routing r = {};
  r.num_tokens = (int)a.num_tokens;
  r.E = a.E;
  r.K = a.topk;
  if (a.w_router) {
    rc = MOE_DISPATCH_DTYPE(a.dtype, T, [&] { return few_router_launch<T>(a, logits, counters, num_counters); });
    if (rc) return rc;
    r.logits = logits;
  } else {
    r.weights = a.weights;
    r.indices = a.indices;
    if (tc) {
      if ((rc = zero_counters(counters, num_counters, a.stream))) return rc;
    }
  }
  if (tc) return few_tc_launch(a, r, w);
  return MOE_DISPATCH_DTYPE(a.dtype, T, [&] {
    const bool vec = (a.d * sizeof(T)) % 16 == 0 && (a.hidden * sizeof(T)) % 16 == 0 && aligned16(a.x) &&
                     aligned16(a.w_gate) && aligned16(a.w_up) && aligned16(a.w_down);
    return vec ? few_simt_launch<T, true>(a, r, w) : few_simt_launch<T, false>(a, r, w);
  });
}

}  // namespace moe

using namespace moe;

extern "C" {

size_t moe_few_tokens_workspace_bytes(int64_t num_tokens, int64_t d, int64_t hidden,
                                      int32_t num_experts, int32_t topk, int dtype) {
  if (num_tokens <= 0 || num_tokens > few::kMaxTokens || d < 0 || hidden < 0 || num_experts <= 0 ||
      topk <= 0 || topk > few::kMaxTopk)
    return 0;
  return few_workspace(num_tokens, d, hidden, num_experts, topk, dtype).total;
}

int moe_few_tokens_fwd(const void* x, const void* w_router, const float* router_bias,
                       const void* w_gate, const void* w_up, const void* w_down, int dtype,
                       int64_t num_tokens, int64_t d, int64_t hidden, int32_t num_experts,
                       int32_t topk, void* out, void* workspace, size_t workspace_bytes,
                       void* stream) {
  MOE_REQUIRE(w_router || num_tokens == 0, "few_tokens: w_router is NULL");
  FewArgs a = {};
  a.x = x; a.w_router = w_router; a.router_bias = router_bias;
  a.w_gate = w_gate; a.w_up = w_up; a.w_down = w_down; a.dtype = dtype;
  a.num_tokens = num_tokens; a.d = d; a.hidden = hidden; a.E = num_experts; a.topk = topk;
  a.out = out; a.workspace = workspace; a.workspace_bytes = workspace_bytes;
  a.stream = (cudaStream_t)stream;
  return few_tokens_run(a);
}

int moe_few_experts_fwd(const void* x, const float* weights, const int32_t* indices,
                        const void* w_gate, const void* w_up, const void* w_down, int dtype,
                        int64_t num_tokens, int64_t d, int64_t hidden, int32_t num_experts,
                        int32_t topk, void* out, void* workspace, size_t workspace_bytes,
                        void* stream) {
  FewArgs a = {};
  a.x = x; a.weights = weights; a.indices = indices;
  a.w_gate = w_gate; a.w_up = w_up; a.w_down = w_down; a.dtype = dtype;
  a.num_tokens = num_tokens; a.d = d; a.hidden = hidden; a.E = num_experts; a.topk = topk;
  a.out = out; a.workspace = workspace; a.workspace_bytes = workspace_bytes;
  a.stream = (cudaStream_t)stream;
  return few_tokens_run(a);
}

}  // extern "C"
