// A whole SwiGLU mixture-of-experts layer for a few tokens (decoding).
//
//   l = x . Wr^T + b          p, idx = softmax over the K largest l, per token
//   h[t,k] = silu(x[t] . Wg[idx]^T) * (x[t] . Wu[idx]^T)
//   y[t]   = sum_k p[t,k] * (h[t,k] . Wd[idx]^T)
//
// With a few tokens every picked expert sees one row or a few, so the layer is a single
// stream over the picked experts' weights: 3 * d * H elements each, against 2 * T * d for the
// activations.  The time floor is those bytes over the HBM rate.
//
// This file holds the router, the routing plan that every block of the expert kernels builds
// for itself in shared memory, and the CUDA-core expert kernels (fp32, and 16-bit operands
// whose rows are not 16-byte multiples).
#pragma once

#include "common.cuh"
#include "swiglu.cuh"

namespace moe {
namespace few {

constexpr int kMaxTokens = 128;
constexpr int kMaxTopk = 16;
constexpr int kMaxExperts = 1024;

// ------------------------------------------------------------------------- router
// logits[t, e] = x[t] . Wr[e] + bias[e] in fp32, never rounded to the operands' type: the
// top-k is a comparison, and logits rounded to bf16 tie often.  Products of 16-bit operands
// are exact in fp32; each lane adds runs of 8 products in fp32 and the runs in fp64, so the
// logit carries the error of a few fp32 roundings at any d.
// One warp per (expert, group of kRouterTokens tokens).
constexpr int kRouterTokens = 4;

template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
router_kernel(const T* __restrict__ x, const T* __restrict__ wr, const float* __restrict__ bias,
              float* __restrict__ logits, int num_tokens, int d, int E, int* __restrict__ zero,
              int num_zero) {
  pdl_launch_dependents();
  // The counters of the expert kernel that follows (a previous call may still have run when
  // this launch was queued, but not once its blocks start).
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < num_zero; i += gridDim.x * blockDim.x)
    zero[i] = 0;
  const int lane = threadIdx.x & 31;
  const int groups = (num_tokens + kRouterTokens - 1) / kRouterTokens;
  const int warps = gridDim.x * (blockDim.x >> 5);
  constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
  for (int64_t w = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
       w < (int64_t)groups * E; w += warps) {
    const int e = (int)(w % E), t0 = (int)(w / E) * kRouterTokens;
    const T* row = wr + (int64_t)e * d;
    double acc[kRouterTokens] = {};
    for (int k = lane * V; k < d; k += 32 * V) {
      float wv[V];
      if constexpr (VEC) {
        const uint4 raw = __ldg(reinterpret_cast<const uint4*>(row + k));
#pragma unroll
        for (int j = 0; j < V; ++j) wv[j] = to_f32(reinterpret_cast<const T*>(&raw)[j]);
      } else {
        wv[0] = to_f32(row[k]);
      }
#pragma unroll
      for (int i = 0; i < kRouterTokens; ++i) {
        if (t0 + i >= num_tokens) break;
        const T* xr = x + (int64_t)(t0 + i) * d + k;
        float s = 0.f;
        if constexpr (VEC) {
          const uint4 raw = __ldg(reinterpret_cast<const uint4*>(xr));
#pragma unroll
          for (int j = 0; j < V; ++j) s = fmaf(to_f32(reinterpret_cast<const T*>(&raw)[j]), wv[j], s);
        } else {
          s = to_f32(xr[0]) * wv[0];
        }
        acc[i] += (double)s;
      }
    }
#pragma unroll
    for (int i = 0; i < kRouterTokens; ++i) {
      if (t0 + i >= num_tokens) break;
      double v = acc[i];
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
      if (lane == 0) {
        if (bias) v += (double)bias[e];
        logits[(int64_t)(t0 + i) * E + e] = (float)v;
      }
    }
  }
}

// ------------------------------------------------------------------------- top-k
// Order-preserving map of a float to an unsigned key: larger float, larger key; -0 and +0 are
// equal; NaN is above everything (it is picked, and its token's weights become NaN).  Every
// key of a float is at least 1 (0 marks a value already picked).
__device__ __forceinline__ uint32_t rank_key(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0xffffffffu) return __uint_as_float(0x7fffffffu);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// One warp: the K largest of row[0..E) (ties to the lower index) and the softmax over them.
// An expert whose logit is -inf is masked: its slot gets index -1 and weight 0, so a token
// with no unmasked expert has an all-zero output row.
// VPT = logits held per lane (E <= 32 * VPT).
template <int VPT>
__device__ __forceinline__ void topk_token(const float* __restrict__ row, int E, int K, int lane,
                                           int16_t* __restrict__ idx, float* __restrict__ w) {
  uint32_t key[VPT];
  uint32_t best = 0;
  int best_e = 0x7fffffff;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    key[j] = 0;
    if (j * 32 < E) {
      const int e = j * 32 + lane;
      if (e < E) key[j] = rank_key(__ldcg(row + e));
      if (key[j] > best) { best = key[j]; best_e = e; }
    }
  }
  uint32_t mine = 0;  // lane k keeps pick k
  int my_e = -1;
  for (int k = 0; k < K; ++k) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    const int e = __reduce_min_sync(0xffffffffu, best == top ? best_e : 0x7fffffff);
    if (lane == k) { mine = top; my_e = e; }
    if (best == top && best_e == e) {  // the owner finds its next best
      best = 0;
      best_e = 0x7fffffff;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        if (j * 32 < E) {
          if (j * 32 + lane == e) key[j] = 0;
          if (key[j] > best) { best = key[j]; best_e = j * 32 + lane; }
        }
      }
    }
  }
  const float v = lane < K ? key_value(mine) : -INFINITY;
  const float m = key_value(__shfl_sync(0xffffffffu, mine, 0));
  const bool masked = v == -INFINITY;
  float ex = masked ? 0.f : expf(v - m);
  float s = ex;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  if (lane < K) {
    idx[lane] = masked ? (int16_t)-1 : (int16_t)my_e;
    w[lane] = masked ? 0.f : ex / s;
  }
}

// ------------------------------------------------------------------------- plan
// What a block needs to know about the routing: for each slot s = t*K + k its weight and its
// position in expert order (stable: experts ascending, slots ascending within an expert; -1
// for a dropped slot), the slot at each position, and the list of work units: at most
// `rows_per_unit` consecutive positions of one expert.
struct Plan {
  float* w;           // [S]
  int* cnt;           // [E] rows of expert e
  int* off;           // [E + 1]
  int16_t* pos;       // [S]; holds the slot's expert while the plan is built
  int16_t* rank;      // [S] scratch
  uint16_t* slot;     // [S]
  int16_t* unit_e;    // [U]
  uint16_t* unit_pos; // [U] first position
  uint16_t* unit_n;   // [U] rows
  int* num_units;
};

__host__ __device__ inline int plan_max_units(int S, int E, int rows_per_unit) {
  return (S < E ? S : E) + S / rows_per_unit;
}
__host__ __device__ inline int plan_bytes(int S, int E, int rows_per_unit) {
  const int U = plan_max_units(S, E, rows_per_unit);
  return ((4 * S + 4 * E + 4 * (E + 1) + 2 * S * 3 + 2 * U * 3 + 4 + 4) + 15) / 16 * 16;
}
__device__ inline Plan plan_view(uint8_t* mem, int S, int E, int rows_per_unit) {
  const int U = plan_max_units(S, E, rows_per_unit);
  Plan p;
  p.w = reinterpret_cast<float*>(mem);
  p.cnt = reinterpret_cast<int*>(p.w + S);
  p.off = p.cnt + E;
  p.num_units = p.off + E + 1;
  p.pos = reinterpret_cast<int16_t*>(p.num_units + 1);
  p.rank = p.pos + S;
  p.slot = reinterpret_cast<uint16_t*>(p.rank + S);
  p.unit_e = reinterpret_cast<int16_t*>(p.slot + S);
  p.unit_pos = reinterpret_cast<uint16_t*>(p.unit_e + U);
  p.unit_n = p.unit_pos + U;
  return p;
}

struct Routing {
  const float* logits;     // [T, E], or
  const float* weights;    // [T, K] and
  const int32_t* indices;  // [T, K] when logits is NULL
  int num_tokens, E, K;
};

// Built by the whole block (a multiple of 32 threads); ends with a __syncthreads().  Every
// block of a launch builds the same plan from the same inputs, so no block waits for another.
__device__ __forceinline__ void build_plan(const Plan& p, const Routing& r, int rows_per_unit) {
  const int S = r.num_tokens * r.K;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  for (int e = threadIdx.x; e < r.E; e += blockDim.x) p.cnt[e] = 0;
  if (r.logits) {
    for (int t = warp; t < r.num_tokens; t += warps) {
      const float* row = r.logits + (int64_t)t * r.E;
      if (r.E <= 64) topk_token<2>(row, r.E, r.K, lane, p.pos + t * r.K, p.w + t * r.K);
      else if (r.E <= 256) topk_token<8>(row, r.E, r.K, lane, p.pos + t * r.K, p.w + t * r.K);
      else topk_token<kMaxExperts / 32>(row, r.E, r.K, lane, p.pos + t * r.K, p.w + t * r.K);
    }
  } else {
    for (int s = threadIdx.x; s < S; s += blockDim.x) {
      const int e = r.indices[s];
      const bool ok = e >= 0 && e < r.E;
      if (!ok && blockIdx.x == 0) raise_device_error(2);
      p.pos[s] = ok ? (int16_t)e : (int16_t)-1;
      p.w[s] = r.weights[s];
    }
  }
  __syncthreads();
  if (warp == 0) {
    // Stable rank of each slot within its expert, 32 slots at a time.
    for (int s0 = 0; s0 < S; s0 += 32) {
      const int s = s0 + lane;
      const int e = s < S ? p.pos[s] : -1;
      const unsigned same = __match_any_sync(0xffffffffu, e);
      const int base = e >= 0 ? p.cnt[e] : 0;
      __syncwarp();
      if (s < S) p.rank[s] = (int16_t)(base + __popc(same & ((1u << lane) - 1u)));
      if (e >= 0 && (same >> lane) == 1u) p.cnt[e] = base + __popc(same);  // highest lane
      __syncwarp();
    }
    // Offsets and units, 32 experts at a time.
    int rows = 0, units = 0;
    for (int e0 = 0; e0 < r.E; e0 += 32) {
      const int e = e0 + lane;
      const int n = e < r.E ? p.cnt[e] : 0;
      const int u = (n + rows_per_unit - 1) / rows_per_unit;
      int ni = n, ui = u;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, ni, o), b = __shfl_up_sync(0xffffffffu, ui, o);
        if (lane >= o) { ni += a; ui += b; }
      }
      if (e < r.E) {
        const int first = rows + ni - n, unit0 = units + ui - u;
        p.off[e] = first;
        for (int i = 0; i < u; ++i) {
          p.unit_e[unit0 + i] = (int16_t)e;
          p.unit_pos[unit0 + i] = (uint16_t)(first + i * rows_per_unit);
          const int left = n - i * rows_per_unit;
          p.unit_n[unit0 + i] = (uint16_t)(left < rows_per_unit ? left : rows_per_unit);
        }
      }
      rows += __shfl_sync(0xffffffffu, ni, 31);
      units += __shfl_sync(0xffffffffu, ui, 31);
    }
    if (lane == 0) {
      p.off[r.E] = rows;
      *p.num_units = units;
    }
  }
  __syncthreads();
  for (int s = threadIdx.x; s < S; s += blockDim.x) {
    const int e = p.pos[s];
    if (e >= 0) {
      const int at = p.off[e] + p.rank[s];
      p.pos[s] = (int16_t)at;
      p.slot[at] = (uint16_t)s;
    }
  }
  __syncthreads();
}

// ------------------------------------------------------------------------- CUDA cores
// One warp per weight row (and per unit of up to 8 rows of activations), exact fp32 FMAs; h and the
// experts' outputs are kept in fp32.  Three launches: gate and up, down, combine.  Bound by the
// weight stream at one or two rows per expert, by loads in flight at more.
constexpr int kSimtRows = 8;

template <typename T, bool VEC>
__device__ __forceinline__ void load_vec(const T* p, float* v) {
  if constexpr (VEC) {
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(p));
#pragma unroll
    for (int j = 0; j < 16 / (int)sizeof(T); ++j) v[j] = to_f32(reinterpret_cast<const T*>(&raw)[j]);
  } else {
    v[0] = to_f32(*p);
  }
}

// acc[q] += <w, x[q]> over k for this lane (V elements at a time); rows past a unit repeat its first,
// so that no load waits for a branch.
template <typename T, bool VEC, int NW>
__device__ __forceinline__ void lane_dots(const T* const (&w)[NW], const T* const (&x)[kSimtRows], int K,
                                          int lane, float (&acc)[NW][kSimtRows]) {
  constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
#pragma unroll 2
  for (int k = lane * V; k < K; k += 32 * V) {
    float wv[NW][V];
#pragma unroll
    for (int i = 0; i < NW; ++i) load_vec<T, VEC>(w[i] + k, wv[i]);
#pragma unroll
    for (int q = 0; q < kSimtRows; ++q) {
      float xv[V];
      load_vec<T, VEC>(x[q] + k, xv);
#pragma unroll
      for (int i = 0; i < NW; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) acc[i][q] = fmaf(wv[i][j], xv[j], acc[i][q]);
    }
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// h[pos, j]; block 0 also leaves each slot's position (-1: dropped) and weight for the combine.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
gate_up_simt_kernel(const T* __restrict__ x, const T* __restrict__ wg, const T* __restrict__ wu,
                    float* h, int* slot_pos, float* slot_w, Routing r, int d, int H) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int S = r.num_tokens * r.K;
  const Plan p = plan_view(smem, S, r.E, kSimtRows);
  pdl_launch_dependents();
  pdl_wait();
  build_plan(p, r, kSimtRows);
  if (blockIdx.x == 0)
    for (int s = threadIdx.x; s < S; s += blockDim.x) {
      slot_pos[s] = p.pos[s];
      slot_w[s] = p.w[s];
    }
  const int lane = threadIdx.x & 31;
  const int warps = gridDim.x * (blockDim.x >> 5);
  const int64_t total = (int64_t)*p.num_units * H;
  for (int64_t i = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i < total; i += warps) {
    const int u = (int)(i / H), j = (int)(i - (int64_t)u * H);
    const int n = p.unit_n[u], pos0 = p.unit_pos[u];
    const int64_t row = ((int64_t)p.unit_e[u] * H + j) * d;
    const T* const w[2] = {wg + row, wu + row};
    const T* xr[kSimtRows];
#pragma unroll
    for (int q = 0; q < kSimtRows; ++q) xr[q] = x + (int64_t)(p.slot[pos0 + (q < n ? q : 0)] / r.K) * d;
    float acc[2][kSimtRows] = {};
    lane_dots<T, VEC, 2>(w, xr, d, lane, acc);
    float g = 0.f, v = 0.f;
#pragma unroll
    for (int q = 0; q < kSimtRows; ++q) {
      const float a = warp_sum(acc[0][q]), b = warp_sum(acc[1][q]);
      if (lane == q) { g = a; v = b; }
    }
    if (lane < n) h[(int64_t)(pos0 + lane) * H + j] = g * sigmoid_f32(g) * v;
  }
}

// o[pos, n] = h[pos] . Wd[e][n].  h is fp32, so the weights are widened as they are loaded.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
down_simt_kernel(const float* h, const T* __restrict__ wd, float* o, Routing r, int d, int H) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int S = r.num_tokens * r.K;
  const Plan p = plan_view(smem, S, r.E, kSimtRows);
  pdl_launch_dependents();
  pdl_wait();
  build_plan(p, r, kSimtRows);
  constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
  const int lane = threadIdx.x & 31;
  const int warps = gridDim.x * (blockDim.x >> 5);
  const int64_t total = (int64_t)*p.num_units * d;
  for (int64_t i = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i < total; i += warps) {
    const int u = (int)(i / d), col = (int)(i - (int64_t)u * d);
    const int n = p.unit_n[u], pos0 = p.unit_pos[u];
    const T* w = wd + ((int64_t)p.unit_e[u] * d + col) * H;
    const float* hr[kSimtRows];
#pragma unroll
    for (int q = 0; q < kSimtRows; ++q) hr[q] = h + (int64_t)(pos0 + (q < n ? q : 0)) * H;
    float acc[kSimtRows] = {};
#pragma unroll 2
    for (int k = lane * V; k < H; k += 32 * V) {
      float wv[V];
      load_vec<T, VEC>(w + k, wv);
#pragma unroll
      for (int q = 0; q < kSimtRows; ++q) {
        float hv[V];
        if constexpr (VEC) {
#pragma unroll
          for (int j = 0; j < V; j += 4)
            *reinterpret_cast<float4*>(hv + j) = *reinterpret_cast<const float4*>(hr[q] + k + j);
        } else {
          hv[0] = hr[q][k];
        }
#pragma unroll
        for (int j = 0; j < V; ++j) acc[q] = fmaf(wv[j], hv[j], acc[q]);
      }
    }
    float mine = 0.f;
#pragma unroll
    for (int q = 0; q < kSimtRows; ++q) {
      const float a = warp_sum(acc[q]);
      if (lane == q) mine = a;
    }
    if (lane < n) o[(int64_t)(pos0 + lane) * d + col] = mine;
  }
}

// y[t] = sum over t's slots, in order, of their weight times their row of o.
template <typename T>
__global__ void __launch_bounds__(256)
combine_simt_kernel(const float* o, const int* slot_pos, const float* slot_w, T* __restrict__ y,
                    int num_tokens, int K, int d) {
  pdl_wait();
  const int64_t total = (int64_t)num_tokens * d;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int t = (int)(i / d), col = (int)(i - (int64_t)t * d);
    float acc = 0.f;
    for (int k = 0; k < K; ++k) {
      const int pos = slot_pos[t * K + k];
      if (pos >= 0) acc = fmaf(slot_w[t * K + k], o[(int64_t)pos * d + col], acc);
    }
    y[i] = from_f32<T>(acc);
  }
}

}  // namespace few
}  // namespace moe
