// linear / grouped_linear beside the tensor-core row tiles (gmm_sm100.cuh, kModeLinear): the
// CUDA-core epilogue, the backward's elementwise pass and the rows behind the last group.
//
//   z = A . op(B[g])^T + bias[g],  out = act(z) + residual
//   dz = dout * act'(z),  dbias[g] = sum of dz over the rows of g
#pragma once

#include "activation.cuh"
#include "few_tokens.cuh"
#include "gmm_simt.cuh"

namespace moe {

// Epilogue of gmm_rows_simt_kernel.
template <typename T>
struct LinearEpilogue {
  T* out;
  T* preact;          // may be NULL, like the next two
  const T* bias;      // [E, n]
  const T* residual;  // [m, n]
  int act;
  __device__ __forceinline__ void operator()(float acc, int g, int64_t row, int64_t n, int64_t N) const {
    const int64_t at = row * N + n;
    float z = acc;
    if (bias) z += to_f32(bias[(int64_t)g * N + n]);
    if (preact) preact[at] = from_f32<T>(z);
    float y = act_fwd_rt<sizeof(T) == 2>(act, z);
    if (residual) y += to_f32(residual[at]);
    out[at] = from_f32<T>(y);
  }
};

// Row chunks: every group's rows in pieces of `size`, one after the other.  prefix [E + 1] (shared
// memory) receives the first chunk of each group; ends with a __syncthreads().
__device__ __forceinline__ void row_chunks(int* prefix, const int32_t* offsets, int plus_one, int E,
                                           int64_t m, int size) {
  if (threadIdx.x < 32) {
    int run = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + (int)threadIdx.x;
      int c = 0;
      if (e < E) c = (int)((simt::group_range(offsets, plus_one, e, m).rows + size - 1) / size);
      int inc = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if ((int)threadIdx.x >= o) inc += v;
      }
      if (e < E) prefix[e] = run + inc - c;
      run += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (threadIdx.x == 0) prefix[E] = run;
  }
  __syncthreads();
}
// The group of chunk c: the last whose first chunk is not after it.
__device__ __forceinline__ int chunk_group(const int* prefix, int E, int c) {
  int lo = 0, hi = E - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= c) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// A few rows on the CUDA cores: one warp per weight row and up to kWarpRows rows of A, lanes along
// the contraction, so each weight is read once per kWarpRows rows and the latency does not grow
// with K tile by tile.
constexpr int kWarpRows = 8;

// VEC: 16-byte loads (rows that are 16-byte multiples).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
linear_rows_kernel(const T* __restrict__ A, const T* __restrict__ B, const LinearEpilogue<T> epi,
                   const int32_t* __restrict__ offsets, int plus_one, int E, int64_t m, int N, int K) {
  extern __shared__ int prefix[];
  row_chunks(prefix, offsets, plus_one, E, m, kWarpRows);
  constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
  const int lane = threadIdx.x & 31;
  const int64_t total = (int64_t)prefix[E] * N, warps = (int64_t)gridDim.x * 8;
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < total; i += warps) {
    const int c = (int)(i / N), n = (int)(i - (int64_t)c * N);
    const int g = chunk_group(prefix, E, c);
    const simt::GroupRange gr = simt::group_range(offsets, plus_one, g, m);
    const int64_t r0 = gr.start + (int64_t)(c - prefix[g]) * kWarpRows;
    const int rows = (int)min((int64_t)kWarpRows, gr.start + gr.rows - r0);
    const T* w = B + ((int64_t)g * N + n) * K;
    const T* a[kWarpRows];  // a row past the chunk repeats its first: loads need no branch
#pragma unroll
    for (int q = 0; q < kWarpRows; ++q) a[q] = A + (r0 + (q < rows ? q : 0)) * K;
    float acc[kWarpRows] = {};
#pragma unroll 2
    for (int k = lane * V; k < K; k += 32 * V) {
      float wv[V];
      few::load_vec<T, VEC>(w + k, wv);
#pragma unroll
      for (int q = 0; q < kWarpRows; ++q) {
        float av[V];
        few::load_vec<T, VEC>(a[q] + k, av);
#pragma unroll
        for (int j = 0; j < V; ++j) acc[q] = fmaf(av[j], wv[j], acc[q]);
      }
    }
    float mine = 0.f;
#pragma unroll
    for (int q = 0; q < kWarpRows; ++q) {
      float v = acc[q];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == q) mine = v;
    }
    if (lane < rows) epi(mine, g, r0 + lane, n, N);
  }
}

// ------------------------------------------------------------------ backward, elementwise
// One pass over dout and z: dz written (unless the activation is none: dz is dout) and the
// column sums of dz taken from its fp32 values before they are rounded.  A block owns
// kDzRows consecutive rows of one group and 32 V columns; its column sums go to
// partial[chunk, n] and dbias_kernel adds the chunks of a group in order, so the result does
// not depend on the order blocks run in.  HBM-bound: 2 reads + 1 write of m * n elements (bf16,
// 4099 x 7168, cold L2: 27 us at the copy rate, 49 us for relu, gelu and gelu_tanh, 59 us for silu,
// and 10 us with the bias gradient's second launch).  The activation is a template parameter and
// registers are capped at 64: three rows' loads in flight per thread, four blocks per SM (one kernel
// for all activations: silu 78 us; four rows: silu 66 us, relu and silu spill 40 to 52 bytes; two
// rows: gelu 64 us).  relu and silu still spill 16 to 20 bytes.
constexpr int kDzRows = 64;
constexpr int kDzThreads = 256;

// V = elements of a thread's column group (8 for 16-bit and 4 for fp32 when rows are 16-byte
// multiples, else 1); blockDim = (columns / V = 32, 8 rows).
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kDzThreads, 4)
dz_kernel(const T* __restrict__ dout, const T* __restrict__ z, T* __restrict__ dz,
          float* __restrict__ partial, const int32_t* __restrict__ offsets, int plus_one, int E,
          int64_t m, int64_t N) {
  extern __shared__ int prefix[];
  __shared__ float red[8][32 * V + 1];
  row_chunks(prefix, offsets, plus_one, E, m, kDzRows);
  const int chunks = prefix[E];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t n = ((int64_t)blockIdx.x * 32 + tx) * V;
  for (int c = blockIdx.y; c < chunks; c += gridDim.y) {
    const int lo = chunk_group(prefix, E, c);
    const simt::GroupRange gr = simt::group_range(offsets, plus_one, lo, m);
    const int64_t r0 = gr.start + (int64_t)(c - prefix[lo]) * kDzRows;
    const int64_t r1 = min(r0 + kDzRows, gr.start + gr.rows);
    float sum[V] = {};
    if (n < N) {
      union Vec {
        typename std::conditional<V * sizeof(T) == 16, uint4, T>::type u;
        T v[V];
      };
#pragma unroll 3
      for (int64_t r = r0 + ty; r < r1; r += 8) {
        const int64_t at = r * N + n;
        Vec d, zz, o;
        d.u = __ldg(reinterpret_cast<const decltype(d.u)*>(dout + at));
        if constexpr (ACT != MOE_ACT_NONE) zz.u = __ldg(reinterpret_cast<const decltype(d.u)*>(z + at));
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float v = to_f32(d.v[j]);
          if constexpr (ACT != MOE_ACT_NONE) {
            v *= act_bwd<ACT, sizeof(T) == 2>(to_f32(zz.v[j]));
            o.v[j] = from_f32<T>(v);
          }
          sum[j] += v;
        }
        if constexpr (ACT != MOE_ACT_NONE) *reinterpret_cast<decltype(d.u)*>(dz + at) = o.u;
      }
    }
    if (partial) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < V; ++j) red[ty][tx * V + j] = sum[j];
      __syncthreads();
      for (int i = threadIdx.x; i < 32 * V; i += kDzThreads) {
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q) s += red[q][i];
        const int64_t col = (int64_t)blockIdx.x * 32 * V + i;
        if (col < N) partial[(int64_t)c * N + col] = s;
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kDzThreads)
dbias_kernel(const float* __restrict__ partial, T* __restrict__ dbias,
             const int32_t* __restrict__ offsets, int plus_one, int E, int64_t m, int64_t N) {
  extern __shared__ int prefix[];
  __shared__ float red[8][33];
  pdl_wait();
  row_chunks(prefix, offsets, plus_one, E, m, kDzRows);
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t n = (int64_t)blockIdx.x * 32 + tx;
  for (int g = blockIdx.y; g < E; g += gridDim.y) {
    float s = 0.f;
    if (n < N)
      for (int c = prefix[g] + ty; c < prefix[g + 1]; c += 8) s += __ldcg(partial + (int64_t)c * N + n);
    __syncthreads();
    red[ty][tx] = s;
    __syncthreads();
    if (ty == 0 && n < N) {
#pragma unroll
      for (int q = 1; q < 8; ++q) s += red[q][tx];
      dbias[(int64_t)g * N + n] = from_f32<T>(s);
    }
  }
}

// Rows behind the last group (rows >= the last offset) belong to no product: out = residual, or
// zero without one.
template <typename T>
__global__ void __launch_bounds__(256)
tail_rows_kernel(T* __restrict__ out, const T* __restrict__ residual, const int32_t* __restrict__ offsets,
                 int last, int64_t m, int64_t N) {
  int64_t r0 = offsets[last];
  if (r0 < 0) r0 = 0;
  const int64_t total = (m - r0) * N;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x)
    out[r0 * N + i] = residual ? residual[r0 * N + i] : from_f32<T>(0.f);
}

}  // namespace moe
