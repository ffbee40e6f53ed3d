// CUDA-core grouped GEMM for the requests the tensor-core kernel does not take:
// fp32 operands (the reference runs fp32 through its non-TMA Triton kernel,
// triton_gmm_ops/grouped_gemm_ops.py:20-69 and :126-165) and 16-bit operands whose rows
// are not 16-byte multiples (TMA cannot address them).  Exact fp32 FMA accumulation.
//
// 64x64 output tile per 256-thread block, 4x4 outputs per thread, the contraction staged through
// shared memory 32 deep in two buffers: a block loads the next slice into registers while it
// multiplies the present one (fp32 1024^3: 103 us, 21 TFLOP/s; a training step of M = 333, K = 257,
// N = 130, where the latency of a slice counts: 128 us with 16-deep slices and no second buffer,
// 64 us).  Every output is one chain of FMAs in ascending k, whatever the tiling.  Like the
// reference, the row-mode grid is sized by the whole row count per expert slot and tiles past an expert's end
// return at once, so no host synchronisation is needed.
#pragma once

#include "common.cuh"

namespace moe {
namespace simt {

constexpr int TM = 64, TN = 64, TK = 32;
constexpr int kPitch = 68;  // floats between k rows of a staged tile (16-byte aligned)
constexpr int kSlice = TM * TK / 256;  // elements of each operand that a thread stages

struct GroupRange {
  int64_t start, rows;
};

// offsets == nullptr: one group of all m_total rows.
__device__ __forceinline__ GroupRange group_range(const int32_t* offsets, int plus_one, int g,
                                                  int64_t m_total) {
  GroupRange r;
  if (offsets == nullptr) { r.start = 0; r.rows = m_total; return r; }
  if (plus_one) { r.start = offsets[g]; r.rows = (int64_t)offsets[g + 1] - offsets[g]; }
  else { r.start = g > 0 ? offsets[g - 1] : 0; r.rows = (int64_t)offsets[g] - r.start; }
  if (r.rows < 0) r.rows = 0;
  return r;
}

// acc[i][j] += sum over k of a(ty * 4 + i, k) * b(tx * 4 + j, k): load_*(k0, i) fetches staged element
// i of the slice at k0, at_*(i) is its place in the [TK][kPitch] tile.
template <typename LoadA, typename LoadB, typename AtA, typename AtB>
__device__ __forceinline__ void tile_product(float (&acc)[4][4], int64_t Kc, LoadA load_a, LoadB load_b,
                                             AtA at_a, AtB at_b) {
  __shared__ __align__(16) float As[2][TK * kPitch];
  __shared__ __align__(16) float Bs[2][TK * kPitch];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float ra[kSlice], rb[kSlice];
#pragma unroll
  for (int j = 0; j < kSlice; ++j) {
    ra[j] = load_a(0, threadIdx.x + j * 256);
    rb[j] = load_b(0, threadIdx.x + j * 256);
  }
  int buf = 0;
  for (int64_t k0 = 0; k0 < Kc; k0 += TK, buf ^= 1) {
#pragma unroll
    for (int j = 0; j < kSlice; ++j) {
      As[buf][at_a(threadIdx.x + j * 256)] = ra[j];
      Bs[buf][at_b(threadIdx.x + j * 256)] = rb[j];
    }
    // One barrier a slice: this buffer is written again two slices later, after the next barrier.
    __syncthreads();
    if (k0 + TK < Kc) {
#pragma unroll
      for (int j = 0; j < kSlice; ++j) {
        ra[j] = load_a(k0 + TK, threadIdx.x + j * 256);
        rb[j] = load_b(k0 + TK, threadIdx.x + j * 256);
      }
    }
#pragma unroll 8
    for (int kk = 0; kk < TK; ++kk) {
      const float4 a = *reinterpret_cast<const float4*>(&As[buf][kk * kPitch + ty * 4]);
      const float4 b = *reinterpret_cast<const float4*>(&Bs[buf][kk * kPitch + tx * 4]);
      const float av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(av[i], bv[j], acc[i][j]);
    }
  }
}

// What happens to a finished element (row, column n of group g); this one stores it.
template <typename T>
struct StoreEpilogue {
  T* C;
  __device__ __forceinline__ void operator()(float acc, int, int64_t row, int64_t n, int64_t Nout) const {
    C[row * Nout + n] = from_f32<T>(acc);
  }
};

// Row mode: C[start+m, n] = sum_k A[start+m, k] * B(g, n, k),
// B(g, n, k) = b_mn ? B[(g*Kc + k)*Nout + n] : B[(g*Nout + n)*Kc + k].
template <typename T, typename Epi>
__global__ void __launch_bounds__(256)
gmm_rows_simt_kernel(const T* __restrict__ A, const T* __restrict__ B, const Epi epi,
                     const int32_t* __restrict__ offsets, int plus_one, int64_t m_total,
                     int64_t Nout, int64_t Kc, int b_mn) {
  const int g = blockIdx.z;
  const GroupRange gr = group_range(offsets, plus_one, g, m_total);
  const int64_t m0 = (int64_t)blockIdx.x * TM;
  if (m0 >= gr.rows) return;
  const int64_t n0 = (int64_t)blockIdx.y * TN;
  const T* Ag = A + gr.start * Kc;
  const T* Bg = B + (int64_t)g * Nout * Kc;
  float acc[4][4] = {};
  // Slices are read along whichever dimension is contiguous in memory.
  auto load_a = [&](int64_t k0, int i) {
    const int kk = i % TK, mm = i / TK;
    const int64_t m = m0 + mm, k = k0 + kk;
    return (m < gr.rows && k < Kc) ? to_f32(Ag[m * Kc + k]) : 0.f;
  };
  auto load_b = [&](int64_t k0, int i) {
    const int kk = b_mn ? i / TN : i % TK, nn = b_mn ? i % TN : i / TK;
    const int64_t n = n0 + nn, k = k0 + kk;
    return (n < Nout && k < Kc) ? to_f32(b_mn ? Bg[k * Nout + n] : Bg[n * Kc + k]) : 0.f;
  };
  auto at_a = [](int i) { return (i % TK) * kPitch + i / TK; };
  auto at_b = [&](int i) { return b_mn ? (i / TN) * kPitch + i % TN : (i % TK) * kPitch + i / TK; };
  tile_product(acc, Kc, load_a, load_b, at_a, at_b);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty * 4 + i;
    if (m >= gr.rows) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx * 4 + j;
      if (n < Nout) epi(acc[i][j], g, gr.start + m, n, Nout);
    }
  }
}

// Wgrad mode: Out[g, p, q] = sum_{m in expert g} X[m, p] * Y[m, q]  (zeros for empty g).
template <typename T>
__global__ void __launch_bounds__(256)
gmm_wgrad_simt_kernel(const T* __restrict__ X, const T* __restrict__ Y, T* __restrict__ Out,
                      const int32_t* __restrict__ offsets, int plus_one, int64_t m_total,
                      int64_t P, int64_t Q) {
  const int g = blockIdx.z;
  const GroupRange gr = group_range(offsets, plus_one, g, m_total);
  const int64_t p0 = (int64_t)blockIdx.y * TM, q0 = (int64_t)blockIdx.x * TN;
  const T* Xg = X + gr.start * P;
  const T* Yg = Y + gr.start * Q;
  float acc[4][4] = {};
  auto load_x = [&](int64_t r0, int i) {
    const int64_t r = r0 + i / TM, pi = p0 + i % TM;
    return (r < gr.rows && pi < P) ? to_f32(Xg[r * P + pi]) : 0.f;
  };
  auto load_y = [&](int64_t r0, int i) {
    const int64_t r = r0 + i / TN, qi = q0 + i % TN;
    return (r < gr.rows && qi < Q) ? to_f32(Yg[r * Q + qi]) : 0.f;
  };
  auto at = [](int i) { return (i / TM) * kPitch + i % TM; };
  tile_product(acc, gr.rows, load_x, load_y, at, at);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t pi = p0 + ty * 4 + i;
    if (pi >= P) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t qi = q0 + tx * 4 + j;
      if (qi < Q) Out[((int64_t)g * P + pi) * Q + qi] = from_f32<T>(acc[i][j]);
    }
  }
}

}  // namespace simt
}  // namespace moe
