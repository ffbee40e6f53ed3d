// Few rows against many weights on the sm_100a tensor cores: the expert part of the few-token
// MoE layer (kMoe) and linear / grouped_linear for a few rows (kLinear).
//
// With n rows (1 to 64) per weight matrix the product does 2 n flops per 2-byte weight, far
// below the ridge: the kernel is a stream over the weights and everything else hides behind
// it.  So the weights are the MMA's A operand (M = 128 weight rows) and the activations its B
// operand (N = n rounded up to 16): one 64-deep block of 256 weight rows is a 32 KB stage, its
// 8 MMAs take a fraction of the stage's HBM time, and no register touches a weight.
//
//   kMoe     phase 0: a tile is 128 columns of h: 128 gate rows (accumulator D0) and the same
//            128 up rows (D1) of one unit (an expert's rows, at most NB); its epilogue forms
//            h = silu(gate) * up in fp32 and rounds it once to 16 bits (as an MMA operand it
//            has to be).
//            phase 1: a tile is 256 rows of Wd (D0, D1) times the unit's h.  Its fp32 results
//            are stored, never rounded; the block that completes a 256-column strip of y adds
//            p * result over the slots in order.
//   kLinear  one phase: 256 weight rows times up to NB rows; bias, activation, residual.
//
// Work split.  A phase is a flat list of 64-deep blocks (tile-major), cut into G chunks of equal
// size whatever the sizes are, so every SM streams the same number of bytes.  A tile cut by a
// chunk border leaves fp32 partials; the chunk that finds the tile complete (an atomic counter
// of finished blocks) adds them in chunk order, so results do not depend on timing.
//
// kMoe's chunks are handed out by an atomic ticket, phase 0's before phase 1's.  A block waits
// only for phase-0 chunks, each of which a running block has taken and finishes without waiting
// for anyone: the kernel makes progress whatever share of its blocks is resident.  The weight
// producer never waits for h, so the ring (about 200 KB per SM) fills with Wd while the last h
// tiles are finished: the stream does not stop between the phases.
//
// Warp roles (256 threads, one block per SM):
//   warp 0      weights: TMA boxes of 64 x 128, 128-byte swizzle; also fetches the tickets.
//   warp 1      TMEM owner and MMA issuer.
//   warps 2-3   activations: 16-byte cp.async into the same swizzle (rows are gathered: any
//               token, any h row), handed over kLag stages later.
//   warps 4-7   epilogue, one accumulator lane (weight row) per thread.
//
// Every wait is bounded; one that gives up sets the abort flag and device error 1.
#pragma once

#include "activation.cuh"
#include "few_tokens.cuh"
#include "gmm_sm100.cuh"
#include "gmm_simt.cuh"

namespace moe {
namespace fewtc {

constexpr int kThreads = 256;
constexpr int BK = 64;
constexpr uint32_t kBoxBytes = 128 * 128;        // 128 weight rows x 64 16-bit columns
constexpr uint32_t kWBytes = 2 * kBoxBytes;      // weights of a stage
constexpr int kLag = 3;                          // stages between a cp.async and its hand-over
constexpr int kMaxStages = 8;
constexpr uint64_t kWaitNs = gmm::kWaitTimeoutNs;

enum Mode { kMoe = 0, kLinear = 1 };

struct Params {
  // kMoe
  few::Routing r;
  int d, H;
  void* h;       // [S, H]
  float* o;      // [S, strips * 256] results of phase 1 (each tile's first chunk)
  float* extra;  // [max_chunks, NB, 256] the other chunks of a tile
  void* y;       // [T, d]; kLinear: [m, N]
  // kLinear
  const int32_t* offsets;
  int plus_one, E;
  int64_t m;
  int N, K;
  const void* bias;
  const void* residual;
  void* preact;
  int act;
  // both
  const void* x;     // activations, rows of d (K) elements
  float* part;       // [2 * max_chunks, NB, 256] partials of phase 0 (kLinear: of the phase)
  int* counters;     // zeroed before the launch: ticket, tile[max_chunks], done[units], strip[]
  int max_chunks, max_units;
  int min_blocks;    // blocks of a chunk, at least
  int stages;
};

struct Ctl {
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint64_t tmem_full[2], tmem_empty[2];
  uint64_t tk_full[2], tk_empty[2];
  int tk[2];
  uint32_t tmem_base;
  int abort;
  int flag;
  int num_units;
};

// Units of kLinear: at most NB consecutive rows of one group.
struct RowUnits {
  int16_t* e;
  uint16_t* n;
  int* row;
};
__host__ __device__ inline int row_units_max(int64_t m, int E, int nb) {
  return (int)((m < E ? m : E) + m / nb + 1);
}
__host__ __device__ inline int row_units_bytes(int units) { return (8 * units + 15) / 16 * 16; }

// A phase's blocks: `tiles` tiles of KB blocks, cut into G chunks.
struct Phase {
  int KB;
  long long total;
  int G;
  __device__ __forceinline__ void set(long long tiles, int kb, int max_chunks, int min_blocks) {
    KB = kb;
    total = tiles * kb;
    const long long g = total / min_blocks;
    G = total == 0 ? 0 : (int)(g < 1 ? 1 : (g < max_chunks ? g : max_chunks));
  }
  __device__ __forceinline__ long long begin(int c) const { return c * total / G; }
  // The chunk that holds block b: the largest c with begin(c) <= b.
  __device__ __forceinline__ int chunk_of(long long b) const { return (int)(((b + 1) * G - 1) / total); }
};

template <int MODE, int FMT, typename T, int NB>
__global__ void __launch_bounds__(kThreads, 1)
few_kernel(const __grid_constant__ CUtensorMap map0, const __grid_constant__ CUtensorMap map1,
           const __grid_constant__ CUtensorMap map2, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr uint32_t kStage = kWBytes + NB * 128;
  constexpr uint32_t kTmemCols = 4 * NB;  // two accumulator pairs
  const int ST = p.stages;
  Ctl& s = *reinterpret_cast<Ctl*>(smem + ST * kStage);
  uint8_t* plan_mem = smem + ST * kStage + (sizeof(Ctl) + 15) / 16 * 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &s.abort;

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      ptx::mbar_init(ptx::smem_u32(&s.full[i]), 3);
      ptx::mbar_init(ptx::smem_u32(&s.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(ptx::smem_u32(&s.tmem_full[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&s.tmem_empty[i]), 4);
      ptx::mbar_init(ptx::smem_u32(&s.tk_full[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&s.tk_empty[i]), 7);
    }
    s.abort = 0;
    ptx::fence_barrier_init();
    ptx::prefetch_tensormap(&map0);
    if (MODE == kMoe) {
      ptx::prefetch_tensormap(&map1);
      ptx::prefetch_tensormap(&map2);
    }
  }
  if (warp == 1) {
    ptx::tmem_alloc<1>(ptx::smem_u32(&s.tmem_base), kTmemCols);
    ptx::tmem_relinquish<1>();
  }

  // ------------------------------------------------------------ units
  few::Plan plan = {};
  RowUnits ru = {};
  const int S = MODE == kMoe ? p.r.num_tokens * p.r.K : 0;
  if constexpr (MODE == kMoe) {
    plan = few::plan_view(plan_mem, S, p.r.E, NB);
    pdl_wait();
    few::build_plan(plan, p.r, NB);
  } else {
    ru.row = reinterpret_cast<int*>(plan_mem);
    ru.e = reinterpret_cast<int16_t*>(ru.row + p.max_units);
    ru.n = reinterpret_cast<uint16_t*>(ru.e + p.max_units);
    if (p.offsets == nullptr) {
      const int units = (int)((p.m + NB - 1) / NB);
      for (int u = threadIdx.x; u < units; u += kThreads) {
        ru.e[u] = 0;
        ru.row[u] = u * NB;
        ru.n[u] = (uint16_t)min((long long)NB, (long long)p.m - u * NB);
      }
      if (threadIdx.x == 0) s.num_units = units;
    } else if (warp == 0) {
      int units = 0;
      for (int e0 = 0; e0 < p.E; e0 += 32) {
        const int e = e0 + lane;
        simt::GroupRange gr = {0, 0};
        if (e < p.E) gr = simt::group_range(p.offsets, p.plus_one, e, p.m);
        // never past the tensor or the table, whatever the offsets hold
        if (gr.start < 0 || gr.start >= p.m) gr.rows = 0;
        if (gr.rows > p.m - gr.start) gr.rows = p.m - gr.start;
        const int c = (int)((gr.rows + NB - 1) / NB);
        int inc = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += v;
        }
        for (int i = 0; i < c; ++i) {
          const int u = units + inc - c + i;
          if (u >= p.max_units) break;
          ru.e[u] = (int16_t)e;
          ru.row[u] = (int)gr.start + i * NB;
          ru.n[u] = (uint16_t)min((long long)NB, (long long)gr.rows - i * NB);
        }
        units += __shfl_sync(0xffffffffu, inc, 31);
      }
      if (lane == 0) s.num_units = min(units, p.max_units);
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const int U = MODE == kMoe ? *plan.num_units : s.num_units;
  const uint32_t tmem_base = s.tmem_base;
  // Tiles per unit and 64-deep blocks per tile of each phase.
  const int MT = MODE == kMoe ? (p.H + 127) / 128 : (p.N + 255) / 256;
  const int strips = (p.d + 255) / 256;
  Phase ph0, ph1;
  ph0.set((long long)U * MT, ((MODE == kMoe ? p.d : p.K) + BK - 1) / BK, p.max_chunks, p.min_blocks);
  if (MODE == kMoe) ph1.set((long long)U * strips, (p.H + BK - 1) / BK, p.max_chunks, p.min_blocks);
  else { ph1.KB = 1; ph1.total = 0; ph1.G = 0; }
  int* const c_tile = p.counters + 1;
  int* const c_done = c_tile + p.max_chunks;
  int* const c_strip = c_done + p.max_units;

  auto unit = [&](int u, int& e, int& row0, int& n) {
    if constexpr (MODE == kMoe) { e = plan.unit_e[u]; row0 = plan.unit_pos[u]; n = plan.unit_n[u]; }
    else { e = ru.e[u]; row0 = ru.row[u]; n = ru.n[u]; }
  };
  // Tile q of phase 1 is (strip, unit), strip-major; of phase 0 (unit, tile).
  auto decode = [&](int phase, long long q, int& u, int& mt) {
    if (phase) { mt = (int)(q / U); u = (int)(q % U); }
    else { u = (int)(q / MT); mt = (int)(q % MT); }
  };
  // A whole warp's wait: every lane leaves with the same answer, so that no lane meets a warp
  // barrier that another has skipped.
  auto warp_wait = [&](uint64_t& bar, uint32_t parity) {
    return __all_sync(0xffffffffu, ptx::wait_bounded(ptx::smem_u32(&bar), parity, abort_flag, kWaitNs)) != 0;
  };
  // The it-th ticket of this block (kLinear: its one chunk); false at the end.
  auto ticket = [&](int it, int& phase, int& c) -> bool {
    int t;
    if constexpr (MODE == kMoe) {
      const int slot = it & 1;
      if (!warp_wait(s.tk_full[slot], (it >> 1) & 1)) return false;
      t = *(volatile int*)&s.tk[slot];
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&s.tk_empty[slot]));
    } else {
      t = it == 0 ? (int)blockIdx.x : ph0.G;
    }
    phase = t >= ph0.G;
    c = phase ? t - ph0.G : t;
    return t < ph0.G + ph1.G;
  };

  if (MODE == kMoe && U == 0) {
    // Every slot is dropped: y is zero.
    T* y = static_cast<T*>(p.y);
    const int64_t n = (int64_t)p.r.num_tokens * p.d;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads)
      y[i] = from_f32<T>(0.f);
  } else if (warp == 0) {
    // ---------------------------------------------------------- weights
    if (lane == 0) {
      int stage = 0;
      uint32_t parity = 1;
      bool ok = true;
      for (int it = 0; ok; ++it) {
        int t;
        if constexpr (MODE == kMoe) {
          const int slot = it & 1;
          if (!ptx::wait_bounded(ptx::smem_u32(&s.tk_empty[slot]), ((it >> 1) & 1) ^ 1, abort_flag, kWaitNs)) break;
          t = atomicAdd(p.counters, 1);
          *(volatile int*)&s.tk[slot] = t;
          ptx::mbar_arrive(ptx::smem_u32(&s.tk_full[slot]));
        } else {
          t = it == 0 ? (int)blockIdx.x : ph0.G;
        }
        if (t >= ph0.G + ph1.G) break;
        const int phase = t >= ph0.G;
        const Phase& ph = phase ? ph1 : ph0;
        const int c = phase ? t - ph0.G : t;
        long long b = ph.begin(c);
        const long long end = ph.begin(c + 1);
        while (b < end && ok) {
          const long long q = b / ph.KB;
          const int kb0 = (int)(b - q * ph.KB);
          const int len = (int)min((long long)(ph.KB - kb0), end - b);
          int u, mt, e, row0, n;
          decode(phase, q, u, mt);
          unit(u, e, row0, n);
          const CUtensorMap* m0 = MODE == kMoe && phase ? &map2 : &map0;
          const CUtensorMap* m1 = MODE == kMoe && !phase ? &map1 : m0;
          const int r0 = MODE == kMoe && !phase ? mt * 128 : mt * 256;
          const int r1 = MODE == kMoe && !phase ? r0 : r0 + 128;
          for (int kb = kb0; kb < kb0 + len; ++kb) {
            if (!ptx::wait_bounded(ptx::smem_u32(&s.empty[stage]), parity, abort_flag, kWaitNs)) { ok = false; break; }
            const uint32_t bar = ptx::smem_u32(&s.full[stage]);
            const uint32_t dst = ptx::smem_u32(smem) + stage * kStage;
            ptx::mbar_arrive_expect_tx(bar, kWBytes);
            ptx::tma_load_3d(dst, m0, bar, kb * BK, r0, e);
            ptx::tma_load_3d(dst + kBoxBytes, m1, bar, kb * BK, r1, e);
            if (++stage == ST) { stage = 0; parity ^= 1; }
          }
          b += len;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA
    int stage = 0, seg = 0, phase, c;
    uint32_t parity = 0;
    bool ok = true;
    for (int it = 0; ok && ticket(it, phase, c); ++it) {
      const Phase& ph = phase ? ph1 : ph0;
      long long b = ph.begin(c);
      const long long end = ph.begin(c + 1);
      while (b < end && ok) {
        const long long q = b / ph.KB;
        const int kb0 = (int)(b - q * ph.KB);
        const int len = (int)min((long long)(ph.KB - kb0), end - b);
        int u, mt, e, row0, n;
        decode(phase, q, u, mt);
        unit(u, e, row0, n);
        const uint32_t idesc = ptx::make_idesc_f16(FMT, 0, 0, 128, (n + 15) / 16 * 16);
        const int buf = seg & 1;
        if (!warp_wait(s.tmem_empty[buf], ((seg >> 1) & 1) ^ 1)) { ok = false; break; }
        ptx::tc_fence_after();
        const uint32_t d0 = tmem_base + buf * 2 * NB;
        for (int i = 0; i < len; ++i) {
          if (!warp_wait(s.full[stage], parity)) { ok = false; break; }
          ptx::tc_fence_after();
          if (lane == 0) {
            const uint32_t sa = ptx::smem_u32(smem) + stage * kStage;
            const uint32_t sb = sa + kWBytes;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              const uint64_t bd = ptx::make_sw128_desc(sb + kk * 32, 16, 1024);
              ptx::mma_f16_ss<1>(d0, ptx::make_sw128_desc(sa + kk * 32, 16, 1024), bd, idesc, (i | kk) != 0);
              ptx::mma_f16_ss<1>(d0 + NB, ptx::make_sw128_desc(sa + kBoxBytes + kk * 32, 16, 1024), bd,
                                 idesc, (i | kk) != 0);
            }
            ptx::mma_commit<1>(ptx::smem_u32(&s.empty[stage]));
          }
          __syncwarp();
          if (++stage == ST) { stage = 0; parity ^= 1; }
        }
        if (!ok) break;
        if (lane == 0) ptx::mma_commit<1>(ptx::smem_u32(&s.tmem_full[buf]));
        __syncwarp();
        ++seg;
        b += len;
      }
    }
  } else if (warp < 4) {
    // ---------------------------------------------------------- activations
    const int l64 = (warp - 2) * 32 + lane;
    const int c16 = l64 & 7;  // 16-byte column of a 128-byte row
    int stage = 0, held = 0, held_stage = 0, phase, c;
    uint32_t parity = 1;
    bool ok = true;
    // Hands over the oldest `count` stages whose copies have landed.
    auto hand_over = [&](int count) {
      ptx::fence_proxy_async_smem();
      __syncwarp();
      for (int i = 0; i < count; ++i) {
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&s.full[held_stage]));
        if (++held_stage == ST) held_stage = 0;
      }
      held -= count;
    };
    auto drain = [&]() {
      ptx::cp_async_wait<0>();
      hand_over(held);
    };
    for (int it = 0; ok; ++it) {
      drain();  // nothing is held back while this warp waits for a ticket
      if (!ticket(it, phase, c)) break;
      const Phase& ph = phase ? ph1 : ph0;
      long long b = ph.begin(c);
      const long long end = ph.begin(c + 1);
      while (b < end && ok) {
        const long long q = b / ph.KB;
        const int kb0 = (int)(b - q * ph.KB);
        const int len = (int)min((long long)(ph.KB - kb0), end - b);
        int u, mt, e, row0, n;
        decode(phase, q, u, mt);
        unit(u, e, row0, n);
        const int cols = MODE == kLinear ? p.K : phase ? p.H : p.d;
        const T* rows[NB / 8];
#pragma unroll
        for (int i = 0; i < NB / 8; ++i) {
          const int r = (l64 >> 3) + 8 * i;
          int64_t src = row0 + (r < n ? r : 0);
          if (MODE == kMoe && !phase) src = plan.slot[src] / p.r.K;
          rows[i] = static_cast<const T*>(phase ? p.h : p.x) + src * cols + c16 * 8;
        }
        if (MODE == kMoe && phase) {
          // the unit's h: every one of its MT tiles finished
          if (!__all_sync(0xffffffffu, ptx::ld_acquire_gpu(c_done + u) >= MT)) {
            drain();
            const uint64_t t0 = ptx::globaltimer();
            while (ptx::ld_acquire_gpu(c_done + u) < MT) {
              if (*abort_flag || ptx::globaltimer() - t0 > kWaitNs) { *abort_flag = 1; ok = false; break; }
              __nanosleep(64);
            }
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
          }
        }
        for (int kb = kb0; kb < kb0 + len; ++kb) {
          if (!warp_wait(s.empty[stage], parity)) { ok = false; break; }
          const uint32_t dst = ptx::smem_u32(smem) + stage * kStage + kWBytes;
          const bool in = kb * BK + c16 * 8 < cols;  // cols is a multiple of 8
#pragma unroll
          for (int i = 0; i < NB / 8; ++i) {
            const int r = (l64 >> 3) + 8 * i;
            if (r < n)
              ptx::cp_async16(dst + r * 128 + ((c16 ^ (r & 7)) << 4),
                              rows[i] + (in ? kb * BK : -(c16 * 8)), in ? 16u : 0u);
          }
          ptx::cp_async_commit();
          if (++stage == ST) { stage = 0; parity ^= 1; }
          if (++held > kLag) {
            ptx::cp_async_wait<kLag>();
            hand_over(1);
          }
        }
        b += len;
      }
    }
    ptx::cp_async_wait<0>();
  } else {
    // ---------------------------------------------------------- epilogue
    const int row = (warp - 4) * 32 + lane;  // accumulator lane
    const bool lead = row == 0;
    int seg = 0, phase, c;
    bool ok = true;
    if (MODE == kLinear) pdl_wait();  // the counters are zeroed
    // The four warps meet at barriers, so each wait's outcome is agreed on by all of them.
    for (int it = 0; ok; ++it) {
      const bool more = ticket(it, phase, c);
      if (!ptx::named_barrier_all(1, 128, more)) break;
      const Phase& ph = phase ? ph1 : ph0;
      long long b = ph.begin(c);
      const long long end = ph.begin(c + 1);
      for (; b < end && ok; ++seg) {
        const long long q = b / ph.KB;
        const int kb0 = (int)(b - q * ph.KB);
        const int len = (int)min((long long)(ph.KB - kb0), end - b);
        b += len;
        int u, mt, e, row0, n;
        decode(phase, q, u, mt);
        unit(u, e, row0, n);
        const int buf = seg & 1;
        ok = ptx::named_barrier_all(1, 128, warp_wait(s.tmem_full[buf], (seg >> 1) & 1));
        if (!ok) break;
        ptx::tc_fence_after();
        const uint32_t tb = tmem_base + ((uint32_t)((warp - 4) * 32) << 16) + buf * 2 * NB;
        const bool whole = len == ph.KB && !phase;
        // Applies the tile's epilogue to row j of the unit (v0, v1: this thread's D0 and D1).
        float bias0 = 0.f, bias1 = 0.f;
        const int col0 = MODE == kMoe ? mt * 128 + row : mt * 256 + row, col1 = col0 + 128;
        if (MODE == kLinear && p.bias) {
          const T* bp = static_cast<const T*>(p.bias) + (int64_t)e * p.N;
          if (col0 < p.N) bias0 = to_f32(bp[col0]);
          if (col1 < p.N) bias1 = to_f32(bp[col1]);
        }
        auto finish = [&](int j, float v0, float v1) {
          if constexpr (MODE == kMoe) {
            if (col0 < p.H)
              static_cast<T*>(p.h)[(int64_t)(row0 + j) * p.H + col0] = from_f32<T>(v0 * sigmoid_f32(v0) * v1);
          } else {
            const int64_t at = (int64_t)(row0 + j) * p.N;
            auto put = [&](int col, float z) {
              if (col >= p.N) return;
              if (p.preact) static_cast<T*>(p.preact)[at + col] = from_f32<T>(z);
              float y = act_fwd_rt(p.act, z);
              if (p.residual) y += to_f32(static_cast<const T*>(p.residual)[at + col]);
              static_cast<T*>(p.y)[at + col] = from_f32<T>(y);
            };
            put(col0, v0 + bias0);
            put(col1, v1 + bias1);
          }
        };
        // Where the partial sums of a cut tile (or of any phase-1 tile) go: [row][256].
        float* dst;
        int64_t pitch = 256;
        if (phase) {
          if (kb0 == 0) { pitch = (int64_t)strips * 256; dst = p.o + row0 * pitch + mt * 256; }
          else dst = p.extra + (int64_t)c * NB * 256;
        } else {
          dst = p.part + ((int64_t)2 * c + (kb0 == 0)) * NB * 256;
        }
        for (int j0 = 0; j0 < n; j0 += 16) {
          uint32_t v0[16], v1[16];
          ptx::tmem_ld_32x32b_x16(tb + j0, v0);
          ptx::tmem_ld_32x32b_x16(tb + NB + j0, v1);
          ptx::tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (j0 + j < n) {
              const float a = __uint_as_float(v0[j]), g = __uint_as_float(v1[j]);
              if (whole) finish(j0 + j, a, g);
              else {
                dst[(j0 + j) * pitch + row] = a;
                dst[(j0 + j) * pitch + 128 + row] = g;
              }
            }
          }
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&s.tmem_empty[buf]));

        if (!phase) {
          if (!whole) {
            // Cut tile: the chunk that completes its block count adds the partials in order.
            const int f = ph.chunk_of(q * ph.KB), l = ph.chunk_of(q * ph.KB + ph.KB - 1);
            __threadfence();
            ptx::named_barrier(1, 128);
            if (lead) s.flag = ptx::atom_add_acq_rel_gpu(c_tile + f, len) + len == ph.KB;
            ptx::named_barrier(1, 128);
            if (!*(volatile int*)&s.flag) continue;
            __threadfence();
            for (int j = 0; j < n; ++j) {
              const float* src = p.part + ((int64_t)(2 * f + 1) * NB + j) * 256 + row;
              float a = __ldcg(src), g = __ldcg(src + 128);
              for (int cc = f + 1; cc <= l; ++cc) {
                src = p.part + ((int64_t)2 * cc * NB + j) * 256 + row;
                a += __ldcg(src);
                g += __ldcg(src + 128);
              }
              finish(j, a, g);
            }
          }
          if (MODE == kMoe) {
            __threadfence();
            ptx::named_barrier(1, 128);
            if (lead) ptx::atom_add_acq_rel_gpu(c_done + u, 1);
          }
        } else {
          // The strip's last finished chunk forms its 256 columns of y.
          __threadfence();
          ptx::named_barrier(1, 128);
          if (lead)
            s.flag = (long long)ptx::atom_add_acq_rel_gpu(c_strip + mt, len) + len == (long long)U * ph.KB;
          ptx::named_barrier(1, 128);
          if (!*(volatile int*)&s.flag) continue;
          __threadfence();
          const int64_t ld = (int64_t)strips * 256;
          for (int item = warp - 4; item < p.r.num_tokens * 4; item += 4) {
            const int t = item >> 2, at = (item & 3) * 64 + lane * 2;  // columns at, at + 1
            float2 acc = make_float2(0.f, 0.f);
#pragma unroll 4
            for (int k = 0; k < p.r.K; ++k) {
              const int sl = t * p.r.K + k;
              const int pos = plan.pos[sl];
              if (pos < 0) continue;
              const int uu = plan.unit_of[pos], j = pos - plan.unit_pos[uu];
              float2 v = __ldcg(reinterpret_cast<const float2*>(p.o + pos * ld + mt * 256 + at));
              const long long q0 = ((long long)mt * U + uu) * ph.KB;
              const int f = ph.chunk_of(q0), l = ph.chunk_of(q0 + ph.KB - 1);
              for (int cc = f + 1; cc <= l; ++cc) {
                const float2 w = __ldcg(reinterpret_cast<const float2*>(
                    p.extra + ((int64_t)cc * NB + j) * 256 + at));
                v.x += w.x;
                v.y += w.y;
              }
              acc.x = fmaf(plan.w[sl], v.x, acc.x);
              acc.y = fmaf(plan.w[sl], v.y, acc.y);
            }
            const int col = mt * 256 + at;
            T* yr = static_cast<T*>(p.y) + (int64_t)t * p.d;
            if (col < p.d) yr[col] = from_f32<T>(acc.x);
            if (col + 1 < p.d) yr[col + 1] = from_f32<T>(acc.y);
          }
        }
      }
    }
  }

  // ------------------------------------------------------------ teardown
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) raise_device_error(1);
    if (warp == 1) __nanosleep(100000);  // copies and MMAs still in flight land first
    __syncwarp();
  }
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<1>(tmem_base, kTmemCols);
  }
}

// Zeroes the counters of a kernel that follows with programmatic serialization.
__global__ void zero_counters_kernel(int* c, int n) {
  pdl_launch_dependents();
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) c[i] = 0;
}

}  // namespace fewtc
}  // namespace moe
