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
// Work split.  Every tile's contraction is cut into `parts` chunks (fixed by the host from the
// sizes, so results do not depend on routing or timing), small enough for about
// kChunksPerSm chunks per SM: SMs do not all stream equally fast, and with one equal share each
// the slowest held the others up (one token, d = 4096, H = 11008: 15 us of 115).  An atomic
// ticket hands the chunks out in order, phase 0's before phase 1's.  A block waits only for
// chunks with smaller tickets, each of which a running block has taken and finishes without
// waiting for a later one: the kernel makes progress whatever share of its blocks is resident.
// Partial sums are fp32 and added in chunk order: those of h by the block that finishes a tile
// last, those of the outputs in a final stage that all blocks share once the tickets are used
// up.
//
// The weight producer never waits for h, so the ring (about 200 KB per SM) fills with Wd while
// the last h tiles are finished.  Phase 1 goes unit by unit in phase 0's order, so that the h
// it needs first was finished first: the stream does not stop between the phases.
//
// Warp roles (256 threads, one block per SM):
//   warp 0      weights: TMA boxes of 64 x 128, 128-byte swizzle; also fetches the tickets.
//   warp 1      TMEM owner and MMA issuer.
//   warps 2-3   activations: 16-byte cp.async into the same swizzle (rows are gathered: any
//               token, any h row), handed over kLag stages later.
//   warps 4-7   epilogue, one accumulator lane (weight row) per thread.
//
// While the weights saturate HBM a fence or an atomic takes microseconds (measured: 6 us and 5 us
// for the first ones of a block), as long as a chunk's loads.  So they stay off the chunk's path:
// there are several accumulator pairs, a finished h tile is published only when the next
// chunk's accumulator is ready (its stores have long landed, the fence is short) or when there is
// nothing else to do, and finished output chunks are counted once per block.
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
  void* y;           // [T, d]; kLinear: [m, N]
  int parts0, parts1;  // chunks per tile of each phase
  float* part0;      // [parts0, rows, MT * 256] partials of phase 0 (parts0 > 1); rows: S or m
  float* part1;      // [parts1, S, strips * 256] results of phase 1
  int rows;          // S (kMoe) or m
  int* counters;     // zeroed before the launch: ticket; finished chunks of the outputs; kMoe:
                     // done[max_units] finished h tiles of a unit, tile[max_units * MT] finished
                     // chunks of an h tile (parts0 > 1)
  int max_units;
  int stages;
};

constexpr int kTickets = 4;  // ticket ring

// Accumulator pairs of a unit size: 256 TMEM columns, 512 for NB = 64.
__host__ __device__ constexpr int acc_bufs(int nb) { return nb == 16 ? 8 : 4; }

struct Ctl {
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint64_t tmem_full[8], tmem_empty[8];
  uint64_t tk_full[kTickets], tk_empty[kTickets];
  int tk[kTickets];
  uint32_t tmem_base;
  int abort;
  int flag;
  int num_units;
};

constexpr int kCtlBytes = (int)((sizeof(Ctl) + 15) / 16 * 16);
constexpr int kStagedBytes = 8 * 256 * 4;  // accumulators of 8 rows on their way out

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

// Contraction blocks [first, first + len) of chunk `part` of a tile of KB blocks.
__device__ __forceinline__ void part_range(int KB, int parts, int part, int& first, int& len) {
  const int L = (KB + parts - 1) / parts;
  first = part * L;
  len = min(L, KB - first);
}

// kLinear's epilogue on one element: z = the products' sum, of group e.
template <typename T>
__device__ __forceinline__ void linear_out(const Params& p, int e, int64_t row, int col, float z) {
  if (col >= p.N) return;
  if (p.bias) z += to_f32(static_cast<const T*>(p.bias)[(int64_t)e * p.N + col]);
  const int64_t at = row * p.N + col;
  if (p.preact) static_cast<T*>(p.preact)[at] = from_f32<T>(z);
  float y = act_fwd_rt(p.act, z);
  if (p.residual) y += to_f32(static_cast<const T*>(p.residual)[at]);
  static_cast<T*>(p.y)[at] = from_f32<T>(y);
}

template <int MODE, int FMT, typename T, int NB>
__global__ void __launch_bounds__(kThreads, 1)
few_kernel(const __grid_constant__ CUtensorMap map0, const __grid_constant__ CUtensorMap map1,
           const __grid_constant__ CUtensorMap map2, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr uint32_t kStage = kWBytes + NB * 128;
  constexpr int kBufs = acc_bufs(NB);
  constexpr uint32_t kTmemCols = kBufs * 2 * NB;
  const int ST = p.stages;
  Ctl& s = *reinterpret_cast<Ctl*>(smem + ST * kStage);
  float* const staged = reinterpret_cast<float*>(smem + ST * kStage + kCtlBytes);  // [8][256]
  uint8_t* plan_mem = smem + ST * kStage + kCtlBytes + kStagedBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &s.abort;

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      ptx::mbar_init(ptx::smem_u32(&s.full[i]), 3);
      ptx::mbar_init(ptx::smem_u32(&s.empty[i]), 1);
    }
    for (int i = 0; i < kBufs; ++i) {
      ptx::mbar_init(ptx::smem_u32(&s.tmem_full[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&s.tmem_empty[i]), 4);
    }
    for (int i = 0; i < kTickets; ++i) {
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
  // Tiles per unit, 64-deep blocks per tile and chunks of each phase.
  const int MT = MODE == kMoe ? (p.H + 127) / 128 : (p.N + 255) / 256;
  const int strips = MODE == kMoe ? (p.d + 255) / 256 : 0;
  const int KB0 = ((MODE == kMoe ? p.d : p.K) + BK - 1) / BK, KB1 = (p.H + BK - 1) / BK;
  const int G0 = U * MT * p.parts0, G1 = MODE == kMoe ? U * strips * p.parts1 : 0;
  int* const c_out = p.counters + 1;
  int* const c_done = p.counters + 2;
  int* const c_tile = c_done + p.max_units;

  // Chunk t: unit u (expert e, first row row0, n rows), tile mt, blocks [kb0, kb0 + len).
  struct Chunk {
    int phase, u, mt, part, kb0, len, e, row0, n;
  };
  auto decode = [&](int t) {
    Chunk c;
    c.phase = MODE == kMoe && t >= G0;
    const int i = c.phase ? t - G0 : t;
    const int parts = c.phase ? p.parts1 : p.parts0, tiles = c.phase ? strips : MT;
    const int q = i / parts;
    c.part = i - q * parts;
    c.u = q / tiles;
    c.mt = q - c.u * tiles;
    part_range(c.phase ? KB1 : KB0, parts, c.part, c.kb0, c.len);
    if constexpr (MODE == kMoe) {
      c.e = plan.unit_e[c.u]; c.row0 = plan.unit_pos[c.u]; c.n = plan.unit_n[c.u];
    } else {
      c.e = ru.e[c.u]; c.row0 = ru.row[c.u]; c.n = ru.n[c.u];
    }
    return c;
  };
  // A whole warp's wait: every lane leaves with the same answer, so that no lane meets a warp
  // barrier that another has skipped.
  auto warp_wait = [&](uint64_t& bar, uint32_t parity) {
    return __all_sync(0xffffffffu, ptx::wait_bounded(ptx::smem_u32(&bar), parity, abort_flag, kWaitNs)) != 0;
  };
  // This block's it-th ticket, for the warps that follow the producer; false at the end.
  auto ticket = [&](int it, Chunk& c) -> bool {
    const int slot = it % kTickets;
    if (!warp_wait(s.tk_full[slot], (it / kTickets) & 1)) return false;
    const int t = *(volatile int*)&s.tk[slot];
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&s.tk_empty[slot]));
    if (t >= G0 + G1) return false;
    c = decode(t);
    return true;
  };

  if (warp == 0) {
    // ---------------------------------------------------------- weights
    if (lane == 0) {
      if (MODE == kLinear) pdl_wait();  // the counters are zeroed
      int stage = 0;
      uint32_t parity = 1;
      bool ok = true;
      for (int it = 0; ok; ++it) {
        const int slot = it % kTickets;
        // The next ticket is taken when the last chunk's loads have been issued, so a slower
        // SM takes fewer; its latency hides behind the ring.
        if (!ptx::wait_bounded(ptx::smem_u32(&s.tk_empty[slot]), ((it / kTickets) & 1) ^ 1, abort_flag, kWaitNs)) break;
        const int t = atomicAdd(p.counters, 1);
        *(volatile int*)&s.tk[slot] = t;
        ptx::mbar_arrive(ptx::smem_u32(&s.tk_full[slot]));
        if (t >= G0 + G1) break;
        const Chunk c = decode(t);
        const bool gate_up = MODE == kMoe && !c.phase;
        const CUtensorMap* m0 = MODE == kMoe && c.phase ? &map2 : &map0;
        const CUtensorMap* m1 = gate_up ? &map1 : m0;
        const int r0 = gate_up ? c.mt * 128 : c.mt * 256;
        const int r1 = gate_up ? r0 : r0 + 128;
        for (int kb = c.kb0; kb < c.kb0 + c.len; ++kb) {
          if (!ptx::wait_bounded(ptx::smem_u32(&s.empty[stage]), parity, abort_flag, kWaitNs)) { ok = false; break; }
          const uint32_t bar = ptx::smem_u32(&s.full[stage]);
          const uint32_t dst = ptx::smem_u32(smem) + stage * kStage;
          ptx::mbar_arrive_expect_tx(bar, kWBytes);
          ptx::tma_load_3d(dst, m0, bar, kb * BK, r0, c.e);
          ptx::tma_load_3d(dst + kBoxBytes, m1, bar, kb * BK, r1, c.e);
          if (++stage == ST) { stage = 0; parity ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA
    int stage = 0;
    uint32_t parity = 0;
    bool ok = true;
    Chunk c;
    for (int it = 0; ok && ticket(it, c); ++it) {
      const uint32_t idesc = ptx::make_idesc_f16(FMT, 0, 0, 128, (c.n + 15) / 16 * 16);
      const int buf = it % kBufs;
      if (!warp_wait(s.tmem_empty[buf], ((it / kBufs) & 1) ^ 1)) break;
      ptx::tc_fence_after();
      const uint32_t d0 = tmem_base + buf * 2 * NB;
      for (int i = 0; i < c.len; ++i) {
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
    }
  } else if (warp < 4) {
    // ---------------------------------------------------------- activations
    const int l64 = (warp - 2) * 32 + lane;
    const int c16 = l64 & 7;  // 16-byte column of a 128-byte row
    int stage = 0, held = 0, held_stage = 0;
    uint32_t parity = 1;
    bool ok = true;
    Chunk c;
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
      if (held == 0) return;
      ptx::cp_async_wait<0>();
      hand_over(held);
    };
    for (int it = 0; ok; ++it) {
      // Nothing is held back while this warp waits for a ticket (or, below, for h).
      if (!__all_sync(0xffffffffu, ptx::mbar_try_wait(ptx::smem_u32(&s.tk_full[it % kTickets]),
                                                      (it / kTickets) & 1)))
        drain();
      if (!ticket(it, c)) break;
      const int cols = MODE == kLinear ? p.K : c.phase ? p.H : p.d;
      const T* rows[NB / 8];
#pragma unroll
      for (int i = 0; i < NB / 8; ++i) {
        const int r = (l64 >> 3) + 8 * i;
        int64_t src = c.row0 + (r < c.n ? r : 0);
        if (MODE == kMoe && !c.phase) src = plan.slot[src] / p.r.K;
        rows[i] = static_cast<const T*>(MODE == kMoe && c.phase ? p.h : p.x) + src * cols + c16 * 8;
      }
      if (MODE == kMoe && c.phase) {
        // the unit's h: every one of its MT tiles finished
        if (!__all_sync(0xffffffffu, ptx::ld_acquire_gpu(c_done + c.u) >= MT)) {
          drain();
          const uint64_t t0 = ptx::globaltimer();
          while (ptx::ld_acquire_gpu(c_done + c.u) < MT) {
            if (*abort_flag || ptx::globaltimer() - t0 > kWaitNs) { *abort_flag = 1; ok = false; break; }
            __nanosleep(32);
          }
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
      }
      for (int kb = c.kb0; kb < c.kb0 + c.len; ++kb) {
        if (!warp_wait(s.empty[stage], parity)) { ok = false; break; }
        const uint32_t dst = ptx::smem_u32(smem) + stage * kStage + kWBytes;
        const bool in = kb * BK + c16 * 8 < cols;  // cols is a multiple of 8
#pragma unroll
        for (int i = 0; i < NB / 8; ++i) {
          const int r = (l64 >> 3) + 8 * i;
          if (r < c.n)
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
    }
    drain();
  } else {
    // ---------------------------------------------------------- epilogue
    const int row = (warp - 4) * 32 + lane;  // accumulator lane
    const bool lead = row == 0;
    const int64_t ld0 = (int64_t)MT * 256, ld1 = (int64_t)strips * 256;
    Chunk c, held = {};
    bool pending = false;  // `held` is a phase-0 chunk of kMoe that is stored but not published
    int outputs = 0;       // chunks of the outputs that this block has stored
    // h of column `row` of a tile: D0 is its gate, D1 its up.
    auto store_h = [&](const Chunk& k, int j, float gate, float up) {
      const int col = k.mt * 128 + row;
      if (col < p.H)
        static_cast<T*>(p.h)[(int64_t)(k.row0 + j) * p.H + col] = from_f32<T>(gate * sigmoid_f32(gate) * up);
    };
    // Counts `held`; of a cut tile, the block that finishes it last adds the parts in order.
    auto publish = [&]() {
      pending = false;
      ptx::fence_acq_rel_gpu();
      ptx::named_barrier(1, 128);
      if (p.parts0 > 1) {
        if (lead) s.flag = ptx::atom_add_gpu(c_tile + held.u * MT + held.mt, 1) + 1 == p.parts0;
        ptx::named_barrier(1, 128);
        if (!*(volatile int*)&s.flag) return;
        ptx::fence_acq_rel_gpu();
        const float* src = p.part0 + (int64_t)held.row0 * ld0 + held.mt * 256 + row;
        const int64_t step = (int64_t)p.rows * ld0;
#pragma unroll 1
        for (int j = 0; j < held.n; ++j) {
          float a = 0.f, g = 0.f;
#pragma unroll 8
          for (int q = 0; q < p.parts0; ++q) {
            a += __ldcg(src + q * step + j * ld0);
            g += __ldcg(src + q * step + j * ld0 + 128);
          }
          store_h(held, j, a, g);
        }
        ptx::fence_acq_rel_gpu();
        ptx::named_barrier(1, 128);
      }
      if (lead) ptx::atom_add_gpu(c_done + held.u, 1);
    };
    // The four warps meet at barriers, so each wait's outcome is agreed on by all of them.
    for (int it = 0;; ++it) {
      const int buf = it % kBufs;
      const uint32_t parity = (it / kBufs) & 1;
      if (pending) {
        const bool ready = ptx::mbar_try_wait(ptx::smem_u32(&s.tk_full[it % kTickets]), (it / kTickets) & 1) &&
                           ptx::mbar_try_wait(ptx::smem_u32(&s.tmem_full[buf]), parity);
        if (!ptx::named_barrier_all(1, 128, ready)) publish();
      }
      const bool more = ticket(it, c);
      if (!ptx::named_barrier_all(1, 128, more)) break;
      if (!ptx::named_barrier_all(1, 128, warp_wait(s.tmem_full[buf], parity))) break;
      if (pending) publish();
      ptx::tc_fence_after();
      const uint32_t tb = tmem_base + ((uint32_t)((warp - 4) * 32) << 16) + buf * 2 * NB;
      const bool whole = !c.phase && p.parts0 == 1;
      // Partial sums: this thread's two columns of the tile, row by row.
      const int64_t ld = c.phase ? ld1 : ld0;
      float* dst = (c.phase ? p.part1 : p.part0) + ((int64_t)c.part * p.rows + c.row0) * ld + c.mt * 256 + row;
#pragma unroll 1
      for (int j0 = 0; j0 < c.n; j0 += 8) {
        uint32_t v0[8], v1[8];
        ptx::tmem_ld_32x32b_x8(tb + j0, v0);
        ptx::tmem_ld_32x32b_x8(tb + NB + j0, v1);
        ptx::tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          staged[j * 256 + row] = __uint_as_float(v0[j]);
          staged[j * 256 + 128 + row] = __uint_as_float(v1[j]);
        }
        // each thread reads back what it wrote
        const int m = min(8, c.n - j0);
#pragma unroll 1
        for (int j = 0; j < m; ++j) {
          const float a = staged[j * 256 + row], g = staged[j * 256 + 128 + row];
          if (!whole) {
            dst[(j0 + j) * ld] = a;
            dst[(j0 + j) * ld + 128] = g;
          } else if constexpr (MODE == kMoe) {
            store_h(c, j0 + j, a, g);
          } else {
#pragma unroll 1
            for (int i = 0; i < 2; ++i)
              linear_out<T>(p, c.e, c.row0 + j0 + j, c.mt * 256 + i * 128 + row, i ? g : a);
          }
        }
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&s.tmem_empty[buf]));
      if (MODE == kMoe && !c.phase) {
        held = c;
        pending = true;
      } else {
        ++outputs;
      }
    }
    // Abandoned work is not published (the wait that gave up has set the abort flag).
    if (pending && !ptx::named_barrier_all(1, 128, *abort_flag != 0)) publish();
    if (MODE == kMoe || p.parts0 > 1) {
      ptx::fence_acq_rel_gpu();
      ptx::named_barrier(1, 128);
      if (lead && outputs > 0) ptx::atom_add_gpu(c_out, outputs);
    }
  }

  // ------------------------------------------------------------ final stage
  // Every ticket is taken.  64 columns of one output row at a time: 4 threads per column each
  // add a quarter of the terms, then the quarters are added in order.
  __syncthreads();
  if (!*abort_flag && (MODE == kMoe || p.parts0 > 1)) {
    float* red = reinterpret_cast<float*>(smem);  // the ring is idle
    if (threadIdx.x == 0) {
      const int want = MODE == kMoe ? G1 : G0;
      const uint64_t t0 = ptx::globaltimer();
      s.flag = 1;
      while (ptx::ld_acquire_gpu(c_out) < want) {
        if (ptx::globaltimer() - t0 > kWaitNs) { s.flag = 0; *abort_flag = 1; break; }
        __nanosleep(32);
      }
    }
    __syncthreads();
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    const int width = MODE == kMoe ? p.d : p.N;
    const int groups = (width + 63) / 64;
    const int out_rows = MODE == kMoe ? p.r.num_tokens : p.rows;
    const int64_t ld = (int64_t)(MODE == kMoe ? strips : MT) * 256;
    const int parts = MODE == kMoe ? p.parts1 : p.parts0;
    const int64_t step = (int64_t)p.rows * ld;
    const int items = *(volatile int*)&s.flag ? groups * out_rows : 0;
    for (int i = blockIdx.x; i < items; i += gridDim.x) {
      const int r = i / groups, g = i - r * groups, col = g * 64 + tx;
      int unit = 0;
      if constexpr (MODE == kLinear) {  // the row's unit: the last that starts at or before it
        int hi = U - 1;
        while (unit < hi) {
          const int mid = (unit + hi + 1) >> 1;
          if (ru.row[mid] <= r) unit = mid; else hi = mid - 1;
        }
        if (U == 0 || r < ru.row[unit] || r >= ru.row[unit] + ru.n[unit]) continue;  // in no group
      }
      float acc = 0.f;
      if constexpr (MODE == kMoe) {
        const int terms = p.r.K * parts;
#pragma unroll 4
        for (int j = ty; j < terms; j += 4) {
          const int k = j / parts, sl = r * p.r.K + k, pos = plan.pos[sl];
          if (pos >= 0)
            acc = fmaf(plan.w[sl], __ldcg(p.part1 + (int64_t)(j - k * parts) * step + pos * ld + col), acc);
        }
      } else {
#pragma unroll 4
        for (int j = ty; j < parts; j += 4) acc += __ldcg(p.part0 + j * step + r * ld + col);
      }
      red[threadIdx.x] = acc;
      __syncthreads();
      if (ty == 0 && col < width) {
        const float v = ((red[tx] + red[64 + tx]) + red[128 + tx]) + red[192 + tx];
        if constexpr (MODE == kMoe) {
          static_cast<T*>(p.y)[(int64_t)r * p.d + col] = from_f32<T>(v);
        } else {
          linear_out<T>(p, ru.e[unit], r, col, v);
        }
      }
      __syncthreads();
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
