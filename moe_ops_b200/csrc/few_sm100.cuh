// Few rows against many weights on the sm_100a tensor cores: the expert part of the few-token
// MoE layer (kMoe) and linear / grouped_linear for a few rows (kLinear).
//
// With n rows (1 to 64) per weight matrix the product does 2 n flops per 2-byte weight, far
// below the ridge: the kernel is a stream over the weights and everything else hides behind it.
// The weights are the MMA's A operand (M = 128 weight rows) and the activations its B operand
// (N = n rounded up to 16).  A tcgen05.mma takes its thread about 80 cycles however small it is (the
// same measured for M = 64 and 128, N = 16 to 112), 51 bytes of weights per cycle when its 128
// rows are all in use, against the 26 that an SM's share of HBM delivers: M tiles should be full.
// (With the roles swapped, 256 weight rows as N, an instruction covers twice the weights but
// multiplies them with 128 rows, nearly all of them padding: the power that takes made 32 tokens
// at d = 7168 5 to 20 % slower.)
//
//   kMoe     phase 0: a tile is up to 128 columns of h: those gate rows and the same up rows of
//            one unit (an expert's rows of activations, at most NB), in one M tile (up to 64
//            columns: gate in its first half, up in its second) or two.  Its epilogue forms
//            h = silu(gate) * up in fp32 and rounds it once to 16 bits (as an MMA operand it
//            has to be).
//            phase 1: a tile is up to 256 rows of Wd times the unit's h.  Its fp32 results are
//            stored, never rounded; when all are there, y adds p * result over a token's slots.
//   kLinear  one phase: up to 256 weight rows times up to NB rows; bias, activation, residual.
//
// Work split.  The host picks each phase's tile height and the number of chunks that a tile's
// contraction is cut into (`parts`) from the sizes alone, so that the chunks fill whole waves of
// the SMs (results depend on neither routing nor timing).  Phase 0 is never cut: adding up
// parts of h before phase 1 costs a fence, an atomic and a second pass per cut, and while the
// weights saturate HBM each of these takes microseconds (6 and 5 us measured for a block's first
// ones).  Parts of the outputs are fp32 and cost little: all are added at the end, in order.
//
// kMoe (and a cut kLinear) hands its chunks out by an atomic ticket, phase 0's before phase 1's.
// A block waits only for phase-0 tiles, each of which a running block has taken and finishes
// without waiting for anyone, and at the very end for all chunks: the kernel makes progress
// whatever share of its blocks is resident.  The weight producer never waits for h, so the ring
// fills with Wd while the last h tiles are finished; phase 1 goes unit by unit in phase 0's
// order.  A finished h tile is published (barrier and releasing atomic) only when the next chunk's
// accumulator is ready or there is nothing else to do, and output chunks are counted once per
// block.
//
// Warp roles (256 threads, one block per SM):
//   warp 0      weights: TMA boxes 64 elements wide, 128-byte swizzle; also fetches the tickets.
//   warp 1      TMEM owner and MMA issuer.
//   warps 2-3   activations: 16-byte cp.async into the same swizzle (rows are gathered: any
//               token, any h row), which arrive on the stage's barrier when they land: these
//               warps run ahead by the whole ring, as the weights do (handing each stage over 3
//               later: 32 tokens, d = 7168, E = 256, H = 2048 2019 us, so 1950 us).
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
constexpr int kMaxStages = 12;
constexpr int kMaxBlocksPerStage = 4;
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
  struct Shape {
    int rows;        // weight rows of a tile = of its TMA box (a gate/up tile: of each of its two)
    int tiles;       // tiles of a unit
    int blocks;      // 64-deep blocks of a stage
    int m_tiles;     // M tiles of a tile: 1 or 2
    int second;      // bytes from a block's first box to its second box or M tile (0: none)
    int block_bytes; // weights of a block
  } shape[2];
  int stage_bytes, stages;
  int parts;         // chunks that a tile's contraction is cut into (kMoe: in phase 1)
  float* part;       // kMoe: [parts, S, d] results of phase 1; kLinear: [parts, m, N] (parts > 1)
  int* counters;     // zeroed before the launch (kLinear: parts > 1): ticket; finished chunks of
                     // the outputs; kMoe: done[units] finished h tiles of a unit
  int max_units;
};

constexpr int kTickets = 4;  // ticket ring

struct Ctl {
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint64_t tmem_full[4], tmem_empty[4];
  uint64_t tk_full[kTickets], tk_empty[kTickets];
  int tk[kTickets];
  uint32_t tmem_base;
  int abort;
  int flag;
  int num_units;
};

constexpr int kCtlBytes = (int)((sizeof(Ctl) + 15) / 16 * 16);
// Accumulators on their way out: two buffers of 8 rows of activations x 256 weight rows.
constexpr int kStagedBytes = 2 * 8 * 256 * 4;

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
  float y = act_fwd_rt<true>(p.act, z);
  if (p.residual) y += to_f32(static_cast<const T*>(p.residual)[at]);
  static_cast<T*>(p.y)[at] = from_f32<T>(y);
}

// A value that is the same in every lane, in a form that tells the compiler so.
template <typename V>
__device__ __forceinline__ V warp_uniform(V v) { return __shfl_sync(0xffffffffu, v, 0); }

template <int MODE, int FMT, typename T, int NB>
__global__ void __launch_bounds__(kThreads, 1)
few_kernel(const __grid_constant__ CUtensorMap map0, const __grid_constant__ CUtensorMap map1,
           const __grid_constant__ CUtensorMap map2, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // Accumulator sets: 2 M tiles x 2 accumulators of NB columns, or 4 of one M tile, which the
  // epilogue adds.  An MMA that adds to the one before it starts later (linear, 1 row, one M tile:
  // 26.6 us with one accumulator, 24.6 us with four).
  constexpr int kBufs = NB == 64 ? 2 : 4;
  constexpr uint32_t kTmemCols = kBufs * 4 * NB;
  const int ST = p.stages;
  const uint32_t stage_bytes = (uint32_t)p.stage_bytes;
  // After the ring, at least the 16 KB that an MMA of a low tile may read past the last stage.
  Ctl& s = *reinterpret_cast<Ctl*>(smem + ST * stage_bytes);
  float* const staged = reinterpret_cast<float*>(smem + ST * stage_bytes + kCtlBytes);
  uint8_t* plan_mem = smem + ST * stage_bytes + kCtlBytes + kStagedBytes;
  const int warp = warp_uniform((int)(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  volatile int* abort_flag = &s.abort;

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      ptx::mbar_init(ptx::smem_u32(&s.full[i]), 1 + 64);  // weights, and each lane of warps 2-3
      ptx::mbar_init(ptx::smem_u32(&s.empty[i]), 1);
    }
    for (int i = 0; i < 4; ++i) {
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
    // A cut product follows the kernel that zeroes its counters, which started after everything
    // before it had ended: only the counters have to wait.
    if (p.parts == 1) pdl_wait();
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
  // 64-deep blocks per tile and chunks of each phase.
  const int KB0 = ((MODE == kMoe ? p.d : p.K) + BK - 1) / BK, KB1 = (p.H + BK - 1) / BK;
  const int G0 = U * p.shape[0].tiles * (MODE == kLinear ? p.parts : 1);
  const int G1 = MODE == kMoe ? U * p.shape[1].tiles * p.parts : 0;
  int* const c_out = p.counters + 1;
  int* const c_done = p.counters + 2;
  // Without a cut, kLinear's blocks depend on nobody: tiles at a fixed stride, no counters.
  const bool tickets = MODE == kMoe || p.parts > 1;

  // Chunk t: unit u (expert e, first row row0, n rows), weight rows from w0, blocks
  // [kb0, kb0 + len) of the contraction.
  struct Chunk {
    int phase, u, w0, part, kb0, len, e, row0, n;
  };
  auto decode = [&](int t) {
    Chunk c;
    c.phase = MODE == kMoe && t >= G0;
    const int q = c.phase ? t - G0 : t;
    const auto& sh = p.shape[c.phase];
    const int parts = MODE == kMoe && !c.phase ? 1 : p.parts;
    const int tile = q / parts;
    c.part = q - tile * parts;
    c.u = tile / sh.tiles;
    c.w0 = (tile - c.u * sh.tiles) * sh.rows;
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
    int t;
    if (tickets) {
      const int slot = it % kTickets;
      if (!warp_wait(s.tk_full[slot], (it / kTickets) & 1)) return false;
      t = *(volatile int*)&s.tk[slot];
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&s.tk_empty[slot]));
    } else {
      t = blockIdx.x + it * gridDim.x;
    }
    if (t >= G0 + G1) return false;
    c = decode(t);
    return true;
  };

  if (warp == 0) {
    // ---------------------------------------------------------- weights
    if (lane == 0) {
      if (MODE == kLinear && tickets) pdl_wait();  // the counters are zeroed
      int stage = 0;
      uint32_t parity = 1;
      bool ok = true;
      for (int it = 0; ok; ++it) {
        int t;
        if (tickets) {
          const int slot = it % kTickets;
          // The next ticket is taken when the last chunk's loads have been issued, so a slower
          // SM takes fewer; its latency hides behind the ring.
          if (!ptx::wait_bounded(ptx::smem_u32(&s.tk_empty[slot]), ((it / kTickets) & 1) ^ 1, abort_flag, kWaitNs)) break;
          t = atomicAdd(p.counters, 1);
          *(volatile int*)&s.tk[slot] = t;
          ptx::mbar_arrive(ptx::smem_u32(&s.tk_full[slot]));
        } else {
          t = blockIdx.x + it * gridDim.x;
        }
        if (t >= G0 + G1) break;
        const Chunk c = decode(t);
        const bool gate_up = MODE == kMoe && !c.phase;
        const CUtensorMap* m0 = MODE == kMoe && c.phase ? &map2 : &map0;
        const auto& sh = p.shape[c.phase];
        for (int kb = c.kb0, left = c.len; left > 0; left -= sh.blocks) {
          if (!ptx::wait_bounded(ptx::smem_u32(&s.empty[stage]), parity, abort_flag, kWaitNs)) { ok = false; break; }
          const uint32_t bar = ptx::smem_u32(&s.full[stage]);
          uint32_t dst = ptx::smem_u32(smem) + stage * stage_bytes;
          const int nb = min(left, sh.blocks);
          ptx::mbar_arrive_expect_tx(bar, nb * (gate_up ? 2 : 1) * sh.rows * 128);
          for (int j = 0; j < nb; ++j, ++kb) {
            ptx::tma_load_3d(dst, m0, bar, kb * BK, c.w0, c.e);
            if (gate_up) ptx::tma_load_3d(dst + sh.second, &map1, bar, kb * BK, c.w0, c.e);
            dst += sh.block_bytes;
          }
          if (++stage == ST) { stage = 0; parity ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA
    // The whole warp runs this code and one lane issues.  tcgen05.mma takes its operands from
    // uniform registers: every value and branch here goes through warp_uniform(), which lets the
    // compiler keep them there.
    const uint32_t issue = lane == 0;
    const uint32_t ring = warp_uniform(ptx::smem_u32(smem)), tmem = warp_uniform(tmem_base);
    const int g0 = warp_uniform(G0), g = warp_uniform(G0 + G1);
    auto wait = [&](uint64_t& bar, uint32_t par) { return warp_uniform((int)warp_wait(bar, par)) != 0; };
    int stage = 0, buf = 0;
    uint32_t parity = 0, buf_parity = 1;
    bool ok = true;
    for (int it = 0; ok; ++it) {
      int t;
      if (tickets) {
        const int slot = it % kTickets;
        if (!wait(s.tk_full[slot], (it / kTickets) & 1)) break;
        t = warp_uniform(*(volatile int*)&s.tk[slot]);
        if (issue) ptx::mbar_arrive(ptx::smem_u32(&s.tk_empty[slot]));
        __syncwarp();
      } else {
        t = blockIdx.x + it * gridDim.x;
      }
      if (t >= g) break;
      const bool second = MODE == kMoe && t >= g0;
      const int parts = MODE == kMoe && !second ? 1 : p.parts;
      int kb0, len;
      part_range(second ? KB1 : KB0, parts, (second ? t - g0 : t) % parts, kb0, len);
      const int blocks = second ? p.shape[1].blocks : p.shape[0].blocks;
      const uint32_t block_bytes = second ? p.shape[1].block_bytes : p.shape[0].block_bytes;
      const int m_tiles = second ? p.shape[1].m_tiles : p.shape[0].m_tiles;
      const uint32_t next = (uint32_t)(second ? p.shape[1].second : p.shape[0].second) >> 4;
      const int u = ((second ? t - g0 : t) / parts) / (second ? p.shape[1].tiles : p.shape[0].tiles);
      const int n = warp_uniform(MODE == kMoe ? (int)plan.unit_n[u] : (int)ru.n[u]);
      const uint32_t idesc = ptx::make_idesc_f16(FMT, 0, 0, 128, (n + 15) / 16 * 16);
      if (!wait(s.tmem_empty[buf], buf_parity)) break;
      ptx::tc_fence_after();
      const uint32_t d = tmem + buf * 4 * NB;
      uint32_t more = 0;
      for (int left = len; left > 0; left -= blocks) {
        if (!wait(s.full[stage], parity)) { ok = false; break; }
        ptx::tc_fence_after();
        ptx::fence_proxy_async_smem();  // the copies of warps 2-3 before the MMAs' reads
        const uint32_t sw = ring + stage * stage_bytes;
        uint32_t dw = ptx::sw128_desc_lo(sw), da = ptx::sw128_desc_lo(sw + blocks * block_bytes);
        const int nb = min(left, blocks);
        for (int j = 0; j < nb; ++j) {
          if (m_tiles == 2) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              ptx::mma_f16_sw128(issue, d + (kk & 1) * NB, dw + 2 * kk, da + 2 * kk, idesc, kk > 1 ? 1u : more);
              ptx::mma_f16_sw128(issue, d + (2 + (kk & 1)) * NB, dw + next + 2 * kk, da + 2 * kk, idesc,
                                 kk > 1 ? 1u : more);
            }
          } else {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              ptx::mma_f16_sw128(issue, d + kk * NB, dw + 2 * kk, da + 2 * kk, idesc, more);
          }
          dw += block_bytes >> 4;
          da += NB * 8;
          more = 1;
        }
        if (issue) ptx::mma_commit<1>(ptx::smem_u32(&s.empty[stage]));
        __syncwarp();
        if (++stage == ST) { stage = 0; parity ^= 1; }
      }
      if (!ok) break;
      if (issue) ptx::mma_commit<1>(ptx::smem_u32(&s.tmem_full[buf]));
      __syncwarp();
      if (++buf == kBufs) { buf = 0; buf_parity ^= 1; }
    }
  } else if (warp < 4) {
    // ---------------------------------------------------------- activations
    const int l64 = (warp - 2) * 32 + lane;
    const int c16 = l64 & 7;  // 16-byte column of a 128-byte row
    int stage = 0;
    uint32_t parity = 1;
    bool ok = true;
    Chunk c;
    for (int it = 0; ok && ticket(it, c); ++it) {
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
        // the unit's h: every one of its tiles finished
        const int want = p.shape[0].tiles;
        if (!__all_sync(0xffffffffu, ptx::ld_acquire_gpu(c_done + c.u) >= want)) {
          const uint64_t t0 = ptx::globaltimer();
          while (ptx::ld_acquire_gpu(c_done + c.u) < want) {
            if (*abort_flag || ptx::globaltimer() - t0 > kWaitNs) { *abort_flag = 1; ok = false; break; }
            __nanosleep(32);
          }
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
      }
      const auto& sh = p.shape[c.phase];
      const uint32_t w_bytes = sh.blocks * sh.block_bytes;
      for (int kb = c.kb0, left = c.len; left > 0; left -= sh.blocks) {
        if (!warp_wait(s.empty[stage], parity)) { ok = false; break; }
        uint32_t dst = ptx::smem_u32(smem) + stage * stage_bytes + w_bytes;
        const int nb = min(left, sh.blocks);
        for (int j = 0; j < nb; ++j, ++kb, dst += NB * 128) {
          const bool in = kb * BK + c16 * 8 < cols;  // cols is a multiple of 8
#pragma unroll
          for (int i = 0; i < NB / 8; ++i) {
            const int r = (l64 >> 3) + 8 * i;
            if (r < c.n)
              ptx::cp_async16(dst + r * 128 + ((c16 ^ (r & 7)) << 4),
                              rows[i] + (in ? kb * BK : -(c16 * 8)), in ? 16u : 0u);
          }
        }
        ptx::cp_async_arrive(ptx::smem_u32(&s.full[stage]));
        if (++stage == ST) { stage = 0; parity ^= 1; }
      }
    }
    ptx::cp_async_wait_all();
  } else {
    // ---------------------------------------------------------- epilogue
    const int row = threadIdx.x - 128;  // accumulator lane
    const bool lead = row == 0;
    int buf = 0, half = 0;
    uint32_t parity = 0;
    Chunk c;
    int held_unit = -1;  // kMoe: the unit of an h tile that is stored but not published
    int outputs = 0;     // chunks of the outputs that this block has stored
    // The barrier orders every thread's stores before the lead's release, which is cumulative over
    // them; a fence of each thread before the barrier would not be part of that release.
    auto publish = [&]() {
      ptx::named_barrier(1, 128);
      if (lead) ptx::red_add_release_gpu(c_done + held_unit, 1);
      held_unit = -1;
    };
    // The four warps meet at barriers, so each wait's outcome is agreed on by all of them.
    for (int it = 0;; ++it) {
      if (MODE == kMoe && held_unit >= 0) {
        const bool ready = ptx::mbar_try_wait(ptx::smem_u32(&s.tk_full[it % kTickets]), (it / kTickets) & 1) &&
                           ptx::mbar_try_wait(ptx::smem_u32(&s.tmem_full[buf]), parity);
        if (!ptx::named_barrier_all(1, 128, ready)) publish();
      }
      const bool more = ticket(it, c);
      if (!ptx::named_barrier_all(1, 128, more)) break;
      if (!ptx::named_barrier_all(1, 128, warp_wait(s.tmem_full[buf], parity))) break;
      if (MODE == kMoe && held_unit >= 0) publish();
      ptx::tc_fence_after();
      const uint32_t tb = tmem_base + ((uint32_t)((warp - 4) * 32) << 16) + buf * 4 * NB;
      const auto& sh = p.shape[c.phase];
      const bool gate_up = MODE == kMoe && !c.phase;
      const bool pair = gate_up && sh.m_tiles == 1;  // gate in lanes 0-63, up in lanes 64-127
      const int limit = MODE == kLinear ? p.N : c.phase ? p.d : p.H;
      // This thread's columns of the output: one per M tile; of a pair, column row % 64 of every
      // second row of activations.
      const int at = pair ? row & 63 : row;
      const int col0 = at < sh.rows ? c.w0 + at : limit;
      const int col1 = !gate_up && 128 + at < sh.rows ? c.w0 + 128 + at : limit;
#pragma unroll 1
      for (int j0 = 0; j0 < c.n; j0 += 8, half ^= 1) {
        float* st = staged + half * 8 * 256;
        uint32_t v[4][8];
#pragma unroll
        for (int q = 0; q < 4; ++q) ptx::tmem_ld_32x32b_x8(tb + q * NB + j0, v[q]);
        ptx::tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float a = __uint_as_float(v[0][j]) + __uint_as_float(v[1][j]);
          const float b = __uint_as_float(v[2][j]) + __uint_as_float(v[3][j]);
          st[j * 256 + row] = sh.m_tiles == 2 ? a : a + b;
          st[j * 256 + 128 + row] = b;
        }
        const int m = min(8, c.n - j0);
        // A pair's halves meet here (this buffer is written again two turns later, after the next
        // turn's barrier); otherwise each thread reads back what it wrote.
        if (pair) ptx::named_barrier(1, 128);
        const int up = pair ? 64 : 128;
#pragma unroll 1
        for (int j = pair ? row >> 6 : 0; j < m; j += pair ? 2 : 1) {
          const float a = st[j * 256 + at], b = st[j * 256 + up + at];
          const int64_t r = c.row0 + j0 + j;
          if (gate_up) {
            if (col0 < limit) static_cast<T*>(p.h)[r * p.H + col0] = from_f32<T>(a * sigmoid_f32(a) * b);
          } else if (tickets) {
            float* dst = p.part + (c.part * (int64_t)(MODE == kMoe ? S : p.m) + r) * limit;
            if (col0 < limit) dst[col0] = a;
            if (col1 < limit) dst[col1] = b;
          } else {
#pragma unroll 1
            for (int i = 0; i < 2; ++i) linear_out<T>(p, c.e, r, i ? col1 : col0, i ? b : a);
          }
        }
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&s.tmem_empty[buf]));
      if (++buf == kBufs) { buf = 0; parity ^= 1; }
      if (gate_up) held_unit = c.u;
      else ++outputs;
    }
    // Abandoned work is not published (the wait that gave up has set the abort flag).
    if (MODE == kMoe && held_unit >= 0 && ptx::named_barrier_all(1, 128, *abort_flag == 0)) publish();
    if (tickets) {
      ptx::named_barrier(1, 128);
      if (lead && outputs > 0) ptx::red_add_release_gpu(c_out, outputs);
    }
  }

  // ------------------------------------------------------------ final stage
  // Every ticket is taken.  Four neighbouring elements of an output row at a time; when there are
  // many terms to add, 2 to 8 neighbouring lanes each add every split-th and then join.
  __syncthreads();
  if (!*abort_flag && tickets) {
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
    const int width = MODE == kMoe ? p.d : p.N;  // a multiple of 8
    const int out_rows = MODE == kMoe ? p.r.num_tokens : (int)p.m;
    const int terms = MODE == kMoe ? p.r.K * p.parts : p.parts;
    const int split = terms <= 4 ? 1 : terms <= 8 ? 2 : terms <= 16 ? 4 : 8;
    const int sub = lane & (split - 1);
    const int quads = width / 4;
    const long long items = (long long)quads * out_rows;
    const long long stride = (long long)gridDim.x * kThreads / split;
    // every lane of a warp makes the same number of turns (the join is a warp shuffle)
    const long long first = (long long)(blockIdx.x * kThreads + warp * 32) / split;
    for (long long i0 = first; *(volatile int*)&s.flag && i0 < items; i0 += stride) {
      const long long i = i0 + lane / split;
      const bool live = i < items;
      const int r = live ? (int)(i / quads) : 0, col = live ? (int)(i - (long long)r * quads) * 4 : 0;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int k = sub; k < terms; k += split) {
        float w = 1.f;
        int64_t at;
        if constexpr (MODE == kMoe) {
          const int slot = k / p.parts, sl = r * p.r.K + slot, pos = plan.pos[sl];
          if (pos < 0) continue;
          w = plan.w[sl];
          at = (int64_t)(k - slot * p.parts) * S + pos;
        } else {
          at = (int64_t)k * p.m + r;
        }
        const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part + at * width + col));
        acc.x = fmaf(w, v.x, acc.x);
        acc.y = fmaf(w, v.y, acc.y);
        acc.z = fmaf(w, v.z, acc.z);
        acc.w = fmaf(w, v.w, acc.w);
      }
      for (int o = 1; o < split; o <<= 1) {
        acc.x += __shfl_xor_sync(0xffffffffu, acc.x, o);
        acc.y += __shfl_xor_sync(0xffffffffu, acc.y, o);
        acc.z += __shfl_xor_sync(0xffffffffu, acc.z, o);
        acc.w += __shfl_xor_sync(0xffffffffu, acc.w, o);
      }
      if (!live || sub != 0) continue;
      int e = 0;
      if constexpr (MODE == kLinear) {  // the row's unit: the last that starts at or before it
        int lo = 0, hi = U - 1;
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (ru.row[mid] <= r) lo = mid; else hi = mid - 1;
        }
        if (U == 0 || r < ru.row[lo] || r >= ru.row[lo] + ru.n[lo]) continue;  // in no group
        e = ru.e[lo];
      }
#pragma unroll 1
      for (int q = 0; q < 4; ++q) {
        const float v = q == 0 ? acc.x : q == 1 ? acc.y : q == 2 ? acc.z : acc.w;
        if constexpr (MODE == kMoe) static_cast<T*>(p.y)[(int64_t)r * width + col + q] = from_f32<T>(v);
        else linear_out<T>(p, e, r, col + q, v);
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
