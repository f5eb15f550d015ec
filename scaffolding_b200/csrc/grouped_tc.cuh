// Grouped GEMM on tcgen05 for 16-bit operands: one persistent kernel over the
// tiles of every group, whatever the group sizes are.
//
//   D[n, i] = sum_k B[g][n, k] A[r(i), k]      n: 128 weight rows, i: rows of a group
//
// The weights fill the 128-row side of the MMA and the group's rows its N
// side, because N is free: a tile with 5 rows issues N = 16, one with 130 N =
// 144, so a ragged group pads to 16 rows and not to 128, and one kernel serves
// a decoding batch (a few rows per expert, bound by the weight stream) and a
// prompt (bound by the tensor core).  A group of more than BN rows is cut into
// even tiles.  The kernel reads the offsets itself: every CTA sums the groups'
// tile counts into shared memory and takes every gridDim.x-th tile, row tiles
// of one weight block next to each other so that the CTAs at work share it in
// L2.  The gated activation runs two weight blocks (gate and value rows)
// against the same rows into two accumulators, so both halves of an output
// meet in one thread.
//
// Rows are gathered by TMA: one tile::gather4 copy fetches four rows of A by
// index straight into the swizzled operand tile, and the gathered copy of A is
// never written.  Without indices the rows come in boxes.  A copy that runs
// past the group's end brings rows of the next group into columns that are
// not stored.
//
// CTA layout as the dense kernel (gemm_tc.cuh): warp 0 feeds the ring (all
// lanes issue the row copies), warp 1 owns TMEM and issues the MMAs, warps 2-9
// drain the accumulators, two of which let tile t + 1 start under t's stores.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "gemm_tc.cuh"
#include "grouped_args.cuh"

namespace sf {

template <int BN_, int STAGES_, int FMT_, bool GATE_>
struct GroupedCfg {
  static constexpr int BM = 128;
  static constexpr int BN = BN_;  // most rows of a group in one tile
  static constexpr int STAGES = STAGES_;
  static constexpr int FMT = FMT_;  // 0 f16, 1 bf16
  static constexpr bool GATE = GATE_;
  static constexpr int HALVES = GATE ? 2 : 1;
  static constexpr int BK = 64;
  static constexpr int BOX = BN <= 32 ? 16 : 32;  // rows per ungathered copy
  static constexpr int A_BYTES = BM * 128;        // one weight block
  static constexpr int STAGE_BYTES = HALVES * A_BYTES + BN * 128;
  static constexpr int ACC_COLS = HALVES * BN;
  static constexpr int TMEM_COLS = 2 * ACC_COLS <= 64 ? 64 : 2 * ACC_COLS <= 128 ? 128 : 512;
  static constexpr int CH = BN < 64 ? 16 : 32;  // accumulator columns per load
  static constexpr int EPI_THREADS = 256;
  static constexpr int THREADS = 64 + EPI_THREADS;
  static constexpr int RING_BYTES = STAGES * STAGE_BYTES + 1024;  // + alignment slack
  static_assert(BN % 32 == 0 && BN <= 256 && 2 * ACC_COLS <= 512, "TMEM columns");
};

// One tile: rows [row0, row0 + rows) of group g against weight rows n0 ...
struct GroupedTile {
  int g, n0, row0, rows;
};

// Maps tile numbers to tiles.  firsts[g] is the first row of group g (that of
// the next group ends it), starts[g] its first tile.
template <int BN>
struct GroupedTiles {
  int groups;
  const int* firsts;
  const int* starts;
  __device__ __forceinline__ bool get(int u, GroupedTile& t) const {
    if (u >= starts[groups]) return false;
    int lo = 0, hi = groups;  // starts[lo] <= u < starts[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (starts[mid] <= u) lo = mid; else hi = mid;
    }
    const int first = firsts[lo], rows = firsts[lo + 1] - first;
    const int cuts = (rows + BN - 1) / BN;
    const int per = ((rows + cuts - 1) / cuts + 15) / 16 * 16;
    const int r = u - starts[lo];
    const int nb = r / cuts, cut = r - nb * cuts;
    t.g = lo;
    t.n0 = nb * 128;
    t.row0 = first + cut * per;
    t.rows = min(per, rows - cut * per);
    return true;
  }
};

// Four rows of a 2-D tensor by index, 128 bytes of each, into consecutive
// 128-byte rows of a swizzled tile.  The map's box is one row high.
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* map, uint64_t* bar,
                                            int x, int r0, int r1, int r2, int r3) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(r0), "r"(r1), "r"(r2),
      "r"(r3)
      : "memory");
}

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x,
                                            int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}

// tmW: weights {K, rows per group, groups}, box {64, 128}.  tmX: A {K, a_rows},
// box {64, 1} for the gather, {64, BOX} otherwise.
template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, 1)
    grouped_tc_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                      const GroupedArgs p) {
  constexpr int BN = Cfg::BN, BK = Cfg::BK, STAGES = Cfg::STAGES, HALVES = Cfg::HALVES;
  constexpr int CH = Cfg::CH;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  int* firsts = reinterpret_cast<int*>(smem + STAGES * Cfg::STAGE_BYTES);  // [groups + 1]
  int* starts = firsts + p.groups + 1;                                     // [groups + 1]

  __shared__ __align__(8) uint64_t full_bar[STAGES];
  __shared__ __align__(8) uint64_t empty_bar[STAGES];
  __shared__ __align__(8) uint64_t tfull_bar[2];
  __shared__ __align__(8) uint64_t tempty_bar[2];
  __shared__ __align__(8) uint64_t drain_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int n_tiles = (p.N + 127) / 128;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], Cfg::EPI_THREADS);
    }
    mbar_init(&drain_bar, 1);
    abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  if (warp == 2) {
    // First row and tile of every group, 32 groups at a time.
    int at = 0, floor = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 32) {
      int lo, hi;
      group_bounds(p, g0, floor, lo, hi);
      const int tiles = (hi - lo + BN - 1) / BN * n_tiles;
      int end = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end += v;
      }
      if (g0 + lane < p.groups) {
        firsts[g0 + lane] = lo;
        starts[g0 + lane] = at + end - tiles;
      }
      at += __shfl_sync(0xffffffffu, end, 31);
    }
    if (lane == 0) {
      firsts[p.groups] = floor;
      starts[p.groups] = at;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  volatile int* abortp = &abort_flag;
  const GroupedTiles<BN> tiles{p.groups, firsts, starts};
  const int k_blocks = (p.K + BK - 1) / BK;

  if (warp == 0) {
    // ───────────── producer ─────────────
    int stage = 0;
    uint32_t phase = 0;
    int issued = 0;
    bool ok = true;
    GroupedTile t;
    for (int u = blockIdx.x; ok && tiles.get(u, t); u += gridDim.x) {
      // Lane l copies rows 8 l .. 8 l + 7 of the tile (two gathers), or box l.
      const int gathers = (t.rows + 3) / 4, boxes = (t.rows + Cfg::BOX - 1) / Cfg::BOX;
      int idx[8];
      uint32_t bytes = HALVES * Cfg::A_BYTES;
      if (p.rows) {
        bytes += gathers * 512;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int r = 8 * lane + j;
          int i = r < t.rows ? p.rows[t.row0 + r] : 0;
          // an index outside A reads zeros, as does any past the last row
          idx[j] = i < 0 || i >= p.a_rows ? static_cast<int>(p.a_rows) : i;
        }
      } else {
        bytes += boxes * Cfg::BOX * 128;
      }
      for (int kb = 0; kb < k_blocks; ++kb) {
        if (lane == 0) ok = mbar_wait(&empty_bar[stage], phase ^ 1u, p.err, kDevTimeoutProducer, abortp);
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        if (!ok) break;
        uint8_t* sw = smem + stage * Cfg::STAGE_BYTES;
        const uint32_t sx = smem_u32(sw + HALVES * Cfg::A_BYTES);
        if (lane == 0) {
          mbar_arrive_expect_tx(&full_bar[stage], bytes);
          tma_load_4d(sw, &tmW, &full_bar[stage], kb * BK, t.n0, t.g, 0);
          if constexpr (Cfg::GATE)
            tma_load_4d(sw + Cfg::A_BYTES, &tmW, &full_bar[stage], kb * BK, p.N + t.n0, t.g, 0);
        }
        __syncwarp();
        if (p.rows) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (2 * lane + h < gathers)
              tma_gather4(sx + (2 * lane + h) * 512, &tmX, &full_bar[stage], kb * BK, idx[4 * h],
                          idx[4 * h + 1], idx[4 * h + 2], idx[4 * h + 3]);
        } else if (lane < boxes) {
          tma_load_2d(sx + lane * Cfg::BOX * 128, &tmX, &full_bar[stage], kb * BK, t.row0 + lane * Cfg::BOX);
        }
        ++issued;
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (!ok && lane == 0) {
      // Abort: wait (bounded) for the copies still in flight.
      const int n = issued < STAGES ? issued : STAGES;
      int s = stage;
      uint32_t ph = phase;
      for (int j = 0; j < n; ++j) {
        if (--s < 0) {
          s = STAGES - 1;
          ph ^= 1u;
        }
        if (!mbar_wait_quiet(&full_bar[s], ph, 200000000ull)) atomicCAS(p.err, 0, kDevTimeoutDrain);
      }
    }
  } else if (warp == 1) {
    // ───────────── MMA issuer ─────────────
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      bool issued_any = false;
      GroupedTile t;
      for (int u = blockIdx.x; ok && tiles.get(u, t); u += gridDim.x) {
        const uint32_t idesc = make_idesc(Cfg::FMT, 128, (t.rows + 15) / 16 * 16, 0u, 0u);
        if (!mbar_wait(&tempty_bar[acc], acc_phase ^ 1u, p.err, kDevTimeoutMma, abortp)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + static_cast<uint32_t>(acc * Cfg::ACC_COLS);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase, p.err, kDevTimeoutMma, abortp)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t w_addr = smem_u32(smem + stage * Cfg::STAGE_BYTES);
          const uint32_t x_addr = w_addr + HALVES * Cfg::A_BYTES;
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const uint64_t xd = make_sw128_desc(x_addr + ks * 32, 16, 1024);
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
              umma_f16(d + h * BN, make_sw128_desc(w_addr + h * Cfg::A_BYTES + ks * 32, 16, 1024), xd,
                       idesc, (kb > 0 || ks > 0) ? 1u : 0u);
          }
          issued_any = true;
          umma_commit(&empty_bar[stage]);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit(&tfull_bar[acc]);
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      if (!ok && issued_any) {
        // Abort: no tcgen05.mma may still be writing TMEM when it is freed.
        umma_commit(&drain_bar);
        if (!mbar_wait_quiet(&drain_bar, 0, 200000000ull)) atomicCAS(p.err, 0, kDevTimeoutDrain);
      }
    }
  } else {
    // ───────────── epilogue (warps 2..9) ─────────────
    const int quad = warp & 3;
    const int half = (warp - 2) >> 2;
    int acc = 0;
    uint32_t acc_phase = 0;
    GroupedTile t;
    for (int u = blockIdx.x; tiles.get(u, t); u += gridDim.x) {
      const int n = t.n0 + quad * 32 + lane;  // this thread's weight row
      float bias0 = 0.0f, bias1 = 0.0f;
      if (p.bias && n < p.N) {
        bias0 = load_as_f32(p.bias, t.g * p.bias_stride + n, p.bias_dtype);
        if constexpr (Cfg::GATE) bias1 = load_as_f32(p.bias, t.g * p.bias_stride + p.N + n, p.bias_dtype);
      }
      if (!mbar_wait(&tfull_bar[acc], acc_phase, p.err, kDevTimeoutEpilogue, abortp)) break;
      tc_fence_after();
      const uint32_t tbase = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) +
                             static_cast<uint32_t>(acc * Cfg::ACC_COLS);
#pragma unroll 1
      for (int c = half * CH; c < t.rows; c += 2 * CH) {
        float v[CH], w[Cfg::GATE ? CH : 1];
        tmem_load_chunk<CH>(tbase + c, v);
        if constexpr (Cfg::GATE) tmem_load_chunk<CH>(tbase + BN + c, w);
        if (n < p.N) {
          const int64_t at = static_cast<int64_t>(t.row0 + c) * p.ldc + n;
#pragma unroll
          for (int i = 0; i < CH; ++i) {
            if (c + i >= t.rows) break;
            const float up = Cfg::GATE ? w[Cfg::GATE ? i : 0] + bias1 : 0.0f;
            store_from_f32(p.C, at + i * p.ldc, p.out_dtype,
                           grouped_act(v[i] + bias0, up, p.act, p.fast_act != 0));
          }
        }
      }
      tc_fence_before();
      mbar_arrive(&tempty_bar[acc]);
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

}  // namespace sf
