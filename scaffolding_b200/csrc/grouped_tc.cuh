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
// Gathered rows are copied by index by one to eight more warps (10 on), 16
// bytes per cp.async, into the swizzled operand tile; the copies arrive on the
// stage's barrier themselves, and the MMA thread orders them before its reads.
// (TMA's tile::gather4 does the same in one instruction per four rows, but
// takes about 70 cycles for it: 4324 us where this takes 1198 us, 35552 rows of
// 1920 against 8 experts of 7680.)  Without indices the rows come in TMA
// boxes of 128 rows (16 in small tiles; boxes of 32 cost 16 % at that size).
// A box that runs past the group's end brings rows of the next group into
// columns that are not stored.
//
// CTA layout as the dense kernel (gemm_tc.cuh): warp 0 feeds the ring, warp 1
// owns TMEM and issues the MMAs, warps 2-9 drain the accumulators, two of which
// let tile t + 1 start under t's stores.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "gemm_tc.cuh"
#include "grouped_args.cuh"

namespace sf {

template <int BN_, int STAGES_, int FMT_, bool GATE_, bool SPLIT_ = false>
struct GroupedCfg {
  static constexpr int BM = 128;
  static constexpr int BN = BN_;  // most rows of a group in one tile
  static constexpr int STAGES = STAGES_;
  static constexpr int FMT = FMT_;  // 0 f16, 1 bf16
  static constexpr bool GATE = GATE_;
  static constexpr bool SPLIT = SPLIT_;  // a cluster of CTAs shares a tile's k-blocks
  static constexpr int HALVES = GATE ? 2 : 1;
  static constexpr int BK = 64;
  static constexpr int BOX = BN <= 32 ? 16 : BN <= 64 ? 32 : 128;  // rows per ungathered copy
  static constexpr int A_BYTES = BM * 128;        // one weight block
  static constexpr int STAGE_BYTES = HALVES * A_BYTES + BN * 128;
  static constexpr int ACC_COLS = HALVES * BN;
  static constexpr int TMEM_COLS = 2 * ACC_COLS <= 64 ? 64 : 2 * ACC_COLS <= 128 ? 128 : 2 * ACC_COLS <= 256 ? 256 : 512;
  static constexpr int CH = BN <= 32 ? 16 : 32;  // accumulator columns per load
  static constexpr int EPI_THREADS = 256;
  static constexpr int THREADS = 64 + EPI_THREADS;  // without the gather warps
  // One 16-byte copy per row and lane keeps one warp busy up to 32 rows; more
  // arrivals per stage than the rows need cost time (1 against 8 warps at 2 rows
  // per group: 46.8 / 50.4 us).
  static constexpr int GATHER_WARPS = BN <= 32 ? 1 : BN <= 64 ? 2 : 8;
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

// 16 bytes global -> shared, of which the first `bytes` are read and the rest
// are zeros.
__device__ __forceinline__ void gather_copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}

// The float at shared::cta address `addr` of CTA `rank` of the cluster.
__device__ __forceinline__ float load_cluster_f32(uint32_t addr, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(addr, rank)) : "memory");
  return v;
}

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x,
                                            int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}

// The activation of CH values, chosen once.
template <int CH>
__device__ __forceinline__ void activate(float (&v)[CH], int act, bool fast) {
  if (act == kActNone) return;
  if (!fast) {
#pragma unroll
    for (int i = 0; i < CH; ++i) v[i] = act_apply(v[i], act);
  } else if (act == kActSilu) {
#pragma unroll
    for (int i = 0; i < CH; ++i) v[i] = act_apply_fast(v[i], kActSilu);
  } else {
#pragma unroll
    for (int i = 0; i < CH; ++i) v[i] = act_apply_fast(v[i], kActGeluTanh);
  }
}

// CH values of one output column: rows at, at + ld, ..., the first `left` of
// them.  Neighbouring lanes hold neighbouring columns.
template <int CH>
__device__ __forceinline__ void store_column(void* C, int64_t at, int64_t ld, int dtype, const float (&v)[CH],
                                             int left) {
  if (dtype == kF32) {
    float* p = static_cast<float*>(C) + at;
#pragma unroll
    for (int i = 0; i < CH; ++i, p += ld)
      if (i < left) *p = v[i];
  } else if (dtype == kBF16) {
    __nv_bfloat16* p = static_cast<__nv_bfloat16*>(C) + at;
#pragma unroll
    for (int i = 0; i < CH; ++i, p += ld)
      if (i < left) *p = __float2bfloat16_rn(v[i]);
  } else {
    __half* p = static_cast<__half*>(C) + at;
#pragma unroll
    for (int i = 0; i < CH; ++i, p += ld)
      if (i < left) *p = __float2half_rn(v[i]);
  }
}

// tmW: weights {K, rows per group, groups}, box {64, 128}.  tmX: A {K, a_rows},
// box {64, BOX}; not used when the rows are gathered.  Launched with
// Cfg::THREADS threads, and the gather warps on top when p.rows is given.
template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS + 32 * Cfg::GATHER_WARPS, 1)
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
      mbar_init(&full_bar[s], p.rows ? 1 + 32 * Cfg::GATHER_WARPS : 1);
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
  pdl_wait();  // offsets, rows, A and C belong to the previous grid until it completes
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
  // Only now: a dependent CTA that took TMEM first and waited for this grid
  // would keep this one from getting its own.
  pdl_launch_dependents();
  const uint32_t tmem_base = tmem_slot;
  volatile int* abortp = &abort_flag;
  const GroupedTiles<BN> tiles{p.groups, firsts, starts};
  const int k_blocks = (p.K + BK - 1) / BK;
  // Tiles u0, u0 + step, ... and the k-blocks of each that are this CTA's: all,
  // or in a cluster of p.splits CTAs the rank's share of one tile (the host
  // launches a cluster for every tile that there can be).
  int u0 = blockIdx.x, step = gridDim.x, kb0 = 0, kb1 = k_blocks;
  uint32_t rank = 0;
  if constexpr (Cfg::SPLIT) {
    rank = cluster_ctarank();
    u0 = blockIdx.x / p.splits;
    step = INT_MAX / 2;
    const int per = (k_blocks + p.splits - 1) / p.splits;
    kb0 = min(k_blocks, static_cast<int>(rank) * per);
    kb1 = min(k_blocks, kb0 + per);
  }

  if (warp == 0) {
    // ───────────── TMA producer ─────────────
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      bool ok = true;
      GroupedTile t;
      for (int u = u0; ok && tiles.get(u, t); u += step) {
        const int boxes = p.rows ? 0 : (t.rows + Cfg::BOX - 1) / Cfg::BOX;
        const uint32_t bytes = HALVES * Cfg::A_BYTES + boxes * Cfg::BOX * 128;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1u, p.err, kDevTimeoutProducer, abortp)) {
            ok = false;
            break;
          }
          uint8_t* sw = smem + stage * Cfg::STAGE_BYTES;
          const uint32_t sx = smem_u32(sw + HALVES * Cfg::A_BYTES);
          mbar_arrive_expect_tx(&full_bar[stage], bytes);
          tma_load_4d(sw, &tmW, &full_bar[stage], kb * BK, t.n0, t.g, 0);
          if constexpr (Cfg::GATE)
            tma_load_4d(sw + Cfg::A_BYTES, &tmW, &full_bar[stage], kb * BK, p.N + t.n0, t.g, 0);
          for (int b = 0; b < boxes; ++b)
            tma_load_2d(sx + b * Cfg::BOX * 128, &tmX, &full_bar[stage], kb * BK, t.row0 + b * Cfg::BOX);
          ++issued;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) {
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
    }
  } else if (warp >= 10) {
    // ───────────── gather (warps 10..17) ─────────────
    // Eight threads per row, 16 bytes each; thread i takes rows i / 8 + RP j.
    constexpr int RP = 4 * Cfg::GATHER_WARPS, J = BN / RP;
    const int i = threadIdx.x - Cfg::THREADS;
    const int r0 = i >> 3, c = i & 7;
    const uint32_t dst0 = r0 * 128 + ((c ^ (r0 & 7)) << 4);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    GroupedTile t;
    for (int u = u0; ok && tiles.get(u, t); u += step) {
      const uint16_t* from[J];
      uint32_t live = 0;  // rows that exist
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int r = r0 + RP * j;
        const int row = r < t.rows ? p.rows[t.row0 + r] : -1;
        const bool in = row >= 0 && row < p.a_rows;
        live |= in ? 1u << j : 0u;
        from[j] = static_cast<const uint16_t*>(p.A) + (in ? row * p.lda + kb0 * BK + 8 * c : 0);
      }
      for (int kb = kb0; kb < kb1; ++kb) {
        if (lane == 0) ok = mbar_wait(&empty_bar[stage], phase ^ 1u, p.err, kDevTimeoutProducer, abortp);
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        if (!ok) break;
        const uint32_t dst = smem_u32(smem + stage * Cfg::STAGE_BYTES + HALVES * Cfg::A_BYTES);
        const int in_row = min(max(p.K - (kb * BK + 8 * c), 0), 8) * 2;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          if (RP * j >= t.rows) break;
          const int bytes = (live >> j) & 1u ? in_row : 0;
          // RP j rows further on; with RP = 4 every other one is in the swizzle's other half
          gather_copy16(dst + j * (RP * 128) + (dst0 ^ (((RP * j) & 7) << 4)), from[j], bytes);
          from[j] += BK;
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full_bar[stage]))
                     : "memory");
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
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
      for (int u = u0; ok && tiles.get(u, t); u += step) {
        const uint32_t idesc = make_idesc(Cfg::FMT, 128, (t.rows + 15) / 16 * 16, 0u, 0u);
        if (!mbar_wait(&tempty_bar[acc], acc_phase ^ 1u, p.err, kDevTimeoutMma, abortp)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + static_cast<uint32_t>(acc * Cfg::ACC_COLS);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase, p.err, kDevTimeoutMma, abortp)) {
            ok = false;
            break;
          }
          if (p.rows) fence_proxy_async_smem();  // the gathered rows were written by cp.async
          tc_fence_after();
          const uint32_t w_addr = smem_u32(smem + stage * Cfg::STAGE_BYTES);
          const uint32_t x_addr = w_addr + HALVES * Cfg::A_BYTES;
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const uint64_t xd = make_sw128_desc(x_addr + ks * 32, 16, 1024);
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
              umma_f16(d + h * BN, make_sw128_desc(w_addr + h * Cfg::A_BYTES + ks * 32, 16, 1024), xd,
                       idesc, (kb > kb0 || ks > 0) ? 1u : 0u);
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
    for (int u = u0; tiles.get(u, t); u += step) {
      if constexpr (Cfg::SPLIT) {
        // The partial sums take the ring's place: every copy into it was
        // waited for and every MMA that read it has completed.
        if (kb0 >= kb1) break;
        // One outcome for the warp, here and below: TMEM loads of all its lanes follow.
        if (!__all_sync(0xffffffffu, mbar_wait(&tfull_bar[0], 0, p.err, kDevTimeoutEpilogue, abortp))) break;
        tc_fence_after();
        float* part = reinterpret_cast<float*>(smem) + quad * 32 + lane;
        for (int c = half * CH; c < t.rows; c += 2 * CH)
#pragma unroll
          for (int h = 0; h < HALVES; ++h) {
            float v[CH];
            tmem_load_chunk<CH>(tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + h * BN + c, v);
#pragma unroll
            for (int i = 0; i < CH; ++i) part[(h * BN + c + i) * 128] = v[i];
          }
        break;
      }
      const int n = t.n0 + quad * 32 + lane;  // this thread's weight row
      float bias0 = 0.0f, bias1 = 0.0f;
      if (p.bias && n < p.N) {
        bias0 = load_as_f32(p.bias, t.g * p.bias_stride + n, p.bias_dtype);
        if constexpr (Cfg::GATE) bias1 = load_as_f32(p.bias, t.g * p.bias_stride + p.N + n, p.bias_dtype);
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&tfull_bar[acc], acc_phase, p.err, kDevTimeoutEpilogue, abortp)))
        break;
      tc_fence_after();
      const uint32_t tbase = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) +
                             static_cast<uint32_t>(acc * Cfg::ACC_COLS);
#pragma unroll 1
      for (int c = half * CH; c < t.rows; c += 2 * CH) {
        float v[CH];
        tmem_load_chunk<CH>(tbase + c, v);
        if constexpr (Cfg::GATE) {
          float w[CH];
          tmem_load_chunk<CH>(tbase + BN + c, w);
#pragma unroll
          for (int i = 0; i < CH; ++i) {
            const float z = v[i] + bias0;
            v[i] = (p.fast_act ? act_apply_fast(z, kActSilu) : act_apply(z, kActSilu)) * (w[i] + bias1);
          }
        } else {
#pragma unroll
          for (int i = 0; i < CH; ++i) v[i] += bias0;
          activate<CH>(v, p.act, p.fast_act != 0);
        }
        if (n < p.N)
          store_column<CH>(p.C, static_cast<int64_t>(t.row0 + c) * p.ldc + n, p.ldc, p.out_dtype, v, t.rows - c);
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
  if constexpr (Cfg::SPLIT) {
    // Every CTA of the cluster sums every splits-th row of the tile over the
    // cluster's shared memory, in rank order.
    cluster_sync();
    GroupedTile t;
    if (tiles.get(u0, t)) {
      const int per = (k_blocks + p.splits - 1) / p.splits;
      const int ranks = (k_blocks + per - 1) / per;  // ranks with k-blocks
      const int i = threadIdx.x & 127, n = t.n0 + i;
      const uint32_t part = smem_u32(smem) + i * 4;
      if (n < p.N)
        for (int r = rank + p.splits * (threadIdx.x >> 7); r < t.rows; r += p.splits * (blockDim.x >> 7)) {
          if (static_cast<int>(threadIdx.x >> 7) >= static_cast<int>(blockDim.x >> 7)) break;
          float v[2] = {0.0f, 0.0f};
          for (int s = 0; s < ranks; ++s)
#pragma unroll
            for (int h = 0; h < HALVES; ++h) v[h] += load_cluster_f32(part + (h * BN + r) * 512, s);
          if (p.bias)
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
              v[h] += load_as_f32(p.bias, t.g * p.bias_stride + h * p.N + n, p.bias_dtype);
          store_from_f32(p.C, (static_cast<int64_t>(t.row0) + r) * p.ldc + n, p.out_dtype,
                         grouped_act(v[0], v[1], p.act, p.fast_act != 0));
        }
    }
    cluster_sync();  // no CTA leaves while its sums are being read
  }
}

}  // namespace sf
