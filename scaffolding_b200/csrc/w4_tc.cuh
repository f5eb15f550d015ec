// 4-bit linear on tcgen05 with the unpacked weights in tensor memory.
//
//   D[n, m] = sum over a group's k of (q[n, k] - zero[n]) x[m, k]
//   y[m, n] = act(sum over groups of scale[n] D[n, m] + bias[n])
//
// 128 weight rows are the MMA's row side and the rows of x (padded to 16) its
// N side, so the unpacking -- what has to keep up with the weight stream -- is
// done once per weight whatever the number of rows of x is, and neither x nor
// the unpacked weights pass through a thread's or shared memory's bandwidth:
// packed words arrive by TMA (64 bytes of 128 rows per 128-column block), a
// thread unpacks one row of a block (sixteen words into 64 operand registers)
// into the TMEM columns that the MMA reads its A operand from, x arrives by TMA
// in the layout that the MMA reads.  The integers q - zero are exact in 16 bits
// and every group's sum has an accumulator of its own; more warps add the group
// sums up in fp32 registers, scaled, while later groups are in the MMA.
//
// CTA: warp 0 TMA, warp 1 MMA and TMEM, warps 2-5 unpacking, warps 6-13 sums
// (half of the rows of x each), one 32-lane TMEM quadrant per warp.  Two CTAs
// share an SM.  A cluster of `splits` CTAs shares the blocks of one row tile;
// the partial sums meet in shared memory and are added in rank order.
//
// An MMA with its A operand in TMEM takes about 65 cycles for 128 x 16 however
// few rows of x there are, 520 per block, which caps an SM at 16 bytes of
// packed words per cycle; up to 16 rows of x the mma.sync kernel is as fast
// or faster.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "ptx.cuh"
#include "w4_unpack.cuh"

namespace sf {

template <bool BF16_, int GW_>
struct W4TcCfg {
  static constexpr bool BF16 = BF16_;
  static constexpr int NT = 64;          // most rows of x
  static constexpr int GW = GW_;         // 32-column words per group: 1, 2, 4
  static constexpr int NG = 4 / GW;      // groups per block
  static constexpr int W_BYTES = 128 * 64;
  static constexpr int X_BYTES = 2 * NT * 128;
  static constexpr int STAGE_BYTES = W_BYTES + X_BYTES;
  static constexpr int STAGES = 4;
  static constexpr int A_BUFS = 2, A_COLS = 64;  // unpacked blocks
  static constexpr int D_BUFS = 2;               // group accumulators
  static constexpr int D_COL = A_BUFS * A_COLS;
  static constexpr int TMEM_COLS = 256;
  static constexpr int SUM_COLS = 32;            // rows of x per summing warp
  static constexpr int THREADS = 64 + 128 + 256;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024;
  static_assert(D_COL + D_BUFS * NT <= TMEM_COLS, "TMEM columns");
  static_assert(STAGES * STAGE_BYTES >= NT * 512, "partial sums fit the ring");
  static_assert(SMEM_BYTES <= 113 * 1024, "two CTAs per SM");
};

// acc[2 i], acc[2 i + 1] += s * d[2 i], s * d[2 i + 1] as one packed operation.
__device__ __forceinline__ void fma2(float& a0, float& a1, float s, uint32_t d0, uint32_t d1) {
  uint64_t a, b, c;
  asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "r"(__float_as_uint(a0)), "r"(__float_as_uint(a1)));
  asm("mov.b64 %0, {%1, %1};" : "=l"(b) : "r"(__float_as_uint(s)));
  asm("mov.b64 %0, {%1, %2};" : "=l"(c) : "r"(d0), "r"(d1));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(a) : "l"(b), "l"(c));
  uint32_t r0, r1;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(r0), "=r"(r1) : "l"(a));
  a0 = __uint_as_float(r0);
  a1 = __uint_as_float(r1);
}

__device__ __forceinline__ void w4_load_2d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}

__device__ __forceinline__ void w4_prefetch_2d(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y)
               : "memory");
}

// tmW: packed words {16 per block, N}, box {16, 128}, 64-byte swizzle.  tmX: x
// {K, M}, box {64, n_rows}, 128-byte swizzle.  n_rows: M rounded up to 16.
template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, 2)
    w4_tc_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                 const W4Args a, int splits, int n_rows, int* err) {
  constexpr int STAGES = Cfg::STAGES, NG = Cfg::NG, GW = Cfg::GW, NT = Cfg::NT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES];
  __shared__ __align__(8) uint64_t afull_bar[Cfg::A_BUFS], aempty_bar[Cfg::A_BUFS];
  __shared__ __align__(8) uint64_t dfull_bar[Cfg::D_BUFS], dempty_bar[Cfg::D_BUFS];
  __shared__ __align__(8) uint64_t drain_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int n0 = static_cast<int>(blockIdx.x / splits) * 128;
  const int blocks = (a.K + 127) / 128;
  const int per = (blocks + splits - 1) / splits;
  const int b0 = min(blocks, static_cast<int>(rank) * per), b1 = min(blocks, b0 + per);

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full_bar[i], 1);
      mbar_init(&empty_bar[i], 5);  // the four unpacking warps and the MMA
    }
    for (int i = 0; i < Cfg::A_BUFS; ++i) {
      mbar_init(&afull_bar[i], 4);
      mbar_init(&aempty_bar[i], 1);
    }
    for (int i = 0; i < Cfg::D_BUFS; ++i) {
      mbar_init(&dfull_bar[i], 1);
      mbar_init(&dempty_bar[i], 8);
    }
    mbar_init(&drain_bar, 1);
    abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmX);
    for (int b = b0; b < min(b1, b0 + STAGES); ++b) w4_prefetch_2d(&tmW, 16 * b, n0);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Only now: a dependent CTA that took TMEM first and waited for this grid
  // would keep this one from getting its own.
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t tmem_base = tmem_slot;
  volatile int* abortp = &abort_flag;
  float* const part = reinterpret_cast<float*>(smem);
  if (warp == 0) {
    // ───────────── TMA producer ─────────────
    if (lane == 0) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t bytes = Cfg::W_BYTES + 2 * n_rows * 128;
      for (int b = b0; b < b1; ++b) {
        ok = mbar_wait(&empty_bar[stage], phase ^ 1u, err, kDevTimeoutProducer, abortp);
        if (!ok) break;
        const uint32_t sw = smem_u32(smem + stage * Cfg::STAGE_BYTES);
        mbar_arrive_expect_tx(&full_bar[stage], bytes);
        w4_load_2d(sw, &tmW, &full_bar[stage], 16 * b, n0);
        w4_load_2d(sw + Cfg::W_BYTES, &tmX, &full_bar[stage], 128 * b, 0);
        w4_load_2d(sw + Cfg::W_BYTES + NT * 128, &tmX, &full_bar[stage], 128 * b + 64, 0);
        ++issued;
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) {
        // Abort: wait (bounded) for the copies still in flight.
        const int n = issued < STAGES ? issued : STAGES;
        for (int j = 0; j < n; ++j) {
          if (--stage < 0) {
            stage = STAGES - 1;
            phase ^= 1u;
          }
          if (!mbar_wait_quiet(&full_bar[stage], phase, 200000000ull)) atomicCAS(err, 0, kDevTimeoutDrain);
        }
      }
    }
  } else if (warp == 1) {
    // ───────────── MMA issuer ─────────────
    if (lane == 0) {
      const uint32_t idesc = make_idesc(Cfg::BF16 ? 1u : 0u, 128, n_rows, 0u, 0u);
      int stage = 0, ab = 0, db = 0;
      uint32_t phase = 0, aphase = 0, dphase = 0;
      bool ok = true, issued_any = false;
      for (int b = b0; ok && b < b1; ++b) {
        ok = mbar_wait(&full_bar[stage], phase, err, kDevTimeoutMma, abortp) &&
             mbar_wait(&afull_bar[ab], aphase, err, kDevTimeoutMma, abortp);
        if (!ok) break;
        const uint32_t x_addr = smem_u32(smem + stage * Cfg::STAGE_BYTES + Cfg::W_BYTES);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          ok = mbar_wait(&dempty_bar[db], dphase ^ 1u, err, kDevTimeoutMma, abortp);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int j = 0; j < 2 * GW; ++j) {
            const int ks = 2 * GW * g + j;  // 16 columns of the block
            umma_f16_tmem_a(tmem_base + Cfg::D_COL + db * NT, tmem_base + ab * Cfg::A_COLS + ks * 8,
                            make_sw128_desc(x_addr + (ks >> 2) * (NT * 128) + (ks & 3) * 32, 16, 1024), idesc,
                            j > 0 ? 1u : 0u);
          }
          issued_any = true;
          umma_commit(&dfull_bar[db]);
          if (++db == Cfg::D_BUFS) {
            db = 0;
            dphase ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit(&empty_bar[stage]);
        umma_commit(&aempty_bar[ab]);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
        if (++ab == Cfg::A_BUFS) {
          ab = 0;
          aphase ^= 1u;
        }
      }
      if (!ok && issued_any) {
        // Abort: no tcgen05.mma may still be at work when TMEM is freed.
        umma_commit(&drain_bar);
        if (!mbar_wait_quiet(&drain_bar, 0, 200000000ull)) atomicCAS(err, 0, kDevTimeoutDrain);
      }
    }
  } else {
    const int quad = warp & 3;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const int n = min(n0 + quad * 32 + lane, a.N - 1);  // this thread's weight row
    const int groups = (a.K + 32 * GW - 1) / (32 * GW);
    if (warp < 6) {
      // ───────────── unpacking (warps 2..5) ─────────────
      const uint16_t* zp = static_cast<const uint16_t*>(a.zeros) + n;
      const bool zeros = a.zeros != nullptr;
      const uint32_t row = quad * 32 + lane;
      const uint32_t sw64 = (row >> 1) & 3;
      int stage = 0, ab = 0;
      uint32_t phase = 0, aphase = 0;
      uint32_t zn[2][NG];  // two blocks ahead
      auto load_zeros = [&](uint32_t (&to)[NG], int b) {
        if (!zeros) return;
#pragma unroll
        for (int g = 0; g < NG; ++g) to[g] = load_ahead(zp + min(b * NG + g, groups - 1) * a.lds);
      };
      load_zeros(zn[0], b0);
      load_zeros(zn[1], b0 + 1);
      // A lane whose wait gives up (limit or abort flag), here or among the sums,
      // does not leave the others, whose TMEM accesses are the whole warp's: it goes
      // on with what is there and hands nothing on, the later waits end by the flag,
      // and the status is in the error word.  (Leaving by a vote of the warp instead:
      // 22.1 -> 22.7 us at 64 x 4096 -> 11008, 27.0 -> 28.4 us at 64 x 11008 -> 4096
      // with groups of 32.)
      for (int b = b0; b < b1; b += 2) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (b + i >= b1) break;
          uint2 z[NG];
#pragma unroll
          for (int g = 0; g < NG; ++g)
            z[g] = zeros ? zero_pair<Cfg::BF16>(zn[i][g])
                         : make_uint2(Cfg::BF16 ? 0x43084308u : 0x64086408u, 0x54805480u);  // + 8
          load_zeros(zn[i], b + i + 2);
          bool ok = mbar_wait(&full_bar[stage], phase, err, kDevTimeoutEpilogue, abortp);
          const uint8_t* src = smem + stage * Cfg::STAGE_BYTES + row * 64;
          uint4 q[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) q[t] = *reinterpret_cast<const uint4*>(src + ((t ^ sw64) << 4));
          ok = mbar_wait(&aempty_bar[ab], aphase ^ 1u, err, kDevTimeoutEpilogue, abortp) && ok;
          tc_fence_after();
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t p[16];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              uint32_t(&p4)[4] = *reinterpret_cast<uint32_t(*)[4]>(p + 4 * t);
              unpack_word<Cfg::BF16>(w == 0 ? q[t].x : w == 1 ? q[t].y : w == 2 ? q[t].z : q[t].w, z[w / GW], p4);
            }
            tmem_st16(tmem_base + lanes + ab * Cfg::A_COLS + 16 * w, p);
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0 && ok) {
            mbar_arrive(&empty_bar[stage]);
            mbar_arrive(&afull_bar[ab]);
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
          if (++ab == Cfg::A_BUFS) {
            ab = 0;
            aphase ^= 1u;
          }
        }
      }
    } else {
      // ───────────── sums (warps 6..13) ─────────────
      constexpr int SC = Cfg::SUM_COLS;
      const int col = ((warp - 6) >> 2) * SC;  // first row of x of this warp
      float acc[SC];
#pragma unroll
      for (int i = 0; i < SC; ++i) acc[i] = 0.0f;
      const uint16_t* sp = static_cast<const uint16_t*>(a.scales) + n;
      auto scale = [&](int grp) { return load_ahead(sp + min(grp, groups - 1) * a.lds); };
      int db = 0;
      uint32_t dphase = 0;
      constexpr int AHEAD = 4;  // groups
      uint32_t next[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) next[i] = scale(b0 * NG + i);
      for (int g0 = b0 * NG; g0 < b1 * NG; g0 += AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          if (g0 + i >= b1 * NG) break;
          const float s = g0 + i < groups ? w4_float<Cfg::BF16>(next[i]) : 0.0f;
          next[i] = scale(g0 + i + AHEAD);
          const bool ok = mbar_wait(&dfull_bar[db], dphase, err, kDevTimeoutEpilogue, abortp);
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < SC; c += 16) {
            if (col + c >= n_rows) break;
            uint32_t d[16];
            tmem_ld16(tmem_base + lanes + Cfg::D_COL + db * NT + col + c, d);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; j += 2) fma2(acc[c + j], acc[c + j + 1], s, d[j], d[j + 1]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0 && ok) mbar_arrive(&dempty_bar[db]);
          if (++db == Cfg::D_BUFS) {
            db = 0;
            dphase ^= 1u;
          }
        }
      }
      // [row of x][weight row] partial sums in the ring's place: with the last
      // group's MMA every copy into the ring has been used.
#pragma unroll
      for (int i = 0; i < SC; ++i)
        if (col + i < a.M) part[(col + i) * 128 + quad * 32 + lane] = acc[i];
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
  cluster_sync();
  const int i = threadIdx.x & 127, n = n0 + i, group = threadIdx.x >> 7;
  constexpr int kGroups = Cfg::THREADS / 128;  // whole groups of 128 threads
  if (group < kGroups && n < a.N) {
    const uint32_t mine = smem_u32(part) + i * 4;
    const float bias = a.bias ? load_as_f32(a.bias, n, a.bias_dtype) : 0.0f;
    for (int m = rank + splits * group; m < a.M; m += kGroups * splits) {
      float v = 0.0f;
      for (int s = 0; s < splits; ++s) {
        float f;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(mapa_shared(mine + m * 512, s)) : "memory");
        v += f;
      }
      v += bias;
      v = a.fast_act ? act_apply_fast(v, a.act) : act_apply(v, a.act);
      store_from_f32(a.y, m * a.ldy + n, a.out_dtype, v);
    }
  }
  cluster_sync();  // no CTA leaves while its sums are being read
}

}  // namespace sf
