// 4-bit linear for up to 16 rows of x on mma.m16n8k16.
//
// The weight stream is half a byte per weight against 16 multiply-adds at most
// 8 rows of x, and what has to keep up with it is the unpacking: at 6.5 TB/s a
// lane has 2.8 issue slots per weight.  A packed word becomes four operand
// registers by masking two nibbles at a time into the mantissas of 128 (bf16)
// or 1024 (fp16) and subtracting that plus the zero point, which is exact: 1.1
// to 1.4 operations per weight, one scale and four multiply-adds per group, and
// the tensor core does the products.  Everything else is kept away from the
// unpacking warps: words and x arrive by TMA in the order in which the lanes
// read them.
//
// A CTA takes 128 weight rows, a warp 32 of them.  In a 128-column block, lane
// (g, t) = (lane / 4, lane % 4) reads 16 bytes of each of rows g, g + 8, g + 16,
// g + 24: words 4 t .. 4 t + 3, whose columns 32 w + 8 t .. + 7 are one 16-byte
// piece of x for token g.  The order of k within an mma is free as long as both
// operands agree, so the layout makes every read of both operands 16 bytes and
// word w of all four t one 32-column group.  A cluster of `splits` CTAs shares
// the blocks of the 128 rows; the partial sums meet in shared memory and are
// added in rank order.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "ptx.cuh"
#include "w4_unpack.cuh"

namespace sf {

template <bool BF16_, int NT_, int GW_>
struct W4StreamCfg {
  static constexpr bool BF16 = BF16_;
  static constexpr int NT = NT_;     // rows of x / 8
  static constexpr int GW = GW_;     // 32-column words per group: 1, 2, 4
  static constexpr int NG = 4 / GW;  // groups per block
  static constexpr int W_BYTES = 128 * 64;
  static constexpr int X_BYTES = NT * 8 * 256;
  static constexpr int S_BYTES = NG * 256;  // scales of a block; as much again for zeros
  static constexpr int STAGE_BYTES = W_BYTES + X_BYTES + 2 * S_BYTES;
  static constexpr int STAGES = 4;
  static constexpr int THREADS = 160;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 128;
  static_assert(STAGES * STAGE_BYTES >= NT * 8 * 512, "partial sums fit the ring");
};

__device__ __forceinline__ void stream_load_2d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}

// tmW: packed words {16 per block, N}, box {16, 128}.  tmX: x as {32, M, K / 32},
// box {32, 8 NT, 4}: a block lands as [word w][row of x][32 columns].  tmS, tmZ:
// scales and zeros {N, groups}, box {128, NG}; tmZ is not used without zeros.
template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, 4)
    w4_stream_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                     const __grid_constant__ CUtensorMap tmS, const __grid_constant__ CUtensorMap tmZ,
                     const W4Args a, int splits, int* err) {
  constexpr int STAGES = Cfg::STAGES, NT = Cfg::NT, NG = Cfg::NG, GW = Cfg::GW;
  constexpr bool BF16 = Cfg::BF16;
  constexpr int NA = w4_accumulators(NT, GW);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~static_cast<uintptr_t>(127));
  __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES];
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int n0 = static_cast<int>(blockIdx.x / splits) * 128;
  const int blocks = (a.K + 127) / 128;
  const int per = (blocks + splits - 1) / splits;
  const int b0 = min(blocks, static_cast<int>(rank) * per), b1 = min(blocks, b0 + per);

  if (threadIdx.x == 128) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full_bar[i], 1);
      mbar_init(&empty_bar[i], 4);
    }
    abort_flag = 0;
    fence_mbar_init();
    for (int b = b0; b < min(b1, b0 + STAGES); ++b)
      asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(
                       reinterpret_cast<uint64_t>(&tmW)),
                   "r"(16 * b), "r"(n0)
                   : "memory");
  }
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();
  volatile int* abortp = &abort_flag;
  const bool zeros = a.zeros != nullptr;

  if (warp == 4) {
    if (lane == 0) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int b = b0; b < b1; ++b) {
        ok = mbar_wait(&empty_bar[stage], phase ^ 1u, err, kDevTimeoutProducer, abortp);
        if (!ok) break;
        const uint32_t sw = smem_u32(smem + stage * Cfg::STAGE_BYTES);
        mbar_arrive_expect_tx(&full_bar[stage], Cfg::STAGE_BYTES - (zeros ? 0 : Cfg::S_BYTES));
        stream_load_2d(sw, &tmW, &full_bar[stage], 16 * b, n0);
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %3, %4}], "
            "[%2];" ::"r"(sw + Cfg::W_BYTES),
            "l"(reinterpret_cast<uint64_t>(&tmX)), "r"(smem_u32(&full_bar[stage])), "r"(0), "r"(4 * b)
            : "memory");
        stream_load_2d(sw + Cfg::W_BYTES + Cfg::X_BYTES, &tmS, &full_bar[stage], n0, b * NG);
        if (zeros) stream_load_2d(sw + Cfg::W_BYTES + Cfg::X_BYTES + Cfg::S_BYTES, &tmZ, &full_bar[stage], n0, b * NG);
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
    __syncwarp();
    __syncthreads();
  } else {
    const int g = lane >> 2, t = lane & 3;
    float acc[2][NT][4] = {};
    const uint8_t* words = smem + (32 * warp + g) * 64 + t * 16;
    const uint8_t* xs = smem + Cfg::W_BYTES + g * 64 + t * 16;
    // scale and zero of row 32 warp + lane, shared out by shuffles
    const uint8_t* ss = smem + Cfg::W_BYTES + Cfg::X_BYTES + (32 * warp + lane) * 2;
    uint32_t phase = 0;
    // A lane whose wait gives up (limit or abort flag) does not leave the others,
    // which shuffle and multiply with it: it goes on with what is there and hands
    // nothing back, the later waits end by the flag, and the status is in the error
    // word.  Leaving by a vote of the warp instead takes 40.5 us where this takes
    // 40.1 (5 x 8192 -> 28672, groups of 64), 34.8 where this takes 34.1 (one row).
#pragma unroll 1
    for (int i0 = b0; i0 < b1; i0 += STAGES, phase ^= 1u) {
#pragma unroll
      for (int u = 0; u < STAGES; ++u) {
        if (i0 + u >= b1) break;
        const bool ok = mbar_wait(&full_bar[u], phase, err, kDevTimeoutEpilogue, abortp);
        uint4 q[4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          q[r] = *reinterpret_cast<const uint4*>(words + u * Cfg::STAGE_BYTES + r * 512);
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          const uint8_t* at = ss + u * Cfg::STAGE_BYTES + j * 256;
          const uint32_t sv = pack_scale<BF16>(
              *reinterpret_cast<const uint16_t*>(at),
              zeros ? *reinterpret_cast<const uint16_t*>(at + Cfg::S_BYTES) : 0u, zeros);
          float s[4];
          uint2 z[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) unpack_scale<BF16>(__shfl_sync(0xffffffffu, sv, 8 * r + g), s[r], z[r]);
          float sum[2][NT][NA][4] = {};
#pragma unroll
          for (int l = 0; l < GW; ++l) {
            const int w = j * GW + l;
            uint32_t p[4][4];
#pragma unroll
            for (int r = 0; r < 4; ++r)
              unpack_word<BF16>(w == 0 ? q[r].x : w == 1 ? q[r].y : w == 2 ? q[r].z : q[r].w, z[r], p[r]);
#pragma unroll
            for (int m = 0; m < NT; ++m) {
              const uint4 x =
                  *reinterpret_cast<const uint4*>(xs + u * Cfg::STAGE_BYTES + (w * NT + m) * 512);
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                const uint32_t a0[4] = {p[2 * r][0], p[2 * r + 1][0], p[2 * r][1], p[2 * r + 1][1]};
                const uint32_t a1[4] = {p[2 * r][2], p[2 * r + 1][2], p[2 * r][3], p[2 * r + 1][3]};
                mma_16816<BF16>(sum[r][m][2 * l % NA], a0, x.x, x.y);
                mma_16816<BF16>(sum[r][m][2 * l % NA + 1], a1, x.z, x.w);
              }
            }
          }
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int m = 0; m < NT; ++m)
#pragma unroll
              for (int c = 0; c < 4; ++c)
                acc[r][m][c] = fmaf(s[2 * r + (c >> 1)], sum_of<NA>(sum[r][m], c), acc[r][m][c]);
        }
        __syncwarp();
        if (lane == 0 && ok) mbar_arrive(&empty_bar[u]);
      }
    }
    __syncthreads();  // every block has been read: the sums take the ring's place
    // [token][row]: acc c is row g + 8 (c / 2), token 2 t + c % 2
    float* part = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int m = 0; m < NT; ++m)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          part[(8 * m + 2 * t + (c & 1)) * 128 + 32 * warp + 16 * r + g + 8 * (c >> 1)] = acc[r][m][c];
  }
  cluster_sync();
  const int n = n0 + static_cast<int>(threadIdx.x);
  if (threadIdx.x < 128 && n < a.N) {
    const uint32_t mine = smem_u32(smem) + threadIdx.x * 4;
    const float bias = a.bias ? load_as_f32(a.bias, n, a.bias_dtype) : 0.0f;
    for (int m = rank; m < a.M; m += splits) {
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
