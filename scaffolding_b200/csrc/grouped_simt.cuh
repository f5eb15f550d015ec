// Grouped GEMM on the FMA pipe, for what the tensor-core kernel cannot take:
// fp32 operands (IEEE fp32 multiply-add) and 16-bit layouts that TMA cannot
// describe (rows that do not start on 16-byte boundaries).
//
// 64 x 64 output tiles, 16-deep k steps staged in shared memory, 4 x 4 outputs
// per thread (4 x 4 of both halves for the gated activation).
#pragma once
#include <cstdint>

#include "grouped_args.cuh"

namespace sf {

constexpr int kGsTile = 64, kGsK = 16, kGsThreads = 256;

template <bool GATE>
static __global__ void __launch_bounds__(kGsThreads) grouped_simt_kernel(const GroupedArgs p) {
  __shared__ float As[kGsK][kGsTile + 4];
  __shared__ float Bs[GATE ? 2 : 1][kGsK][kGsTile + 4];
  __shared__ int found[3];
  const int n0 = blockIdx.x * kGsTile;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  // Tile blockIdx.y of the groups' tiles laid end to end; the host launches
  // as many as there can be (a partial tile per group on top of M / 64).
  if (tid < 32) {
    int at = 0, floor = 0;
    if (tid == 0) found[0] = -1;
    __syncwarp();
    for (int g0 = 0; g0 < p.groups; g0 += 32) {
      int lo, hi;
      group_bounds(p, g0, floor, lo, hi);
      const int tiles = (hi - lo + kGsTile - 1) / kGsTile;
      int end = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, end, o);
        if (tid >= o) end += v;
      }
      end += at;
      const unsigned past = __ballot_sync(0xffffffffu, end > static_cast<int>(blockIdx.y));
      if (past) {
        if (tid == __ffs(past) - 1) {
          found[0] = g0 + tid;
          found[1] = lo + (static_cast<int>(blockIdx.y) - (end - tiles)) * kGsTile;
          found[2] = hi;
        }
        break;
      }
      at = __shfl_sync(0xffffffffu, end, 31);
    }
  }
  __syncthreads();
  const int g = found[0];
  if (g < 0) return;
  const int m0 = found[1], hi = found[2];
  const int64_t brow = static_cast<int64_t>(g) * p.b_stride;

  // The row of A that this thread stages (four threads per row).
  const int sr = tid >> 2, sk = (tid & 3) * 4;
  int64_t arow = -1;
  if (m0 + sr < hi) {
    arow = p.rows ? p.rows[m0 + sr] : m0 + sr;
    if (arow < 0 || arow >= p.a_rows) arow = -1;
  }
  float acc[GATE ? 2 : 1][4][4] = {};
  for (int k0 = 0; k0 < p.K; k0 += kGsK) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int k = k0 + sk + t;
      As[sk + t][sr] = (arow >= 0 && k < p.K) ? load_as_f32(p.A, arow * p.lda + k, p.in_dtype) : 0.0f;
#pragma unroll
      for (int h = 0; h < (GATE ? 2 : 1); ++h)
        Bs[h][sk + t][sr] =
            (n0 + sr < p.N && k < p.K)
                ? load_as_f32(p.B, brow + (n0 + sr + static_cast<int64_t>(h) * p.N) * p.ldb + k, p.in_dtype)
                : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < kGsK; ++kk) {
      const float4 a = *reinterpret_cast<const float4*>(&As[kk][ty * 4]);
      const float av[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int h = 0; h < (GATE ? 2 : 1); ++h) {
        const float4 b = *reinterpret_cast<const float4*>(&Bs[h][kk][tx * 4]);
        const float bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[h][i][j] = fmaf(av[i], bv[j], acc[h][i][j]);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + ty * 4 + i;
    if (m >= hi) break;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx * 4 + j;
      if (n >= p.N) break;
      float v = acc[0][i][j], u = 0.0f;
      if constexpr (GATE) u = acc[GATE ? 1 : 0][i][j];
      if (p.bias) {
        v += load_as_f32(p.bias, g * p.bias_stride + n, p.bias_dtype);
        if constexpr (GATE) u += load_as_f32(p.bias, g * p.bias_stride + p.N + n, p.bias_dtype);
      }
      store_from_f32(p.C, m * p.ldc + n, p.out_dtype, grouped_act(v, u, p.act, p.fast_act != 0));
    }
  }
}

}  // namespace sf
