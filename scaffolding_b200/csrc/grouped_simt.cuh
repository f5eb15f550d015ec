// Grouped GEMM on the FMA pipe, for what the tensor-core kernel cannot take:
// fp32 operands (IEEE fp32 multiply-add) and 16-bit layouts that TMA cannot
// describe (rows that do not start on 16-byte boundaries).
//
// 64 x 64 output tiles, 16-deep k steps staged in shared memory, 4 x 4 outputs
// per thread (4 x 4 of both halves for the gated activation).
#pragma once
#include <cstdint>

#include "epilogue.cuh"

namespace sf {

struct GroupedArgs {
  int groups;
  int M, N, K;            // N: columns of the output
  const void* A;
  int64_t a_rows, lda;
  const int* rows;        // row of A of each output row, or null
  const int* offsets;     // [groups + 1]
  const void* B;          // [groups][N, or 2 N when gated][K]
  int64_t ldb, b_stride;
  const void* bias;       // [groups][N, or 2 N when gated], or null
  int bias_dtype;
  int64_t bias_stride;
  void* C;
  int64_t ldc;
  int in_dtype, out_dtype;
  int act;                // Act, or kActSiluGate
  int fast_act;
  int* err;
};

// Gated SiLU: y = silu(v[n]) * v[N + n]; the grouped GEMM's only, since it
// pairs two weight rows for one output.
constexpr int kActSiluGate = 3;

// First and past-the-last row of group g.  Offsets are device data: each is
// clamped to [0, M], so that no row outside the tensors is reached whatever
// they hold.
__device__ __forceinline__ void group_rows(const GroupedArgs& p, int g, int& lo, int& hi) {
  lo = min(max(p.offsets[g], 0), p.M);
  hi = max(lo, min(p.offsets[g + 1], p.M));
}

__device__ __forceinline__ float grouped_act(float v, float gate_up, int act, bool fast) {
  if (act == kActSiluGate)
    return (fast ? act_apply_fast(v, kActSilu) : act_apply(v, kActSilu)) * gate_up;
  return fast ? act_apply_fast(v, act) : act_apply(v, act);
}

constexpr int kGsTile = 64, kGsK = 16, kGsThreads = 256;

template <bool GATE>
static __global__ void __launch_bounds__(kGsThreads) grouped_simt_kernel(const GroupedArgs p) {
  __shared__ float As[kGsK][kGsTile + 4];
  __shared__ float Bs[GATE ? 2 : 1][kGsK][kGsTile + 4];
  __shared__ int found[2];
  const int n0 = blockIdx.x * kGsTile;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  // Tile blockIdx.y of the groups' tiles laid end to end; the host launches
  // as many as there can be (a partial tile per group on top of M / 64).
  if (tid < 32) {
    int at = 0, g_hit = -1, first = 0;
    for (int g0 = 0; g0 < p.groups && g_hit < 0; g0 += 32) {
      const int g = g0 + tid;
      int lo = 0, hi = 0;
      if (g < p.groups) group_rows(p, g, lo, hi);
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
        const int l = __ffs(past) - 1;
        g_hit = g0 + l;
        first = __shfl_sync(0xffffffffu, end - tiles, l);
      }
      at = __shfl_sync(0xffffffffu, end, 31);
    }
    if (tid == 0) {
      found[0] = g_hit;
      found[1] = static_cast<int>(blockIdx.y) - first;
    }
  }
  __syncthreads();
  const int g = found[0];
  if (g < 0) return;
  int lo, hi;
  group_rows(p, g, lo, hi);
  const int m0 = lo + found[1] * kGsTile;
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
