// Arguments and row bounds shared by the grouped GEMM kernels.
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
  int splits;             // CTAs per tile of the split kernel
  int* err;
};

// Gated SiLU: y = silu(v[n]) * v[N + n]; the grouped GEMM's only, since it
// pairs two weight rows for one output.
constexpr int kActSiluGate = 3;

// Offsets are device data and may hold anything: the kernels use the running
// maximum of the offsets clamped to [0, M], which is the offsets themselves
// when they are as documented, so that no row outside the tensors is reached
// and no row is in two groups.
//
// Bounds of 32 groups g0 + lane at once, by a full warp: lo and hi of this
// lane's group (an empty one past the last), given `floor`, the end of the
// groups in front of g0, which moves on to the end of these.
__device__ __forceinline__ void group_bounds(const GroupedArgs& p, int g0, int& floor, int& lo, int& hi) {
  const int lane = threadIdx.x & 31, g = g0 + lane;
  auto clamped = [&](int i) { return min(max(p.offsets[min(i, p.groups)], 0), p.M); };
  lo = max(clamped(g), floor);
  hi = clamped(g + 1);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, lo, o);
    if (lane >= o) lo = max(lo, v);
  }
  hi = max(hi, lo);
  floor = __shfl_sync(0xffffffffu, hi, 31);
}

__device__ __forceinline__ float grouped_act(float v, float gate_up, int act, bool fast) {
  if (act == kActSiluGate)
    return (fast ? act_apply_fast(v, kActSilu) : act_apply(v, kActSilu)) * gate_up;
  return fast ? act_apply_fast(v, act) : act_apply(v, act);
}

}  // namespace sf
