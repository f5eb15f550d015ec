// Grouped GEMM: one linear per group over rows grouped by expert.
//
//   C[i, :] = act(B[g] . A[r(i), :] + bias[g]),  offsets[g] <= i < offsets[g+1],
//   r(i) = rows[i] or i
//
// Entry point and dispatch; the kernel is grouped_simt.cuh.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "common.h"
#include "grouped_simt.cuh"
#include "tma_host.h"

namespace sf {
namespace {

constexpr int64_t kMaxGroups = 4096;

int32_t run_simt(const GroupedArgs& a, cudaStream_t s) {
  const int64_t row_tiles = ceil_div(a.M, kGsTile) + std::min(a.groups, a.M);
  if (row_tiles > 65535)
    return fail(SF_ERR_UNSUPPORTED, "%d rows in %d groups exceed the grid of the FMA kernel", a.M, a.groups);
  const dim3 grid(static_cast<unsigned>(ceil_div(a.N, kGsTile)), static_cast<unsigned>(row_tiles));
  if (a.act == kActSiluGate)
    grouped_simt_kernel<true><<<grid, kGsThreads, 0, s>>>(a);
  else
    grouped_simt_kernel<false><<<grid, kGsThreads, 0, s>>>(a);
  SF_CUDA_TRY(cudaGetLastError());
  return SF_OK;
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" int32_t sf_gemm_grouped(int64_t groups, int64_t M, int64_t N, int64_t K, const void* A,
                                   int64_t a_rows, int64_t lda, const int32_t* rows,
                                   const int32_t* offsets, const void* B, int64_t ldb,
                                   int64_t b_stride, const void* bias, int32_t bias_dtype,
                                   int64_t bias_stride, void* C, int64_t ldc, int32_t in_dtype,
                                   int32_t out_dtype, int32_t activation, void* stream) {
  if (groups < 0 || M < 0 || N < 0 || K < 0 || a_rows < 0)
    return fail(SF_ERR_INVALID_ARGUMENT, "negative dimension");
  if (activation < SF_ACT_NONE || activation > SF_ACT_SILU_GATE)
    return fail(SF_ERR_INVALID_ARGUMENT, "unknown activation %d", activation);
  for (int dt : {in_dtype, out_dtype})
    if (dt != kF32 && dt != kF16 && dt != kBF16)
      return fail(SF_ERR_INVALID_ARGUMENT, "unknown dtype %d", dt);
  if (groups == 0 || M == 0 || N == 0) return SF_OK;
  const int64_t wide = activation == SF_ACT_SILU_GATE ? 2 * N : N;
  if (M > INT32_MAX || wide > INT32_MAX || K > INT32_MAX || a_rows > INT32_MAX)
    return fail(SF_ERR_UNSUPPORTED, "dimension exceeds 2^31-1");
  if (groups > kMaxGroups)
    return fail(SF_ERR_UNSUPPORTED, "%lld groups (at most %lld)", (long long)groups, (long long)kMaxGroups);
  if (!offsets || !C || (K > 0 && (!A || !B))) return fail(SF_ERR_INVALID_ARGUMENT, "null pointer");
  if (!rows && a_rows < M)
    return fail(SF_ERR_INVALID_ARGUMENT, "A has %lld rows, %lld needed", (long long)a_rows, (long long)M);
  if (ldc < N || lda < K || ldb < K) return fail(SF_ERR_INVALID_ARGUMENT, "leading dimension too small");
  if (bias && bias_dtype != kF32 && bias_dtype != kF16 && bias_dtype != kBF16)
    return fail(SF_ERR_INVALID_ARGUMENT, "unknown bias dtype");
  DeviceInfo* dev = nullptr;
  const int32_t st = current_device_info(&dev, nullptr);
  if (st != SF_OK) return st;
  GroupedArgs a{};
  a.groups = static_cast<int>(groups);
  a.M = static_cast<int>(M);
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  a.A = A;
  a.a_rows = a_rows;
  a.lda = lda;
  a.rows = rows;
  a.offsets = offsets;
  a.B = B;
  a.ldb = ldb;
  a.b_stride = b_stride;
  a.bias = bias;
  a.bias_dtype = bias_dtype;
  a.bias_stride = bias_stride;
  a.C = C;
  a.ldc = ldc;
  a.in_dtype = in_dtype;
  a.out_dtype = out_dtype;
  a.act = activation;
  a.fast_act = out_dtype != kF32 ? 1 : 0;
  a.err = dev->err_word;
  return run_simt(a, static_cast<cudaStream_t>(stream));
}
