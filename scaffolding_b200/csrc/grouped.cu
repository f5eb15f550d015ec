// Grouped GEMM: one linear per group over rows grouped by expert.
//
//   C[i, :] = act(B[g] . A[r(i), :] + bias[g]),  offsets[g] <= i < offsets[g+1],
//   r(i) = rows[i] or i
//
// Entry point and dispatch: 16-bit operands whose rows TMA can describe run on
// tcgen05 (grouped_tc.cuh), everything else on the FMA pipe (grouped_simt.cuh).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "common.h"
#include "grouped_simt.cuh"
#include "grouped_tc.cuh"
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

// 2-D map of A {K, a_rows}, boxes of `box_rows` rows by 64 columns.
int32_t encode_rows(CUtensorMap* m, const GroupedArgs& a, uint32_t box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(SF_ERR_CUDA, "cuTensorMapEncodeTiled unavailable from the driver");
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.K), static_cast<cuuint64_t>(a.a_rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(a.lda) * 2};
  cuuint32_t box[2] = {64, box_rows};
  cuuint32_t step[2] = {1, 1};
  const CUresult r = fn(m, tma_dtype(a.in_dtype), 2, const_cast<void*>(a.A), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(SF_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d): rows of A {%d, %lld}, lda %lld",
                static_cast<int>(r), a.K, (long long)a.a_rows, (long long)a.lda);
  return SF_OK;
}

template <class Cfg>
int32_t launch_tc(const GroupedArgs& a, const DeviceInfo& dev, int device, cudaStream_t s) {
  const int64_t n_tiles = ceil_div(a.N, 128);
  const int64_t most = (ceil_div(a.M, Cfg::BN) + std::min(a.groups, a.M)) * n_tiles;
  if (most > INT32_MAX) return fail(SF_ERR_UNSUPPORTED, "%lld tiles exceed 2^31-1", (long long)most);
  const int64_t wide = Cfg::GATE ? 2LL * a.N : a.N;
  MapSpec w{a.B, 2, tma_dtype(a.in_dtype), static_cast<uint64_t>(a.K), static_cast<uint64_t>(wide),
            static_cast<uint64_t>(a.groups), 1, a.ldb, a.b_stride, 0, 64, 128};
  CUtensorMap mw, mx;
  int32_t st = encode_map(&mw, w);
  if (st == SF_OK) st = encode_rows(&mx, a, a.rows ? 1 : Cfg::BOX);
  if (st != SF_OK) return st;
  // The groups' first rows and tiles follow the ring.
  const size_t smem = Cfg::RING_BYTES + 2 * (static_cast<size_t>(a.groups) + 1) * sizeof(int);
  static size_t allowed[64] = {0};
  if (device >= 64) return fail(SF_ERR_UNSUPPORTED, "device index %d", device);
  constexpr size_t kMost = Cfg::RING_BYTES + 2 * (kMaxGroups + 1) * sizeof(int);
  static_assert(kMost + 512 <= 227 * 1024, "shared memory budget");
  if (allowed[device] == 0) {
    SF_CUDA_TRY(cudaFuncSetAttribute(grouped_tc_kernel<Cfg>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(kMost)));
    allowed[device] = kMost;
  }
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(most, dev.sm_count));
  grouped_tc_kernel<Cfg><<<grid, Cfg::THREADS, smem, s>>>(mw, mx, a);
  SF_CUDA_TRY(cudaGetLastError());
  return SF_OK;
}

template <int FMT>
int32_t run_tc(const GroupedArgs& a, const DeviceInfo& dev, int device, cudaStream_t s) {
  const bool few = a.M <= 32LL * a.groups;
  if (a.act == kActSiluGate)
    return few ? launch_tc<GroupedCfg<32, 5, FMT, true>>(a, dev, device, s)
               : launch_tc<GroupedCfg<128, 4, FMT, true>>(a, dev, device, s);
  return few ? launch_tc<GroupedCfg<32, 9, FMT, false>>(a, dev, device, s)
             : launch_tc<GroupedCfg<256, 4, FMT, false>>(a, dev, device, s);
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
  int device = 0;
  const int32_t st = current_device_info(&dev, &device);
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool describable = in_dtype != kF32 && K > 0 && a_rows > 0 && aligned16(A) && aligned16(B) &&
                           bytes16(lda, 2) && bytes16(ldb, 2) && (groups == 1 || bytes16(b_stride, 2)) &&
                           b_stride >= 0;
  if (!describable) return run_simt(a, s);
  return in_dtype == kBF16 ? run_tc<1>(a, *dev, device, s) : run_tc<0>(a, *dev, device, s);
}
