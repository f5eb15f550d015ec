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
#include <atomic>

#include "common.h"
#include "grouped_simt.cuh"
#include "grouped_tc.cuh"
#include "tma_host.h"

namespace sf {
namespace {

constexpr int64_t kMaxGroups = 4096;
// Mean rows per group up to which the narrow tiles are used (64 columns, or 32
// of both halves).  Narrow / wide tiles, K = 2048, N = 1408, 64 experts: 66.5 /
// 71.3 us at 16 rows per group, 77.8 / 74.9 us at 28; gated 104 / 114 us at 12.5
// and 127 / 117 us at 28.
constexpr int64_t kFewRows = 16;

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

// Rows to gather from which they are copied into grouped order first, when
// there is a workspace.  In the kernel every weight block gathers its rows
// again through the load/store path, which costs 29 % over TMA boxes at 35552
// rows (K = 1920, N = 7680: 1198 against 910 us) and is worth one pass over
// the rows (45 us there) from about 2000 rows and 8 weight blocks on (3000
// rows: 87 against 77 + 5 us; 800 rows: 27 against 25 + 3).
constexpr int64_t kGatherFirstRows = 2048;
constexpr int64_t kGatherFirstCols = 1024;

bool gather_pays(int64_t groups, int64_t M, int64_t N) {
  return M >= kGatherFirstRows && M > kFewRows * groups && N >= kGatherFirstCols;
}

// Elements of a gathered row: K rounded up to 16 bytes.
int64_t gathered_ld(int64_t K) { return (K + 7) / 8 * 8; }

// out[i, :] = A[rows[i], :], zeros for an index outside A; a warp per row, 16
// bytes per lane and step (plain loads: the rows may have been written while
// this grid, launched early, already ran, which read-only loads exclude).  What
// lies past K in a row's last vector is copied along (it is inside the row of A,
// which starts on 16-byte boundaries) and not used.
__global__ void __launch_bounds__(256) gather_rows_kernel(const uint4* A, int64_t ld_vec, int64_t a_rows,
                                                          const int* rows, int M, int vecs, uint4* out) {
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  pdl_wait();
  for (int m = blockIdx.x * 8 + (threadIdx.x >> 5); m < M; m += gridDim.x * 8) {
    const int64_t r = rows[m];
    const bool in = r >= 0 && r < a_rows;
    const uint4* src = A + (in ? r * ld_vec : 0);
    uint4* dst = out + static_cast<int64_t>(m) * vecs;
    for (int v = lane; v < vecs; v += 128) {
      uint4 u[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        u[j] = in && v + 32 * j < vecs ? src[v + 32 * j] : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v + 32 * j < vecs) dst[v + 32 * j] = u[j];
    }
  }
}

int32_t gather_first(GroupedArgs& a, void* ws, const DeviceInfo& dev, cudaStream_t s) {
  const int vecs = static_cast<int>(gathered_ld(a.K) / 8);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(
      std::min<int64_t>(ceil_div(a.M, 8), dev.sm_count * 8LL)));
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  SF_CUDA_TRY(cudaLaunchKernelEx(&cfg, gather_rows_kernel, static_cast<const uint4*>(a.A), a.lda / 8,
                                 a.a_rows, a.rows, a.M, vecs, static_cast<uint4*>(ws)));
  a.A = ws;
  a.a_rows = a.M;
  a.lda = gathered_ld(a.K);
  a.rows = nullptr;
  return SF_OK;
}

// Most tiles that M rows in `groups` groups can make, whatever the offsets say.
int64_t most_tiles(const GroupedArgs& a, int bn) {
  return (a.M / bn + std::min(a.groups, a.M)) * ceil_div(a.N, 128);
}

template <class Cfg>
int32_t launch_tc(GroupedArgs a, const DeviceInfo& dev, int device, cudaStream_t s) {
  const int64_t most = most_tiles(a, Cfg::BN);
  if (most > INT32_MAX / 8) return fail(SF_ERR_UNSUPPORTED, "%lld tiles exceed 2^28", (long long)most);
  const int64_t wide = Cfg::GATE ? 2LL * a.N : a.N;
  MapSpec w{a.B, 2, tma_dtype(a.in_dtype), static_cast<uint64_t>(a.K), static_cast<uint64_t>(wide),
            static_cast<uint64_t>(a.groups), 1, a.ldb, a.b_stride, 0, 64, 128};
  CUtensorMap mw, mx;
  int32_t st = encode_map(&mw, w);
  if (st == SF_OK) st = encode_rows(&mx, a, Cfg::BOX);
  if (st != SF_OK) return st;
  if (device >= 64) return fail(SF_ERR_UNSUPPORTED, "device index %d", device);
  // The groups' first rows and tiles follow the ring.
  constexpr size_t kMost = Cfg::RING_BYTES + 2 * (kMaxGroups + 1) * sizeof(int);
  static_assert(kMost + 512 <= 227 * 1024, "shared memory budget");
  static std::atomic<bool> allowed[64];
  if (!allowed[device].load(std::memory_order_acquire)) {
    SF_CUDA_TRY(cudaFuncSetAttribute(grouped_tc_kernel<Cfg>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(kMost)));
    allowed[device].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(Cfg::SPLIT ? most * a.splits : std::min<int64_t>(most, dev.sm_count)));
  cfg.blockDim = dim3(Cfg::THREADS + (a.rows ? 32 * Cfg::GATHER_WARPS : 0));
  cfg.dynamicSmemBytes = Cfg::RING_BYTES + 2 * (static_cast<size_t>(a.groups) + 1) * sizeof(int);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(a.splits);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = Cfg::SPLIT ? 2 : 1;
  SF_CUDA_TRY(cudaLaunchKernelEx(&cfg, grouped_tc_kernel<Cfg>, mw, mx, a));
  return SF_OK;
}

// CTAs per tile: where the tiles leave SMs idle, a tile's k-blocks (four at
// least each) are shared by a cluster of 2, 4 or 8.  Clusters fill a GPC's SMs
// only in part, and one that has to wait costs more than it saves: measured at
// K = 7680, 16 tiles: 47 us alone, 28 / 17 / 22 us in clusters of 2 / 4 / 8;
// 4 tiles of K = 4096: 26, 17 / 11 / 8.5 us; 22 tiles of K = 2048: 15, 11 / 8.9
// / 14.5 us.
int pick_splits(const GroupedArgs& a, int bn, int sm_count) {
  const int64_t most = most_tiles(a, bn), kb = ceil_div(a.K, 64);
  int s = 1;
  while (s < 8 && most * s * 2 <= (s == 1 ? sm_count : s == 2 ? sm_count * 3 / 4 : sm_count / 3) &&
         kb >= s * 8)
    s *= 2;
  return s;
}

template <int FMT, bool GATE, int BN_FEW, int STAGES_FEW, int BN, int STAGES>
int32_t run_tc_sized(GroupedArgs a, const DeviceInfo& dev, int device, cudaStream_t s) {
  if (a.M > kFewRows * a.groups) return launch_tc<GroupedCfg<BN, STAGES, FMT, GATE>>(a, dev, device, s);
  a.splits = pick_splits(a, BN_FEW, dev.sm_count);
  return a.splits > 1 ? launch_tc<GroupedCfg<BN_FEW, STAGES_FEW, FMT, GATE, true>>(a, dev, device, s)
                      : launch_tc<GroupedCfg<BN_FEW, STAGES_FEW, FMT, GATE>>(a, dev, device, s);
}

template <int FMT>
int32_t run_tc(const GroupedArgs& a, const DeviceInfo& dev, int device, cudaStream_t s) {
  if (a.act == kActSiluGate) return run_tc_sized<FMT, true, 32, 5, 128, 4>(a, dev, device, s);
  return run_tc_sized<FMT, false, 64, 8, 256, 4>(a, dev, device, s);
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" int32_t sf_gemm_grouped(int64_t groups, int64_t M, int64_t N, int64_t K, const void* A,
                                   int64_t a_rows, int64_t lda, const int32_t* rows,
                                   const int32_t* offsets, const void* B, int64_t ldb,
                                   int64_t b_stride, const void* bias, int32_t bias_dtype,
                                   int64_t bias_stride, void* C, int64_t ldc, int32_t in_dtype,
                                   int32_t out_dtype, int32_t activation, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  if (groups < 0 || M < 0 || N < 0 || K < 0 || a_rows < 0)
    return fail(SF_ERR_INVALID_ARGUMENT, "negative dimension");
  if (activation < SF_ACT_NONE || activation > SF_ACT_SILU_GATE)
    return fail(SF_ERR_INVALID_ARGUMENT, "unknown activation %d", activation);
  for (int dt : {in_dtype, out_dtype})
    if (dt != kF32 && dt != kF16 && dt != kBF16)
      return fail(SF_ERR_INVALID_ARGUMENT, "unknown dtype %d", dt);
  if (groups == 0 || M == 0 || N == 0) return SF_OK;
  const int64_t wide = activation == SF_ACT_SILU_GATE ? 2 * N : N;
  // Row and column counts are rounded up to tiles in 32 bits.
  constexpr int64_t kMostRows = INT32_MAX - 4096;
  if (M > kMostRows || wide > kMostRows || K > kMostRows || a_rows > INT32_MAX)
    return fail(SF_ERR_UNSUPPORTED, "dimension exceeds 2^31-4097");
  if (groups > kMaxGroups)
    return fail(SF_ERR_UNSUPPORTED, "%lld groups (at most %lld)", (long long)groups, (long long)kMaxGroups);
  if (!offsets || !C || (K > 0 && (!A || !B))) return fail(SF_ERR_INVALID_ARGUMENT, "null pointer");
  if (!rows && a_rows < M)
    return fail(SF_ERR_INVALID_ARGUMENT, "A has %lld rows, %lld needed", (long long)a_rows, (long long)M);
  if (ldc < N || lda < K || ldb < K) return fail(SF_ERR_INVALID_ARGUMENT, "leading dimension too small");
  if (b_stride < 0 || bias_stride < 0) return fail(SF_ERR_INVALID_ARGUMENT, "negative group stride");
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
                           bytes16(lda, 2) && bytes16(ldb, 2) &&
                           (groups == 1 || (b_stride > 0 && bytes16(b_stride, 2)));
  if (!describable) return run_simt(a, s);
  const size_t gathered = static_cast<size_t>(M) * static_cast<size_t>(gathered_ld(K)) * 2;
  if (rows && gather_pays(groups, M, N) && workspace && aligned16(workspace) && workspace_bytes >= gathered) {
    const int32_t st2 = gather_first(a, workspace, *dev, s);
    if (st2 != SF_OK) return st2;
  }
  return in_dtype == kBF16 ? run_tc<1>(a, *dev, device, s) : run_tc<0>(a, *dev, device, s);
}

extern "C" int32_t sf_gemm_grouped_workspace_size(int64_t groups, int64_t M, int64_t N, int64_t K,
                                                  int32_t in_dtype, void* stream, size_t* bytes) {
  if (!bytes) return fail(SF_ERR_INVALID_ARGUMENT, "null output");
  *bytes = 0;
  if (groups < 0 || M < 0 || N < 0 || K < 0) return fail(SF_ERR_INVALID_ARGUMENT, "negative dimension");
  if (in_dtype == kF32 || K == 0 || !gather_pays(groups, M, N)) return SF_OK;
  int32_t capturing = 0;
  const int32_t st = sf_stream_is_capturing(stream, &capturing);
  if (st != SF_OK) return st;
  if (!capturing)
    *bytes = static_cast<size_t>(M) * static_cast<size_t>(gathered_ld(K)) * 2;
  return SF_OK;
}
