// Linears with 4-bit weights and group scales.
//
//   y[m, n] = act(sum_k x[m, k] W[n, k] + bias[n]),
//   W[n, k] = scale[k / g, n] * (q[n, k] - zero[k / g, n]),  q in 0..15,
//
// zero = 8 where none is stored, else the whole number in 0..15 nearest to the
// stored value.  q, zero and their difference are exact in 16 bits, the scale
// stays out of the products: a group's sum of x * (q - zero) is formed in fp32
// and scaled once.
//
// Layout of q: row n is a run of 32-bit words, 16 per block of 128 columns
// (K is padded to whole blocks; what the padding holds is not used).  Nibble i
// of word 4 t + w of a block holds column
//   32 w + 8 t + (0, 2, 4, 6, 1, 3, 5, 7)[i].
// Scales and zeros are [K / g, N], so that neighbouring rows' are contiguous.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <utility>

#include "common.h"
#include "tma_host.h"
#include "w4_stream.cuh"
#include "w4_tc.cuh"

namespace sf {
namespace {

// A launch in clusters of `splits` CTAs with programmatic stream serialisation.
template <class Kernel, class... Args>
int32_t launch_cluster(Kernel kernel, int64_t grid, int threads, size_t smem, int splits, cudaStream_t s,
                       Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(splits);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  SF_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...));
  return SF_OK;
}

// The opt-in to a kernel's dynamic shared memory, once per device.
template <class Kernel>
int32_t allow_smem(Kernel kernel, int bytes, int device, std::atomic<bool> (&allowed)[64]) {
  if (device >= 64) return fail(SF_ERR_UNSUPPORTED, "device index %d", device);
  if (!allowed[device].load(std::memory_order_acquire)) {
    SF_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    allowed[device].store(true, std::memory_order_release);
  }
  return SF_OK;
}

// ───────────────────────── ring kernel ─────────────────────────
// Up to 16 rows of x, any layout: the unpacking and the fragments of
// w4_stream.cuh with less around them.  A warp owns 32 weight rows and every
// WK-th block of them, and copies its lanes' words and x itself (16 bytes per
// cp.async, kW4Stages blocks ahead); scales are loaded two blocks ahead, one row
// per lane.  The WK partial sums of a row meet in shared memory, in warp order.
// More than 16 rows of x run in passes of 16.

constexpr int kW4Rows = 32;   // weight rows of a warp
constexpr int kW4Stages = 3;  // blocks in flight per warp

// Eight columns of x at p, of which `left` lie before K; 0 past them.
__device__ __forceinline__ uint4 load_x8_ragged(const uint16_t* p, int left) {
  uint4 v = make_uint4(0, 0, 0, 0);
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < left) w[i >> 1] |= static_cast<uint32_t>(p[i]) << (16 * (i & 1));
  return v;
}

__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// Zeros instead of the 16 bytes when !in (nothing is read then).
__device__ __forceinline__ void copy_async16_if(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// GW: 32-column words per group (1, 2, 4).
template <bool BF16, int NT, int GW, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, NT == 1 && WARPS == 8 ? 2 : 1) w4_mma_kernel(const W4Args a, int wk, int x_vec) {
  constexpr int NG = 4 / GW;             // groups per block
  constexpr int NA = w4_accumulators(NT, GW);
  constexpr int kSlot = (4 + 4 * NT) * 32;  // 16-byte vectors per block: a lane's words and x
  // Each lane's own words and x, kW4Stages blocks ahead: a lane reads back only
  // what it copied itself, so its own wait on the copies is all the order needed.
  extern __shared__ __align__(16) uint8_t sm[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int kw = warp % wk, per_cta = (blockDim.x >> 5) / wk;
  const int n0 = (blockIdx.x * per_cta + warp / wk) * kW4Rows;
  const int blocks = (a.K + 127) / 128, groups = (a.K + 32 * GW - 1) / (32 * GW);
  const int mine = n0 < a.N ? (blocks - kw + wk - 1) / wk : 0;  // blocks kw, kw + wk, ...
  uint4* const ring = reinterpret_cast<uint4*>(sm) + warp * (kW4Stages * kSlot) + lane;
  const uint32_t ring_s = smem_u32(ring);

  float acc[2][NT][4] = {};
  // rows past N read row N - 1 and are not stored; tokens past M are not
  // copied (their columns of the products are not stored either)
  const uint4* src[4];  // rows n0 + 8 j + g
#pragma unroll
  for (int j = 0; j < 4; ++j)
    src[j] = reinterpret_cast<const uint4*>(a.packed + min(n0 + 8 * j + g, a.N - 1) * a.ldp) + t + 4 * kw;
  const uint16_t* xp = static_cast<const uint16_t*>(a.x) + g * a.ldx + 128 * kw + 8 * t;
  int left = a.K - (128 * kw + 8 * t);  // columns from xp to the row's end
  // scales and zeros of row n0 + lane, shared out by shuffles
  const uint16_t* sp = static_cast<const uint16_t*>(a.scales) + min(n0 + lane, a.N - 1);
  const uint16_t* zp = static_cast<const uint16_t*>(a.zeros) + min(n0 + lane, a.N - 1);
  const bool zeros = a.zeros != nullptr;

  int copied = 0;
  auto copy_block = [&](int slot) {
    if (copied < mine) {
      const uint32_t dst = ring_s + slot * kSlot * 16;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        copy_async16(dst + j * 32 * 16, src[j]);
        src[j] += 4 * wk;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
        if (8 * n + g < a.M) {
          const uint16_t* p = xp + 8 * n * a.ldx;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            if (x_vec)
              copy_async16_if(dst + (4 + 4 * n + w) * 32 * 16, 32 * w < left ? p + 32 * w : p, 32 * w < left);
            else
              ring[slot * kSlot + (4 + 4 * n + w) * 32] = load_x8_ragged(p + 32 * w, left - 32 * w);
          }
        }
      xp += 128 * wk;
      left -= 128 * wk;
    }
    ++copied;
    copy_async_commit();
  };
  int scaled = 0;
  uint32_t sc[3][NG], ze[3][NG];  // two blocks ahead
  auto load_scales = [&](int to) {
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      const int64_t at = min((kw + scaled * wk) * NG + j, groups - 1) * a.lds;  // past the last group: not used
      sc[to][j] = load_ahead(sp + at);
      if (zeros) ze[to][j] = load_ahead(zp + at);
    }
    ++scaled;
  };
  pdl_launch_dependents();
  pdl_wait();
  load_scales(0);
  load_scales(1);
  for (int i = 0; i < kW4Stages - 1; ++i) copy_block(i);
#pragma unroll 1
  for (int i0 = 0; i0 < mine; i0 += kW4Stages) {
#pragma unroll
    for (int u = 0; u < kW4Stages; ++u) {
      if (i0 + u >= mine) break;
      copy_block((u + kW4Stages - 1) % kW4Stages);
      uint32_t sv[NG];
#pragma unroll
      for (int j = 0; j < NG; ++j)
        sv[j] = pack_scale<BF16>((kw + (i0 + u) * wk) * NG + j < groups ? sc[u][j] : 0u, ze[u][j], zeros);
      load_scales((u + 2) % 3);
      copy_async_wait<kW4Stages - 1>();
      uint4 q[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = ring[u * kSlot + j * 32];
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        float s[4];
        uint2 z[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) unpack_scale<BF16>(__shfl_sync(0xffffffffu, sv[j], 8 * r + g), s[r], z[r]);
        float sum[2][NT][NA][4] = {};
#pragma unroll
        for (int l = 0; l < GW; ++l) {
          const int w = j * GW + l;
          uint32_t p[4][4];
#pragma unroll
          for (int r = 0; r < 4; ++r)
            unpack_word<BF16>(w == 0 ? q[r].x : w == 1 ? q[r].y : w == 2 ? q[r].z : q[r].w, z[r], p[r]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 x = ring[u * kSlot + (4 + 4 * n + w) * 32];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const uint32_t a0[4] = {p[2 * r][0], p[2 * r + 1][0], p[2 * r][1], p[2 * r + 1][1]};
              const uint32_t a1[4] = {p[2 * r][2], p[2 * r + 1][2], p[2 * r][3], p[2 * r + 1][3]};
              mma_16816<BF16>(sum[r][n][2 * l % NA], a0, x.x, x.y);
              mma_16816<BF16>(sum[r][n][2 * l % NA + 1], a1, x.z, x.w);
            }
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              acc[r][n][c] = fmaf(s[2 * r + (c >> 1)], sum_of<NA>(sum[r][n], c), acc[r][n][c]);
      }
    }
  }
  copy_async_wait<0>();
  __syncthreads();  // every warp is done with its ring: the sums take its place
  // [token][row] of this warp: acc c is row g + 8 (c / 2), token 2 t + c % 2
  float* const red = reinterpret_cast<float*>(sm);
  float* const part = red + warp * kW4Rows * (8 * NT);
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        part[(8 * n + 2 * t + (c & 1)) * kW4Rows + 16 * r + g + 8 * (c >> 1)] = acc[r][n][c];
  __syncthreads();
  // token-major: consecutive threads store consecutive columns of y
  const int per_tile = kW4Rows * a.M;
  for (int i = threadIdx.x; i < per_tile * per_cta; i += blockDim.x) {
    const int tl = i / per_tile, e = i - tl * per_tile;
    const int m = e / kW4Rows, r = e % kW4Rows;
    const int n = (blockIdx.x * per_cta + tl) * kW4Rows + r;
    if (n >= a.N) continue;
    float v = 0.0f;
    for (int w = 0; w < wk; ++w) v += red[(tl * wk + w) * kW4Rows * (8 * NT) + e];
    if (a.bias) v += load_as_f32(a.bias, n, a.bias_dtype);
    v = a.fast_act ? act_apply_fast(v, a.act) : act_apply(v, a.act);
    store_from_f32(a.y, m * a.ldy + n, a.out_dtype, v);
  }
}

template <bool BF16, int NT, int GW, int WARPS>
int32_t launch_w4(const W4Args& a, bool x_vec, int device, cudaStream_t s) {
  // Warps along k: as many as there are blocks for, so that every row's
  // stream is spread over the CTA; the rest take further rows.
  const int64_t blocks = ceil_div(a.K, 128);
  int wk = 1;
  while (wk < WARPS && wk < blocks) wk *= 2;
  const int64_t rows = kW4Rows * (WARPS / wk);
  constexpr int smem =
      WARPS * std::max(kW4Stages * (4 + 4 * NT) * 32 * 16, kW4Rows * 8 * NT * static_cast<int>(sizeof(float)));
  static std::atomic<bool> allowed[64];
  const int32_t st = allow_smem(w4_mma_kernel<BF16, NT, GW, WARPS>, smem, device, allowed);
  if (st != SF_OK) return st;
  return launch_cluster(w4_mma_kernel<BF16, NT, GW, WARPS>, ceil_div(a.N, rows), 32 * WARPS, smem, 1, s, a, wk,
                        x_vec ? 1 : 0);
}

// Sixteen warps per CTA where 32-row tiles are no more than the SMs: 4.4 against
// 6.5 us (1 x 4096 x 4096), 13 against 21 us (8 x 11008 -> 4096, groups of 32).
// With eight, two CTAs fit an SM, and the next launch's, which start early, then
// pair up on some SMs while others stay empty.
template <bool BF16, int NT>
int32_t launch_w4_group(const W4Args& a, bool x_vec, const DeviceInfo& dev, int device, cudaStream_t s) {
  if constexpr (NT == 1) {
    if (ceil_div(a.N, kW4Rows) <= dev.sm_count && a.K > 8 * 128) {
      if (a.group == 32) return launch_w4<BF16, NT, 1, 16>(a, x_vec, device, s);
      if (a.group == 64) return launch_w4<BF16, NT, 2, 16>(a, x_vec, device, s);
      return launch_w4<BF16, NT, 4, 16>(a, x_vec, device, s);
    }
  }
  if (a.group == 32) return launch_w4<BF16, NT, 1, 8>(a, x_vec, device, s);
  if (a.group == 64) return launch_w4<BF16, NT, 2, 8>(a, x_vec, device, s);
  return launch_w4<BF16, NT, 4, 8>(a, x_vec, device, s);
}

// ───────────────────────── tcgen05 kernel ─────────────────────────

int32_t encode(CUtensorMap* m, CUtensorMapDataType dt, const void* base, int rank, const cuuint64_t* dims,
               const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(SF_ERR_CUDA, "cuTensorMapEncodeTiled unavailable from the driver");
  const cuuint32_t step[3] = {1, 1, 1};
  const CUresult r = fn(m, dt, rank, const_cast<void*>(base), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(SF_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d): {%llu, %llu} rows of %llu bytes",
                static_cast<int>(r), (unsigned long long)dims[0], (unsigned long long)dims[1],
                (unsigned long long)strides[0]);
  return SF_OK;
}

// Packed words {16 per block, N}, boxes of one block of 128 rows.
int32_t encode_words(CUtensorMap* m, const W4Args& a, CUtensorMapSwizzle swizzle) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(ceil_div(a.K, 128) * 16), static_cast<cuuint64_t>(a.N)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(a.ldp) * 4};
  const cuuint32_t box[2] = {16, 128};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, a.packed, 2, dims, strides, box, swizzle);
}

// CTAs per 128 rows of the streaming kernel: the largest cluster with which all
// clusters run at once, since a second wave costs as much as the first.  The
// launch before this one leaves its places one by one, so a sixteenth is kept
// free.  8192 -> 11008, one row: 38.6 / 32.3 / 23.8 / 19.4 / 17.0 / 15.1 us in
// clusters of 1 to 6, 19.9 in 8 (two waves); 5120 -> 14336: 14.2 in 4, 16.8 in 5,
// which fill the device to the last place.  Where nothing fits, the fewest that
// are more than two per SM (8192 -> 28672, one row: 62.6 / 34.9 / 37.4 / 35.9 us
// for 1 / 2 / 3 / 4).  This is those fewest; 9 if 8 are not enough.
int least_stream_splits(int64_t tiles, int sm_count) {
  int s = 1;
  while (s <= 8 && tiles * s <= 2 * sm_count) ++s;
  return s;
}

// Blocks of 128 x 128 from which the streaming kernel is used.  Its clusters and
// its CTA-wide pipeline cost about 3 us more to start and to end than the ring
// kernel's, and it streams faster, with 9 to 16 rows by more.  Ring / stream,
// groups of 128, one row of x: 6.7 / 8.0 us at 4096 -> 8192 (2048 blocks), 9.8 /
// 10.2 us at 4096 -> 11008 (2752), 16.7 / 14.9 us at 4096 -> 22016 (5504), 38.6 /
// 34.5 us at 8192 -> 28672 (14336); 16 rows: 6.7 / 10.2 us at 4096 x 4096 (1024),
// 13.0 / 11.4, 18.7 / 15.1, 31.2 / 22.6, 68.9 / 51.3 us.  And it needs its CTAs: one
// row 13.0 / 19.0 us at 16384 -> 4096, where clusters of 8 are 256 of them.
constexpr int64_t kStreamBlocks = 4096, kStreamBlocks16 = 2048;

bool use_stream(const W4Args& a, int sm_count) {
  const int64_t tiles = ceil_div(a.N, 128);
  return least_stream_splits(tiles, sm_count) <= 8 &&
         tiles * ceil_div(a.K, 128) >= (a.M <= 8 ? kStreamBlocks : kStreamBlocks16);
}

// Clusters of 1 to 8 CTAs of a kernel that fit the device at once: how many CTAs
// an SM holds, and what packing whole clusters into its groups of SMs leaves over.
// Asked once per kernel and device.
template <class Kernel>
int32_t cluster_capacity(Kernel kernel, int threads, int smem, int device, std::atomic<int> (&known)[64][8],
                         int splits, int* out) {
  std::atomic<int>& entry = known[device][splits - 1];
  int n = entry.load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(splits));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(splits);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    SF_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
    entry.store(n, std::memory_order_relaxed);
  }
  *out = n;
  return SF_OK;
}

template <class Cfg>
int32_t launch_w4_stream(const W4Args& a, const DeviceInfo& dev, int device, cudaStream_t s) {
  CUtensorMap mw, mx;
  int32_t st = encode_words(&mw, a, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (st != SF_OK) return st;
  const cuuint64_t dims[3] = {32, static_cast<cuuint64_t>(a.M), static_cast<cuuint64_t>(a.K / 32)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(a.ldx) * 2, 64};
  const cuuint32_t box[3] = {32, 8 * Cfg::NT, 4};
  st = encode(&mx, tma_dtype(a.dtype), a.x, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (st != SF_OK) return st;
  const int64_t groups = ceil_div(a.K, 32 * Cfg::GW);
  const cuuint64_t sdims[2] = {static_cast<cuuint64_t>(a.N), static_cast<cuuint64_t>(groups)};
  const cuuint64_t sstrides[1] = {static_cast<cuuint64_t>(a.lds) * 2};
  const cuuint32_t sbox[2] = {128, Cfg::NG};
  CUtensorMap ms, mz;
  st = encode(&ms, tma_dtype(a.dtype), a.scales, 2, sdims, sstrides, sbox, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (st == SF_OK)
    st = encode(&mz, tma_dtype(a.dtype), a.zeros ? a.zeros : a.scales, 2, sdims, sstrides, sbox,
                CU_TENSOR_MAP_SWIZZLE_NONE);
  if (st != SF_OK) return st;
  static std::atomic<bool> allowed[64];
  st = allow_smem(w4_stream_kernel<Cfg>, Cfg::SMEM_BYTES, device, allowed);
  if (st != SF_OK) return st;
  static std::atomic<int> known[64][8];
  const int64_t tiles = ceil_div(a.N, 128);
  int splits = least_stream_splits(tiles, dev.sm_count);
  for (int c = 8; c > splits; --c) {
    int fit = 0;
    st = cluster_capacity(w4_stream_kernel<Cfg>, Cfg::THREADS, Cfg::SMEM_BYTES, device, known, c, &fit);
    if (st != SF_OK) return st;
    if (tiles * 16 <= static_cast<int64_t>(fit) * 15) {
      splits = c;
      break;
    }
  }
  return launch_cluster(w4_stream_kernel<Cfg>, ceil_div(a.N, 128) * splits, Cfg::THREADS, Cfg::SMEM_BYTES, splits, s,
                        mw, mx, ms, mz, a, splits, dev.err_word);
}

template <bool BF16, int NT>
int32_t launch_w4_stream_group(const W4Args& a, const DeviceInfo& dev, int device, cudaStream_t s) {
  if (a.group == 32) return launch_w4_stream<W4StreamCfg<BF16, NT, 1>>(a, dev, device, s);
  if (a.group == 64) return launch_w4_stream<W4StreamCfg<BF16, NT, 2>>(a, dev, device, s);
  return launch_w4_stream<W4StreamCfg<BF16, NT, 4>>(a, dev, device, s);
}

// CTAs per row tile, which share its blocks.  A block takes a CTA about as long
// next to another CTA as alone (it waits on its own MMAs), so what counts is the
// number of waves of two CTAs per SM times the blocks of a CTA, plus about four
// blocks' time for its start and end.  Measured, 64 rows of x: 4096 x 4096 34 /
// 23 / 14 / 11 us in clusters of 1 / 2 / 4 / 8; 4096 -> 11008 49 / 29 / 22 / 31 us
// in 1 / 2 / 3 / 4; 8192 -> 28672 75 / 80 / 85 / 101 us in 1 / 2 / 4 / 8.
int pick_w4_splits(const W4Args& a, int sm_count) {
  const int64_t tiles = ceil_div(a.N, 128), blocks = ceil_div(a.K, 128);
  int best = 1;
  int64_t least = INT64_MAX;
  for (int s = 1; s <= 8 && s <= blocks; ++s) {
    const int64_t cost = ceil_div(tiles * s, 2 * sm_count) * (ceil_div(blocks, s) + 4);
    if (cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}

template <class Cfg>
int32_t launch_w4_tc(const W4Args& a, const DeviceInfo& dev, int device, cudaStream_t s) {
  const int n_rows = (a.M + 15) / 16 * 16;
  CUtensorMap mw, mx;
  int32_t st = encode_words(&mw, a, CU_TENSOR_MAP_SWIZZLE_64B);
  if (st != SF_OK) return st;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.K), static_cast<cuuint64_t>(a.M)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(a.ldx) * 2};
  const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(n_rows)};
  st = encode(&mx, tma_dtype(a.dtype), a.x, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (st != SF_OK) return st;
  static std::atomic<bool> allowed[64];
  st = allow_smem(w4_tc_kernel<Cfg>, Cfg::SMEM_BYTES, device, allowed);
  if (st != SF_OK) return st;
  const int splits = pick_w4_splits(a, dev.sm_count);
  return launch_cluster(w4_tc_kernel<Cfg>, ceil_div(a.N, 128) * splits, Cfg::THREADS, Cfg::SMEM_BYTES, splits, s, mw,
                        mx, a, splits, n_rows, dev.err_word);
}

// Up to 16 rows of x run on mma.sync, more on tcgen05 (33 rows: 70 us at 8192 ->
// 28672, 213 in three passes of the ring kernel).  Rows of x that TMA cannot
// describe take the ring kernel.
template <bool BF16>
int32_t run_w4(const W4Args& a, cudaStream_t s) {
  const bool described = a.ldx % 8 == 0 && aligned16(a.x);
  DeviceInfo* dev = nullptr;
  int device = 0;
  int32_t st = current_device_info(&dev, &device);
  if (st != SF_OK) return st;
  if (described && a.M <= 16 && a.K % 32 == 0 && a.lds % 8 == 0 && aligned16(a.scales) && aligned16(a.zeros) &&
      use_stream(a, dev->sm_count))
    return a.M <= 8 ? launch_w4_stream_group<BF16, 1>(a, *dev, device, s)
                    : launch_w4_stream_group<BF16, 2>(a, *dev, device, s);
  if (described && a.M > 16) {
    if (a.group == 32) return launch_w4_tc<W4TcCfg<BF16, 1>>(a, *dev, device, s);
    if (a.group == 64) return launch_w4_tc<W4TcCfg<BF16, 2>>(a, *dev, device, s);
    return launch_w4_tc<W4TcCfg<BF16, 4>>(a, *dev, device, s);
  }
  const bool x_vec = a.K % 8 == 0 && described;
  if (a.M <= 8) return launch_w4_group<BF16, 1>(a, x_vec, *dev, device, s);
  W4Args p = a;
  for (int m0 = 0; m0 < a.M; m0 += 16) {
    p.M = std::min(16, a.M - m0);
    p.x = static_cast<const uint16_t*>(a.x) + m0 * a.ldx;
    p.y = static_cast<char*>(a.y) + m0 * a.ldy * esize(a.out_dtype);
    st = launch_w4_group<BF16, 2>(p, x_vec, *dev, device, s);
    if (st != SF_OK) return st;
  }
  return SF_OK;
}

// Quantisation of one group of one row per warp-quarter is not worth a tuned
// kernel (it runs once, at load): one thread per (row, group).
//   symmetric:  s = max |w| / 7 rounded to the stored type, q = rint(w / s) + 8
//   with zeros: s = (max - min) / 15 rounded likewise, z = rint(-min / s),
//               q = rint(w / s) + z; max and min taken with 0 included, so
//               that z lies in 0..15 and a weight of 0 is kept exactly
// q clamped to 0..15; s = 0 (an all-zero group) stores q = z.  A group with a
// NaN or an infinity, which no q stands for, has a scale of NaN.
__global__ void __launch_bounds__(128) w4_quantize_kernel(int N, int K, const void* W, int w_dtype,
                                                          int64_t ldw, int group, uint8_t* q8,
                                                          int64_t ld8, void* scales, void* zeros,
                                                          int64_t lds, int s_dtype) {
  const int64_t groups = (K + group - 1) / group;
  const int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
  if (i >= groups * N) return;
  const int n = static_cast<int>(i / groups), g = static_cast<int>(i - n * groups);
  const int k0 = g * group, k1 = min(K, k0 + group);
  float lo = 0.0f, hi = 0.0f;
  bool finite = true;
  for (int k = k0; k < k1; ++k) {
    const float w = load_as_f32(W, n * ldw + k, w_dtype);
    finite = finite && fabsf(w) < INFINITY;
    lo = fminf(lo, w);
    hi = fmaxf(hi, w);
  }
  store_from_f32(scales, g * lds + n, s_dtype,
                 !finite ? NAN : zeros ? (hi - lo) / 15.0f : fmaxf(hi, -lo) / 7.0f);
  const float s = load_as_f32(scales, g * lds + n, s_dtype);
  float z = 8.0f;
  if (zeros) {
    z = s > 0.0f ? fminf(fmaxf(rintf(-lo / s), 0.0f), 15.0f) : 0.0f;
    store_from_f32(zeros, g * lds + n, s_dtype, z);
  }
  for (int k = k0; k < k1; ++k) {
    const float w = load_as_f32(W, n * ldw + k, w_dtype);
    const float q = s > 0.0f ? fminf(fmaxf(rintf(w / s) + z, 0.0f), 15.0f) : z;
    // byte of the pair's word; two nibbles of one byte hold columns of the
    // same 8-column run, hence of the same group and the same thread
    const int c = k & 127, run = c & 7;
    const int word = 4 * ((c >> 3) & 3) + (c >> 5);
    const int nib = (run & 1) ? 4 + (run >> 1) : run >> 1;
    uint8_t* b = q8 + n * ld8 + static_cast<int64_t>(k >> 7) * 64 + word * 4 + (nib >> 1);
    const uint8_t v = static_cast<uint8_t>(q);
    *b = (nib & 1) ? static_cast<uint8_t>((*b & 0x0F) | (v << 4)) : static_cast<uint8_t>((*b & 0xF0) | v);
  }
}

__global__ void __launch_bounds__(256) w4_dequantize_kernel(int N, int K, const uint32_t* packed,
                                                            int64_t ldp, const void* scales,
                                                            const void* zeros, int64_t lds, int group,
                                                            int s_dtype, void* W, int w_dtype, int64_t ldw) {
  const int64_t words = (static_cast<int64_t>(K) + 127) / 128 * 16;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < words * N;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t n = i / words;
    const int wd = static_cast<int>(i - n * words);
    const uint32_t q = packed[n * ldp + wd];
    const int base = wd / 16 * 128;
    for (int j = 0; j < 8; ++j) {
      const int k = base + w4_column(wd & 15, j);
      if (k >= K) continue;
      const int64_t at = static_cast<int64_t>(k / group) * lds + n;
      const float z = zeros ? whole_zero(load_as_f32(zeros, at, s_dtype)) : 8.0f;
      store_from_f32(W, n * ldw + k, w_dtype,
                     load_as_f32(scales, at, s_dtype) * (static_cast<float>((q >> (4 * j)) & 15u) - z));
    }
  }
}

bool known_dtype(int dt) { return dt == kF32 || dt == kF16 || dt == kBF16; }

// The checks of a packed weight that the three entry points share.
int32_t check_w4(int64_t N, int64_t K, const void* packed, int64_t ldp, const void* scales,
                 int64_t lds, int32_t group) {
  if (N < 0 || K < 0) return fail(SF_ERR_INVALID_ARGUMENT, "negative dimension");
  // Row and column numbers are rounded up to tiles in 32 bits.
  constexpr int64_t kMost = INT32_MAX - 4096;
  if (N > kMost || K > kMost) return fail(SF_ERR_UNSUPPORTED, "dimension exceeds 2^31-4097");
  if (group != 32 && group != 64 && group != 128)
    return fail(SF_ERR_UNSUPPORTED, "group of %d columns (32, 64 or 128)", group);
  if (N == 0 || K == 0) return SF_OK;
  if (!packed || !scales) return fail(SF_ERR_INVALID_ARGUMENT, "null pointer");
  if (!aligned16(packed) || ldp % 4 != 0)
    return fail(SF_ERR_INVALID_ARGUMENT, "packed rows must start on 16-byte boundaries");
  if (ldp < ceil_div(K, 128) * 16)
    return fail(SF_ERR_INVALID_ARGUMENT, "packed rows of %lld words, %lld needed", (long long)ldp,
                (long long)(ceil_div(K, 128) * 16));
  if (lds < N) return fail(SF_ERR_INVALID_ARGUMENT, "scale rows shorter than N");
  return SF_OK;
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" {

int32_t sf_linear_w4(int64_t M, int64_t N, int64_t K, const void* x, int64_t ldx,
                     const uint32_t* packed, int64_t ldp, const void* scales, const void* zeros,
                     int64_t lds, int32_t group, const void* bias, int32_t bias_dtype, void* y,
                     int64_t ldy, int32_t in_dtype, int32_t out_dtype, int32_t activation,
                     void* stream) {
  if (M < 0) return fail(SF_ERR_INVALID_ARGUMENT, "negative dimension");
  if (M > kW4MaxRows)
    return fail(SF_ERR_UNSUPPORTED, "%lld rows (at most %d; dequantise for more)", (long long)M, kW4MaxRows);
  int32_t st = check_w4(N, K, packed, ldp, scales, lds, group);
  if (st != SF_OK) return st;
  if (in_dtype != kF16 && in_dtype != kBF16)
    return fail(SF_ERR_UNSUPPORTED, "x of dtype %d (bf16 or fp16)", in_dtype);
  if (!known_dtype(out_dtype)) return fail(SF_ERR_INVALID_ARGUMENT, "unknown dtype %d", out_dtype);
  if (activation < SF_ACT_NONE || activation > SF_ACT_GELU_TANH)
    return fail(SF_ERR_INVALID_ARGUMENT, "unknown activation %d", activation);
  if (bias && !known_dtype(bias_dtype)) return fail(SF_ERR_INVALID_ARGUMENT, "unknown bias dtype");
  if (M == 0 || N == 0) return SF_OK;
  if (K == 0) return fail(SF_ERR_INVALID_ARGUMENT, "a 4-bit linear over no columns");
  if (!y || !x) return fail(SF_ERR_INVALID_ARGUMENT, "null pointer");
  if (ldx < K || ldy < N) return fail(SF_ERR_INVALID_ARGUMENT, "leading dimension too small");
  const W4Args a{static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), x, ldx, packed, ldp,
                 scales, zeros, lds, group, in_dtype, bias, bias_dtype, y, ldy, out_dtype, activation,
                 out_dtype != kF32 ? 1 : 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return in_dtype == kBF16 ? run_w4<true>(a, s) : run_w4<false>(a, s);
}

int32_t sf_quantize_w4(int64_t N, int64_t K, const void* W, int32_t w_dtype, int64_t ldw,
                       int32_t group, uint32_t* packed, int64_t ldp, void* scales, void* zeros,
                       int64_t lds, int32_t scale_dtype, void* stream) {
  int32_t st = check_w4(N, K, packed, ldp, scales, lds, group);
  if (st != SF_OK) return st;
  if (!known_dtype(w_dtype) || !known_dtype(scale_dtype))
    return fail(SF_ERR_INVALID_ARGUMENT, "unknown dtype");
  if (N == 0 || K == 0) return SF_OK;
  if (!W) return fail(SF_ERR_INVALID_ARGUMENT, "null pointer");
  if (ldw < K) return fail(SF_ERR_INVALID_ARGUMENT, "leading dimension too small");
  const int64_t work = ceil_div(K, group) * N;
  w4_quantize_kernel<<<static_cast<unsigned>(ceil_div(work, 128)), 128, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<int>(N), static_cast<int>(K), W, w_dtype, ldw, group,
      reinterpret_cast<uint8_t*>(packed), ldp * 4, scales, zeros, lds, scale_dtype);
  SF_CUDA_TRY(cudaGetLastError());
  return SF_OK;
}

int32_t sf_dequantize_w4(int64_t N, int64_t K, const uint32_t* packed, int64_t ldp,
                         const void* scales, const void* zeros, int64_t lds, int32_t group,
                         int32_t scale_dtype, void* W, int32_t w_dtype, int64_t ldw, void* stream) {
  int32_t st = check_w4(N, K, packed, ldp, scales, lds, group);
  if (st != SF_OK) return st;
  if (!known_dtype(w_dtype) || !known_dtype(scale_dtype))
    return fail(SF_ERR_INVALID_ARGUMENT, "unknown dtype");
  if (N == 0 || K == 0) return SF_OK;
  if (!W) return fail(SF_ERR_INVALID_ARGUMENT, "null pointer");
  if (ldw < K) return fail(SF_ERR_INVALID_ARGUMENT, "leading dimension too small");
  DeviceInfo* dev = nullptr;
  st = current_device_info(&dev, nullptr);
  if (st != SF_OK) return st;
  const int64_t work = ceil_div(K, 128) * 16 * N;
  w4_dequantize_kernel<<<static_cast<unsigned>(std::min<int64_t>(ceil_div(work, 256), dev->sm_count * 16LL)),
                         256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<int>(N), static_cast<int>(K), packed, ldp, scales, zeros, lds, group, scale_dtype, W,
      w_dtype, ldw);
  SF_CUDA_TRY(cudaGetLastError());
  return SF_OK;
}

}  // extern "C"
