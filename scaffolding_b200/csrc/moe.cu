// The two ends of a sparse (mixture-of-experts) layer: the router, which
// picks every token's experts and groups the choices by expert, and the
// combine, which sums a token's expert rows.  The products in between are
// grouped.cu.
//
// Router.  For token t with logits z (NaN counts as -inf, -0 as +0):
//   e_0 .. e_{k-1} = the experts of the k largest z, falling, ties to the
//                    lowest expert;
//   w_j = exp(z[e_j] - z[e_0]) / S,  S over the k picks (renormalize) or over
//         all experts; 0 for a pick of -inf, so a row without a finite or
//         +inf logit has weights 0.
// The T * k choices (t, j), in that order, are then sorted by expert with a
// stable counting sort: slot p in [offsets[e], offsets[e+1]) holds token
// rows[p], and slots[t, j] is the slot of choice (t, j).
//
// The work is a few comparisons per logit, so the router is bound by launch
// and reduction latency.  One warp per token: column lane + 32 i of the row in
// register i as an order-preserving integer, each pick one integer max and
// one integer min over the warp.  The sort counts per block of tokens, then a
// second kernel in which every block sums the counts in front of it (no
// serial scan kernel in between) and ranks its own choices; a batch of at
// most kSmallTokens tokens runs both halves in one block of one launch.
// Integer counts only: the result does not depend on the order of atomics.
#include <cuda_runtime.h>

#include <algorithm>

#include "common.h"
#include "epilogue.cuh"
#include "tma_host.h"

namespace sf {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 32;
constexpr int kSmallTokens = 256;
constexpr int kRouteThreads = 256;
constexpr int kSmallThreads = 1024;

struct RouteArgs {
  int tokens, experts, k;
  const void* logits;
  int dtype;
  int64_t ld;
  int renorm;
  int chunk;       // tokens per block
  int* experts_of; // [tokens][k]
  float* weights;  // [tokens][k]
  int* offsets;    // [experts + 1]
  int* rows;       // [tokens * k]
  int* slots;      // [tokens][k]
  int* counts;     // [blocks][experts]
};

// Order-preserving unsigned key of a float; 0 is below every key.
__device__ __forceinline__ uint32_t order_key(float z) {
  z = (z != z) ? -INFINITY : z + 0.0f;
  const uint32_t u = __float_as_uint(z);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
}

// exp(z - m) with m >= z: 0 for z = -inf, 1 for z = m (infinite m included).
__device__ __forceinline__ float exp_below(float z, float m) {
  return z == -INFINITY ? 0.0f : z == m ? 1.0f : expf(z - m);
}

// Picks of the tokens [t0, t1) by the block's warps, counted into hist.
template <int NV>
__device__ __forceinline__ void pick_experts(const RouteArgs& a, int t0, int t1, int* hist) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  for (int t = t0 + warp; t < t1; t += warps) {
    const int64_t base = static_cast<int64_t>(t) * a.ld;
    uint32_t key[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = lane + 32 * i;
      key[i] = c < a.experts ? order_key(load_as_f32(a.logits, base + c, a.dtype)) : 0u;
    }
    float all[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) all[i] = key_value(key[i]);
    uint32_t my_key = 0;
    int my_expert = 0;
    for (int j = 0; j < a.k; ++j) {
      uint32_t best = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) best = max(best, key[i]);
      best = __reduce_max_sync(0xffffffffu, best);
      int at = INT_MAX;
#pragma unroll
      for (int i = NV - 1; i >= 0; --i)
        if (key[i] == best) at = lane + 32 * i;
      at = __reduce_min_sync(0xffffffffu, at);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (at == lane + 32 * i) key[i] = 0u;
      if (lane == j) {
        my_key = best;
        my_expert = at;
      }
    }
    const float top = key_value(__shfl_sync(0xffffffffu, my_key, 0));
    const float e = lane < a.k ? exp_below(key_value(my_key), top) : 0.0f;
    float s = e;
    if (!a.renorm) {
      s = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (lane + 32 * i < a.experts) s += exp_below(all[i], top);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane < a.k) {
      const int64_t p = static_cast<int64_t>(t) * a.k + lane;
      a.experts_of[p] = my_expert;
      a.weights[p] = s > 0.0f ? e / s : 0.0f;
      atomicAdd(&hist[my_expert], 1);
    }
  }
}

__device__ __forceinline__ void pick_experts_any(const RouteArgs& a, int t0, int t1, int* hist) {
  if (a.experts <= 32) pick_experts<1>(a, t0, t1, hist);
  else if (a.experts <= 64) pick_experts<2>(a, t0, t1, hist);
  else if (a.experts <= 128) pick_experts<4>(a, t0, t1, hist);
  else if (a.experts <= 256) pick_experts<8>(a, t0, t1, hist);
  else pick_experts<32>(a, t0, t1, hist);
}

// first[e] += the sum of total[0 .. e), by warp 0; writes offsets when asked.
__device__ __forceinline__ void add_expert_starts(const RouteArgs& a, const int* total, int* first,
                                                  bool write) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int carry = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      const int e = e0 + lane;
      const int v = e < a.experts ? total[e] : 0;
      int s = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += n;
      }
      if (e < a.experts) {
        first[e] += carry + s - v;
        if (write) a.offsets[e] = carry + s - v;
      }
      carry += __shfl_sync(0xffffffffu, s, 31);
    }
    if (write && lane == 0) a.offsets[a.experts] = carry;
  }
}

// Ranks the choices of the tokens [t0, t1): slot = first[e] + the number of
// earlier choices of e in the block.  Warp w takes a contiguous run of the
// choices; mine[w][e] counts, then becomes the start of, its choices of e.
__device__ __forceinline__ void place_choices(const RouteArgs& a, int t0, int t1, const int* first,
                                              int* mine) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int64_t c0 = static_cast<int64_t>(t0) * a.k;
  const int n = (t1 - t0) * a.k;
  const int per = ((n + warps - 1) / warps + 31) / 32 * 32;
  const int lo = min(n, warp * per), hi = min(n, lo + per);
  for (int i = threadIdx.x; i < warps * a.experts; i += blockDim.x) mine[i] = 0;
  __syncthreads();
  for (int i = lo + lane; i < hi; i += 32) atomicAdd(&mine[warp * a.experts + a.experts_of[c0 + i]], 1);
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
    int s = first[e];
    for (int w = 0; w < warps; ++w) {
      const int v = mine[w * a.experts + e];
      mine[w * a.experts + e] = s;
      s += v;
    }
  }
  __syncthreads();
  for (int i0 = lo; i0 < hi; i0 += 32) {
    const int i = i0 + lane;
    const bool live = i < hi;
    const int e = live ? a.experts_of[c0 + i] : -1 - lane;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int before = __popc(same & ((1u << lane) - 1u));
    int start = 0;
    if (live) start = mine[warp * a.experts + e];
    __syncwarp();
    if (live) {
      if (before == 0) mine[warp * a.experts + e] = start + __popc(same);
      const int slot = start + before;
      a.slots[c0 + i] = slot;
      a.rows[slot] = static_cast<int>((c0 + i) / a.k);
    }
    __syncwarp();
  }
}

__global__ void __launch_bounds__(kSmallThreads) route_small_kernel(const RouteArgs a) {
  extern __shared__ int sm[];
  int* total = sm;                // [experts]
  int* first = sm + a.experts;    // [experts]
  int* mine = sm + 2 * a.experts; // [warps][experts]
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) total[e] = first[e] = 0;
  __syncthreads();
  pick_experts_any(a, 0, a.tokens, total);
  __syncthreads();
  add_expert_starts(a, total, first, true);
  __syncthreads();
  place_choices(a, 0, a.tokens, first, mine);
}

__global__ void __launch_bounds__(kRouteThreads) route_pick_kernel(const RouteArgs a) {
  extern __shared__ int sm[];
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) sm[e] = 0;
  __syncthreads();
  const int t0 = blockIdx.x * a.chunk, t1 = min(a.tokens, t0 + a.chunk);
  pick_experts_any(a, t0, t1, sm);
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x)
    a.counts[static_cast<int64_t>(blockIdx.x) * a.experts + e] = sm[e];
}

__global__ void __launch_bounds__(kRouteThreads) route_place_kernel(const RouteArgs a) {
  extern __shared__ int sm[];
  int* total = sm;
  int* first = sm + a.experts;
  int* mine = sm + 2 * a.experts;
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) total[e] = first[e] = 0;
  __syncthreads();
  // Counts of all blocks, and of those in front of this one.
  const int across = min(a.experts, static_cast<int>(blockDim.x));
  const int parts = blockDim.x / across, part = threadIdx.x / across;
  if (part < parts)
    for (int e = threadIdx.x - part * across; e < a.experts; e += across) {
      int all = 0, front = 0;
      for (int b = part; b < static_cast<int>(gridDim.x); b += parts) {
        const int v = a.counts[static_cast<int64_t>(b) * a.experts + e];
        all += v;
        if (b < static_cast<int>(blockIdx.x)) front += v;
      }
      atomicAdd(&total[e], all);
      atomicAdd(&first[e], front);
    }
  __syncthreads();
  add_expert_starts(a, total, first, blockIdx.x == 0);
  __syncthreads();
  const int t0 = blockIdx.x * a.chunk, t1 = min(a.tokens, t0 + a.chunk);
  place_choices(a, t0, t1, first, mine);
}

// Tokens per block: at most 256 blocks, since every block of the second
// kernel reads every block's counts.
int route_chunk(int64_t tokens) {
  return static_cast<int>(std::max<int64_t>(128, ceil_div(tokens, 256)));
}

// ───────────────────────────── combine ─────────────────────────────
//
//   o[t, :] = residual[t, :] + sum_j weights[t, j] * y[slots[t, j], :]
//
// in fp32, j rising, one rounding at the end.  A slot outside [0, y_rows)
// adds nothing.  Bound by HBM: every expert row is read once (the slots of
// all choices are a permutation) and every output row written once, so each
// thread owns 16 bytes of an output row and has the loads of all k expert
// rows in flight.

struct CombineArgs {
  int64_t tokens;
  int cols, k;
  const void* y;
  int64_t y_rows, ldy;
  int dtype;
  const int* slots;
  const float* weights;
  const void* residual;
  int64_t ldr;
  void* out;
  int64_t ldo;
};

__global__ void __launch_bounds__(256) combine_kernel(const CombineArgs a) {
  const int64_t total = a.tokens * a.cols;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t t = i / a.cols;
    const int c = static_cast<int>(i - t * a.cols);
    float acc = a.residual ? load_as_f32(a.residual, t * a.ldr + c, a.dtype) : 0.0f;
    for (int j = 0; j < a.k; ++j) {
      const int64_t s = a.slots[t * a.k + j];
      if (s >= 0 && s < a.y_rows)
        acc = fmaf(a.weights[t * a.k + j], load_as_f32(a.y, s * a.ldy + c, a.dtype), acc);
    }
    store_from_f32(a.out, t * a.ldo + c, a.dtype, acc);
  }
}

bool known_dtype(int dt) { return dt == kF32 || dt == kF16 || dt == kBF16; }

int32_t check_route(int64_t tokens, int64_t experts, int32_t top_k) {
  if (tokens < 0) return fail(SF_ERR_INVALID_ARGUMENT, "negative token count");
  if (experts < 1 || top_k < 1 || top_k > experts)
    return fail(SF_ERR_INVALID_ARGUMENT, "top_k %d of %lld experts", top_k, (long long)experts);
  if (experts > kMaxExperts || top_k > kMaxTopK)
    return fail(SF_ERR_UNSUPPORTED, "top_k %d of %lld experts (at most %d of %d)", top_k,
                (long long)experts, kMaxTopK, kMaxExperts);
  if (tokens > INT32_MAX / top_k)
    return fail(SF_ERR_UNSUPPORTED, "%lld tokens with %d choices exceed 2^31-1 slots",
                (long long)tokens, top_k);
  return SF_OK;
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" int32_t sf_moe_route_workspace_size(int64_t tokens, int64_t experts, int32_t top_k,
                                               size_t* bytes) {
  if (!bytes) return fail(SF_ERR_INVALID_ARGUMENT, "null output");
  *bytes = 0;
  const int32_t st = check_route(tokens, experts, top_k);
  if (st != SF_OK) return st;
  if (tokens > kSmallTokens)
    *bytes = static_cast<size_t>(ceil_div(tokens, route_chunk(tokens))) * experts * sizeof(int);
  return SF_OK;
}

extern "C" int32_t sf_moe_route(int64_t tokens, int64_t experts, int32_t top_k, const void* logits,
                                int32_t dtype, int64_t ld, int32_t renormalize,
                                int32_t* expert_ids, float* weights, int32_t* offsets,
                                int32_t* rows, int32_t* slots, void* workspace,
                                size_t workspace_bytes, void* stream) {
  size_t need = 0;
  int32_t st = sf_moe_route_workspace_size(tokens, experts, top_k, &need);
  if (st != SF_OK) return st;
  if (!known_dtype(dtype)) return fail(SF_ERR_INVALID_ARGUMENT, "dtype %d", dtype);
  if (ld < experts) return fail(SF_ERR_INVALID_ARGUMENT, "leading dimension < experts");
  if (!offsets || (tokens > 0 && (!logits || !expert_ids || !weights || !rows || !slots)))
    return fail(SF_ERR_INVALID_ARGUMENT, "null pointer");
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(SF_ERR_WORKSPACE, "workspace of %zu bytes required (%zu given)", need,
                workspace ? workspace_bytes : size_t(0));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  RouteArgs a{static_cast<int>(tokens), static_cast<int>(experts), top_k, logits, dtype, ld,
              renormalize != 0, 0, expert_ids, weights, offsets, rows, slots,
              static_cast<int*>(workspace)};
  const size_t per_warp = static_cast<size_t>(experts) * sizeof(int);
  if (tokens <= kSmallTokens) {
    // One warp per token where 32 suffice; fewer warps keep the ranking short.
    const int warps = static_cast<int>(std::max<int64_t>(
        1, std::min<int64_t>({tokens, kSmallThreads / 32, (48 * 1024) / static_cast<int64_t>(per_warp) - 2})));
    a.chunk = static_cast<int>(tokens);
    route_small_kernel<<<1, warps * 32, per_warp * (2 + warps), s>>>(a);
  } else {
    a.chunk = route_chunk(tokens);
    const unsigned blocks = static_cast<unsigned>(ceil_div(tokens, a.chunk));
    route_pick_kernel<<<blocks, kRouteThreads, per_warp, s>>>(a);
    SF_CUDA_TRY(cudaGetLastError());
    route_place_kernel<<<blocks, kRouteThreads, per_warp * (2 + kRouteThreads / 32), s>>>(a);
  }
  SF_CUDA_TRY(cudaGetLastError());
  return SF_OK;
}

extern "C" int32_t sf_moe_combine(int64_t tokens, int64_t cols, int32_t top_k, const void* y,
                                  int64_t y_rows, int64_t ldy, int32_t dtype, const int32_t* slots,
                                  const float* weights, const void* residual, int64_t ldr,
                                  void* out, int64_t ldo, void* stream) {
  if (tokens < 0 || cols < 0 || y_rows < 0) return fail(SF_ERR_INVALID_ARGUMENT, "negative size");
  if (top_k < 1) return fail(SF_ERR_INVALID_ARGUMENT, "top_k %d", top_k);
  if (!known_dtype(dtype)) return fail(SF_ERR_INVALID_ARGUMENT, "dtype %d", dtype);
  if (tokens == 0 || cols == 0) return SF_OK;
  if (tokens > INT32_MAX || cols > INT32_MAX)
    return fail(SF_ERR_UNSUPPORTED, "dimension exceeds 2^31-1");
  if (!out || !slots || !weights || (y_rows > 0 && !y))
    return fail(SF_ERR_INVALID_ARGUMENT, "null pointer");
  if (ldy < cols || ldo < cols || (residual && ldr < cols))
    return fail(SF_ERR_INVALID_ARGUMENT, "leading dimension < cols");
  DeviceInfo* dev = nullptr;
  const int32_t st = current_device_info(&dev, nullptr);
  if (st != SF_OK) return st;
  const CombineArgs a{tokens, static_cast<int>(cols), top_k, y, y_rows, ldy, dtype, slots, weights,
                      residual, ldr, out, ldo};
  const unsigned grid = static_cast<unsigned>(
      std::min<int64_t>(ceil_div(tokens * cols, 256), dev->sm_count * 16LL));
  combine_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(a);
  SF_CUDA_TRY(cudaGetLastError());
  return SF_OK;
}
