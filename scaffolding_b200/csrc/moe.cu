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
// Measured: 4.8 us for 64 tokens of 64 experts (top 4), 13.1 us for 17776 (top
// 2), where the logits alone take 0.8 us of HBM time: the picks issue about 230
// instructions per token, some 4 us, and the rest is two dependent launches, in
// the second of which every block reads every block's counts.
// Integer counts only: the result does not depend on the order of atomics.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <utility>

#include "common.h"
#include "epilogue.cuh"
#include "ptx.cuh"
#include "tma_host.h"

namespace sf {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 32;
// Token and choice numbers are 32 bits.  What is added to one past the last
// (the end of a block's chunk, at most 2^22 tokens; a warp's stride) stays in
// range with this many.
constexpr int64_t kMostChoices = INT32_MAX - (1 << 23);
constexpr int kSmallTokens = 256;
constexpr int kRouteThreads = 512;
constexpr int kSmallThreads = 1024;

// Launch with programmatic stream serialisation: every kernel here waits for
// the previous grid (pdl_wait) before it reads or writes memory.
template <class... KArgs, class... Args>
int32_t launch_pdl(void (*kernel)(KArgs...), unsigned grid, unsigned block, size_t smem, cudaStream_t s,
                   Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  SF_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...));
  return SF_OK;
}

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

// Picks of the tokens [t0, t1) by the block's warps, counted into hist and,
// where given, left in picked[t - t0][k].  A warp works on TOK tokens at a time: the picks
// of one token are a chain of reductions, those of several overlap.
template <int NV, int TOK>
__device__ __forceinline__ void pick_experts(const RouteArgs& a, int t0, int t1, int* hist, uint16_t* picked) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  for (int tb = t0 + warp; tb < t1; tb += warps * TOK) {
    // All loads of the TOK tokens first (the branch on the type is outside).
    uint32_t key[TOK][NV];
    if (a.dtype == kF32) {
      const float* z = static_cast<const float*>(a.logits);
#pragma unroll
      for (int q = 0; q < TOK; ++q)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int t = tb + q * warps, c = lane + 32 * i;
          key[q][i] = t < t1 && c < a.experts ? __float_as_uint(z[static_cast<int64_t>(t) * a.ld + c]) : 0u;
        }
    } else {
      const uint16_t* z = static_cast<const uint16_t*>(a.logits);
#pragma unroll
      for (int q = 0; q < TOK; ++q)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int t = tb + q * warps, c = lane + 32 * i;
          key[q][i] = t < t1 && c < a.experts ? z[static_cast<int64_t>(t) * a.ld + c] : 0u;
        }
#pragma unroll
      for (int q = 0; q < TOK; ++q)
#pragma unroll
        for (int i = 0; i < NV; ++i)
          key[q][i] = a.dtype == kBF16
                          ? key[q][i] << 16
                          : __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(key[q][i]))));
    }
#pragma unroll
    for (int q = 0; q < TOK; ++q)
#pragma unroll
      for (int i = 0; i < NV; ++i)
        key[q][i] = lane + 32 * i < a.experts ? order_key(__uint_as_float(key[q][i])) : 0u;
    // Sum over all experts (relative to the largest logit) before the picks
    // take the keys away.
    float s[TOK];
#pragma unroll
    for (int q = 0; q < TOK; ++q) {
      s[q] = 0.0f;
      if (!a.renorm) {
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) best = max(best, key[q][i]);
        const float top = key_value(__reduce_max_sync(0xffffffffu, best));
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (lane + 32 * i < a.experts) s[q] += exp_below(key_value(key[q][i]), top);
      }
    }
    uint32_t my_key[TOK];
    int my_expert[TOK];
#pragma unroll
    for (int q = 0; q < TOK; ++q) my_key[q] = 0, my_expert[q] = 0;
    for (int j = 0; j < a.k; ++j) {
#pragma unroll
      for (int q = 0; q < TOK; ++q) {
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) best = max(best, key[q][i]);
        best = __reduce_max_sync(0xffffffffu, best);
        int at = INT_MAX;
#pragma unroll
        for (int i = NV - 1; i >= 0; --i)
          if (key[q][i] == best) at = lane + 32 * i;
        at = __reduce_min_sync(0xffffffffu, at);
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (at == lane + 32 * i) key[q][i] = 0u;
        if (lane == j) {
          my_key[q] = best;
          my_expert[q] = at;
        }
      }
    }
#pragma unroll
    for (int q = 0; q < TOK; ++q) {
      const int t = tb + q * warps;
      const float top = key_value(__shfl_sync(0xffffffffu, my_key[q], 0));
      const float e = lane < a.k ? exp_below(key_value(my_key[q]), top) : 0.0f;
      if (a.renorm) s[q] = e;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s[q] += __shfl_xor_sync(0xffffffffu, s[q], o);
      if (lane < a.k && t < t1) {
        const int64_t p = static_cast<int64_t>(t) * a.k + lane;
        a.experts_of[p] = my_expert[q];
        a.weights[p] = s[q] > 0.0f ? e / s[q] : 0.0f;
        if (picked) picked[(t - t0) * a.k + lane] = static_cast<uint16_t>(my_expert[q]);
        atomicAdd(&hist[my_expert[q]], 1);
      }
    }
  }
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

// Ranks the n choices of a block, the first of which is choice c0 of the batch:
// slot = first[e] + the number of earlier choices of e in the block.  Each of
// `warps` warps takes a contiguous run of them; mine[w][e] counts, then becomes
// the start of, its choices of e.  expert(i) is choice i's expert.
template <class Expert>
__device__ __forceinline__ void place_choices(const RouteArgs& a, int64_t c0, int n, const int* first,
                                              int* mine, int warps, Expert expert) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = ((n + warps - 1) / warps + 31) / 32 * 32;
  const int lo = warp < warps ? min(n, warp * per) : n, hi = min(n, lo + per);
  for (int i = threadIdx.x; i < warps * a.experts; i += blockDim.x) mine[i] = 0;
  __syncthreads();
  for (int i = lo + lane; i < hi; i += 32) atomicAdd(&mine[warp * a.experts + expert(i)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
    int s = first[e];
#pragma unroll 4
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
    const int e = live ? expert(i) : -1 - lane;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int before = __popc(same & ((1u << lane) - 1u));
    const int start = live ? mine[warp * a.experts + e] : 0;
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

// total[experts], first[experts], mine[warps][experts], picked[tokens * k].
template <int NV, int TOK>
__global__ void __launch_bounds__(kSmallThreads) route_small_kernel(const RouteArgs a, int place_warps) {
  extern __shared__ int sm[];
  int* total = sm;
  int* first = sm + a.experts;
  int* mine = sm + 2 * a.experts;
  uint16_t* picked = reinterpret_cast<uint16_t*>(mine + place_warps * a.experts);
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) total[e] = first[e] = 0;
  pdl_launch_dependents();
  pdl_wait();
  __syncthreads();
  pick_experts<NV, TOK>(a, 0, a.tokens, total, picked);
  __syncthreads();
  add_expert_starts(a, total, first, true);
  __syncthreads();
  place_choices(a, 0, a.tokens * a.k, first, mine, place_warps, [=](int i) { return static_cast<int>(picked[i]); });
}

template <int NV, int TOK>
__global__ void __launch_bounds__(kRouteThreads) route_pick_kernel(const RouteArgs a) {
  extern __shared__ int sm[];
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) sm[e] = 0;
  pdl_launch_dependents();
  pdl_wait();
  __syncthreads();
  const int t0 = blockIdx.x * a.chunk, t1 = min(a.tokens, t0 + a.chunk);
  pick_experts<NV, TOK>(a, t0, t1, sm, nullptr);
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x)
    a.counts[static_cast<int64_t>(blockIdx.x) * a.experts + e] = sm[e];
}

__global__ void __launch_bounds__(kRouteThreads) route_place_kernel(const RouteArgs a, int place_warps) {
  extern __shared__ int sm[];
  int* total = sm;
  int* first = sm + a.experts;
  int* mine = sm + 2 * a.experts;
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) total[e] = first[e] = 0;
  pdl_launch_dependents();
  pdl_wait();
  __syncthreads();
  // Counts of all blocks, and of those in front of this one.
  const int across = min(a.experts, static_cast<int>(blockDim.x));
  const int parts = blockDim.x / across, part = threadIdx.x / across;
  if (part < parts)
    for (int e = threadIdx.x - part * across; e < a.experts; e += across) {
      int all = 0, front = 0;
#pragma unroll 8
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
  const int64_t c0 = static_cast<int64_t>(blockIdx.x) * a.chunk * a.k;
  const int n = min(a.tokens - static_cast<int>(blockIdx.x) * a.chunk, a.chunk) * a.k;
  const int* chosen = a.experts_of + c0;
  place_choices(a, c0, n, first, mine, place_warps, [=](int i) { return chosen[i]; });
}

// Tokens per block: 64 (13.1 us for 17776 tokens of 64 experts, 16.3 with 128:
// four tokens per warp keep twice the warps busy), but at most 512 blocks,
// since every block of the second kernel reads every block's counts.
int route_chunk(int64_t tokens) {
  return static_cast<int>(std::max<int64_t>(64, ceil_div(tokens, 512)));
}

// ───────────────────────────── combine ─────────────────────────────
//
//   o[t, :] = residual[t, :] + sum_j weights[t, j] * y[slots[t, j], :]
//
// in fp32, j rising, one rounding at the end.  A slot outside [0, y_rows)
// adds nothing.  Bound by HBM: every expert row is read once (the slots of
// all choices are a permutation) and every output row written once, so each
// thread owns 16 bytes of an output row and has the loads of up to four expert
// rows in flight.  Measured at 17776 x 1920 bf16, two experts: 40.9 us, 5.01
// TB/s of 6.53.

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

// Any width, alignment and top_k: one element per thread and step.
__global__ void __launch_bounds__(256) combine_kernel(const CombineArgs a) {
  pdl_launch_dependents();
  pdl_wait();
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

template <int DT>
__device__ __forceinline__ void unpack_vec(const uint4& u, float* f) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == kF32) {
      f[i] = __uint_as_float(w[i]);
    } else if constexpr (DT == kBF16) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    } else {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
}

// UU x 16 bytes of the output per thread, 256 vectors apart; KK rows of y of each
// are in flight at once (the last KK - top_k % KK of a token read nothing).
template <int DT, int KK, int UU>
__global__ void __launch_bounds__(256) combine_vec_kernel(const CombineArgs a) {
  constexpr int E = DT == kF32 ? 4 : 8, ES = DT == kF32 ? 4 : 2;
  pdl_launch_dependents();
  const int vecs = a.cols / E;
  const int64_t i0 = blockIdx.x * (256LL * UU) + threadIdx.x;
  int64_t t[UU];
  int c[UU];
#pragma unroll
  for (int u = 0; u < UU; ++u) {
    const int64_t i = i0 + 256 * u;
    t[u] = i <= UINT_MAX ? static_cast<uint32_t>(i) / static_cast<uint32_t>(vecs) : i / vecs;
    c[u] = static_cast<int>(i - t[u] * vecs) * E;
  }
  pdl_wait();
  float acc[UU][E] = {};
  if (a.residual)
#pragma unroll
    for (int u = 0; u < UU; ++u)
      if (t[u] < a.tokens)
        unpack_vec<DT>(*reinterpret_cast<const uint4*>(static_cast<const char*>(a.residual) + (t[u] * a.ldr + c[u]) * ES),
                       acc[u]);
  for (int j0 = 0; j0 < a.k; j0 += KK) {
    uint4 v[UU][KK];
    float w[UU][KK];
    bool live[UU][KK];
#pragma unroll
    for (int u = 0; u < UU; ++u)
#pragma unroll
      for (int j = 0; j < KK; ++j) {
        const bool in = t[u] < a.tokens && j0 + j < a.k;
        const int64_t s = in ? a.slots[t[u] * a.k + j0 + j] : -1;
        live[u][j] = s >= 0 && s < a.y_rows;
        w[u][j] = live[u][j] ? a.weights[t[u] * a.k + j0 + j] : 0.0f;
        if (live[u][j])
          v[u][j] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const char*>(a.y) + (s * a.ldy + c[u]) * ES));
      }
#pragma unroll
    for (int u = 0; u < UU; ++u)
#pragma unroll
      for (int j = 0; j < KK; ++j)
        if (live[u][j]) {
          float f[E];
          unpack_vec<DT>(v[u][j], f);
#pragma unroll
          for (int e = 0; e < E; ++e) acc[u][e] = fmaf(w[u][j], f[e], acc[u][e]);
        }
  }
#pragma unroll
  for (int u = 0; u < UU; ++u) {
    if (t[u] >= a.tokens) break;
    char* o = static_cast<char*>(a.out) + (t[u] * a.ldo + c[u]) * ES;
    const float(&f)[E] = acc[u];
    if constexpr (DT == kF32)
      *reinterpret_cast<float4*>(o) = make_float4(f[0], f[1], f[2], f[3]);
    else
      *reinterpret_cast<uint4*>(o) = make_uint4(pack2(f[0], f[1], DT), pack2(f[2], f[3], DT), pack2(f[4], f[5], DT),
                                                pack2(f[6], f[7], DT));
  }
}

template <int DT>
int32_t launch_combine_vec(const CombineArgs& a, cudaStream_t s) {
  const int64_t vecs = a.tokens * (a.cols / (DT == kF32 ? 4 : 8));
  // Two vectors per thread where one leaves few loads in flight (us at 1920
  // columns, one / two vectors: 17776 tokens bf16, top 1 36 / 29, top 2 42 / 41;
  // 8000 tokens, top 4 32 / 39, fp32 top 2 37 / 39).
  const unsigned two = static_cast<unsigned>(ceil_div(vecs, 512)), one = static_cast<unsigned>(ceil_div(vecs, 256));
  if (a.k == 1) return launch_pdl(combine_vec_kernel<DT, 1, 2>, two, 256, 0, s, a);
  if (a.k == 2 && DT != kF32) return launch_pdl(combine_vec_kernel<DT, 2, 2>, two, 256, 0, s, a);
  if (a.k == 2) return launch_pdl(combine_vec_kernel<DT, 2, 1>, one, 256, 0, s, a);
  return launch_pdl(combine_vec_kernel<DT, 4, 1>, one, 256, 0, s, a);
}

bool known_dtype(int dt) { return dt == kF32 || dt == kF16 || dt == kBF16; }

int32_t check_route(int64_t tokens, int64_t experts, int32_t top_k) {
  if (tokens < 0) return fail(SF_ERR_INVALID_ARGUMENT, "negative token count");
  if (experts < 1 || top_k < 1 || top_k > experts)
    return fail(SF_ERR_INVALID_ARGUMENT, "top_k %d of %lld experts", top_k, (long long)experts);
  if (experts > kMaxExperts || top_k > kMaxTopK)
    return fail(SF_ERR_UNSUPPORTED, "top_k %d of %lld experts (at most %d of %d)", top_k,
                (long long)experts, kMaxTopK, kMaxExperts);
  if (tokens > kMostChoices / top_k)
    return fail(SF_ERR_UNSUPPORTED, "%lld tokens with %d choices exceed 2^31-2^23-1 slots",
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
  const size_t row = static_cast<size_t>(experts) * sizeof(int);
  // Warps that rank choices: no more than have 32 of them, and counts that fit.
  const auto place_warps = [&](int64_t choices, int warps) {
    return static_cast<int>(std::max<int64_t>(
        1, std::min<int64_t>({ceil_div(choices, 32), warps, static_cast<int64_t>(24 * 1024 / row)})));
  };
  if (tokens <= kSmallTokens) {
    a.chunk = static_cast<int>(tokens);
    const int warps = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(tokens, kSmallThreads / 32)));
    const int place = place_warps(tokens * top_k, warps);
    const size_t smem = row * (2 + place) + tokens * top_k * 2;
    if (experts <= 32) return launch_pdl(route_small_kernel<1, 2>, 1, warps * 32, smem, s, a, place);
    if (experts <= 64) return launch_pdl(route_small_kernel<2, 2>, 1, warps * 32, smem, s, a, place);
    if (experts <= 128) return launch_pdl(route_small_kernel<4, 2>, 1, warps * 32, smem, s, a, place);
    if (experts <= 256) return launch_pdl(route_small_kernel<8, 1>, 1, warps * 32, smem, s, a, place);
    return launch_pdl(route_small_kernel<32, 1>, 1, warps * 32, smem, s, a, place);
  }
  a.chunk = route_chunk(tokens);
  const unsigned blocks = static_cast<unsigned>(ceil_div(tokens, a.chunk));
  st = experts <= 32    ? launch_pdl(route_pick_kernel<1, 4>, blocks, kRouteThreads, row, s, a)
       : experts <= 64  ? launch_pdl(route_pick_kernel<2, 4>, blocks, kRouteThreads, row, s, a)
       : experts <= 128 ? launch_pdl(route_pick_kernel<4, 4>, blocks, kRouteThreads, row, s, a)
       : experts <= 256 ? launch_pdl(route_pick_kernel<8, 2>, blocks, kRouteThreads, row, s, a)
                        : launch_pdl(route_pick_kernel<32, 1>, blocks, kRouteThreads, row, s, a);
  if (st != SF_OK) return st;
  const int place = place_warps(static_cast<int64_t>(a.chunk) * top_k, kRouteThreads / 32);
  return launch_pdl(route_place_kernel, blocks, kRouteThreads, row * (2 + place), s, a, place);
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
  if (residual == out && ldr != ldo && tokens > 1)
    return fail(SF_ERR_INVALID_ARGUMENT, "in place needs one leading dimension (%lld, %lld)", (long long)ldr,
                (long long)ldo);
  DeviceInfo* dev = nullptr;
  const int32_t st = current_device_info(&dev, nullptr);
  if (st != SF_OK) return st;
  const CombineArgs a{tokens, static_cast<int>(cols), top_k, y, y_rows, ldy, dtype, slots, weights,
                      residual, ldr, out, ldo};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int es = esize(dtype);
  if (cols % (16 / es) == 0 && tokens * cols / (16 / es) <= 256LL * INT32_MAX && aligned16(y) && aligned16(out) &&
      bytes16(ldy, es) && bytes16(ldo, es) && (!residual || (aligned16(residual) && bytes16(ldr, es)))) {
    if (dtype == kF32) return launch_combine_vec<kF32>(a, s);
    return dtype == kBF16 ? launch_combine_vec<kBF16>(a, s) : launch_combine_vec<kF16>(a, s);
  }
  const unsigned grid = static_cast<unsigned>(
      std::min<int64_t>(ceil_div(tokens * cols, 256), dev->sm_count * 16LL));
  return launch_pdl(combine_kernel, grid, 256, 0, s, a);
}
