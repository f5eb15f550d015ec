// Linears with 4-bit weights and group scales.
//
//   y[m, n] = act(sum_k x[m, k] W[n, k] + bias[n]),
//   W[n, k] = scale[k / g, n] * (q[n, k] - zero[k / g, n]),  q in 0..15,
//
// zero = 8 where none is stored.  q, zero (an integer in practice) and their
// difference are exact in 16 bits, the scale stays out of the products: a
// group's sum of x * (q - zero) is formed in fp32 and scaled once.
//
// Layout of q: row n is a run of 32-bit words, 16 per block of 128 columns
// (K is padded to whole blocks; what the padding holds is not used).  Nibble i
// of word 4 t + w of a block holds column
//   32 w + 8 t + (0, 2, 4, 6, 1, 3, 5, 7)[i].
// Scales and zeros are [K / g, N], so that neighbouring rows' are contiguous.
#include <cuda_runtime.h>

#include <algorithm>

#include "common.h"
#include "epilogue.cuh"
#include "tma_host.h"

namespace sf {
namespace {

constexpr int kW4MaxRows = 64;

struct W4Args {
  int M, N, K;
  const void* x;
  int64_t ldx;
  const uint32_t* packed;
  int64_t ldp;  // words per row
  const void* scales;
  const void* zeros;
  int64_t lds;
  int group;    // 32, 64 or 128
  int dtype;    // of x, scales and zeros
  const void* bias;
  int bias_dtype;
  void* y;
  int64_t ldy;
  int out_dtype;
  int act;
  int fast_act;
};

// Column, within its 128-column block, of nibble i of word j.
__host__ __device__ __forceinline__ int w4_column(int j, int i) {
  return 32 * (j & 3) + 8 * (j >> 2) + (i < 4 ? 2 * i : 2 * i - 7);
}

// One warp per output row n, eight rows of x at a time.
__global__ void __launch_bounds__(256) w4_linear_kernel(const W4Args a) {
  const int lane = threadIdx.x & 31;
  const int n = (blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (n >= a.N) return;
  const int words = static_cast<int>((a.K + 127) / 128 * 16);
  for (int m0 = 0; m0 < a.M; m0 += 8) {
    float acc[8] = {};
    for (int wd = lane; wd < words; wd += 32) {
      const uint32_t q = a.packed[n * a.ldp + wd];
      const int base = wd / 16 * 128;
      for (int i = 0; i < 8; ++i) {
        const int k = base + w4_column(wd & 15, i);
        if (k >= a.K) continue;
        const int64_t at = static_cast<int64_t>(k / a.group) * a.lds + n;
        const float z = a.zeros ? load_as_f32(a.zeros, at, a.dtype) : 8.0f;
        const float w = load_as_f32(a.scales, at, a.dtype) * (static_cast<float>((q >> (4 * i)) & 15u) - z);
        for (int m = 0; m < 8; ++m)
          if (m0 + m < a.M) acc[m] = fmaf(w, load_as_f32(a.x, (m0 + m) * a.ldx + k, a.dtype), acc[m]);
      }
    }
    for (int m = 0; m < 8; ++m) {
      for (int o = 16; o > 0; o >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], o);
      if (lane == 0 && m0 + m < a.M) {
        float v = acc[m] + (a.bias ? load_as_f32(a.bias, n, a.bias_dtype) : 0.0f);
        v = a.fast_act ? act_apply_fast(v, a.act) : act_apply(v, a.act);
        store_from_f32(a.y, (m0 + m) * a.ldy + n, a.out_dtype, v);
      }
    }
  }
}

// Quantisation of one group of one row per warp-quarter is not worth a tuned
// kernel (it runs once, at load): one thread per (row, group).
//   symmetric:  s = max |w| / 7 rounded to the stored type, q = rint(w / s) + 8
//   with zeros: s = (max - min) / 15 rounded likewise, z = rint(-min / s),
//               q = rint(w / s) + z; max and min taken with 0 included, so
//               that z lies in 0..15 and a weight of 0 is kept exactly
// q clamped to 0..15; s = 0 (an all-zero group) stores q = z.
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
  for (int k = k0; k < k1; ++k) {
    const float w = load_as_f32(W, n * ldw + k, w_dtype);
    lo = fminf(lo, w);
    hi = fmaxf(hi, w);
  }
  store_from_f32(scales, g * lds + n, s_dtype, zeros ? (hi - lo) / 15.0f : fmaxf(hi, -lo) / 7.0f);
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
      const float z = zeros ? load_as_f32(zeros, at, s_dtype) : 8.0f;
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
  if (N > INT32_MAX || K > INT32_MAX - 127) return fail(SF_ERR_UNSUPPORTED, "dimension exceeds 2^31-1");
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
  if (!y || (K > 0 && !x)) return fail(SF_ERR_INVALID_ARGUMENT, "null pointer");
  if (ldx < K || ldy < N) return fail(SF_ERR_INVALID_ARGUMENT, "leading dimension too small");
  const W4Args a{static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), x, ldx, packed, ldp,
                 scales, zeros, lds, group, in_dtype, bias, bias_dtype, y, ldy, out_dtype, activation,
                 out_dtype != kF32 ? 1 : 0};
  w4_linear_kernel<<<static_cast<unsigned>(ceil_div(N, 8)), 256, 0, static_cast<cudaStream_t>(stream)>>>(a);
  SF_CUDA_TRY(cudaGetLastError());
  return SF_OK;
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
