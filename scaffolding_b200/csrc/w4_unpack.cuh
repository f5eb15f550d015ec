// Arguments and unpacking of 4-bit weights, shared by the 4-bit linear kernels.
#pragma once
#include <cstdint>

#include "epilogue.cuh"

namespace sf {

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

// (v & mask) | magic as the one logic operation that it is.
__device__ __forceinline__ uint32_t and_or(uint32_t v, uint32_t mask, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "r"(mask), "r"(magic));
  return r;
}

// A stored zero point as the whole number 0..15 it stands for.
__device__ __forceinline__ float whole_zero(float z) { return fminf(fmaxf(rintf(z), 0.0f), 15.0f); }

// fp32 value of 16 stored bits.
template <bool BF16>
__device__ __forceinline__ float w4_float(uint32_t v) {
  return BF16 ? __uint_as_float(v << 16) : __half2float(__ushort_as_half(static_cast<uint16_t>(v)));
}

// Word -> four pairs (columns 2 i, 2 i + 1) of q - z.  z is the pair constant
// of the group: 128 + z (bf16); 1024 + z in .x and 64 + z in .y (fp16).
template <bool BF16>
__device__ __forceinline__ void unpack_word(uint32_t w, uint2 z, uint32_t (&p)[4]) {
  if constexpr (BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = and_or(w >> (4 * i), 0x000F000Fu, 0x43004300u);
      const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v),
                                       *reinterpret_cast<const __nv_bfloat162*>(&z.x));
      p[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
  } else {
    const uint32_t sixteenth = 0x2C002C00u;  // 1/16, 1/16
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t u = h ? w >> 8 : w;
      const uint32_t lo = and_or(u, 0x000F000Fu, 0x64006400u);  // 1024 + q
      const uint32_t hi = and_or(u, 0x00F000F0u, 0x64006400u);  // 1024 + 16 q
      const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&lo), *reinterpret_cast<const __half2*>(&z.x));
      const __half2 b = __hfma2(*reinterpret_cast<const __half2*>(&hi),
                                *reinterpret_cast<const __half2*>(&sixteenth),
                                __hneg2(*reinterpret_cast<const __half2*>(&z.y)));
      p[2 * h] = *reinterpret_cast<const uint32_t*>(&a);
      p[2 * h + 1] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
}

// A scale or zero point ahead of its use.  A register of its own for each, and
// no branch or select on the value: either would make the load be waited for
// where it is issued (250 cycles each, measured).  Not a read-only load: the grid
// may have been launched before what it reads was written.
__device__ __forceinline__ uint32_t load_ahead(const uint16_t* p) {
  uint32_t v;
  asm volatile("{\n\t.reg .u16 t;\n\tld.global.u16 t, [%1];\n\tcvt.u32.u16 %0, t;\n\t}" : "=r"(v) : "l"(p));
  return v;
}

// The pair constant of a stored zero point (16 bits, low half of v): adding
// the magic rounds it to a whole number, the clamp keeps it in 0..15 (a NaN
// becomes 0), as whole_zero does.
template <bool BF16>
__device__ __forceinline__ uint2 zero_pair(uint32_t v) {
  const uint32_t two = v * 0x10001u;
  uint2 r;
  if constexpr (BF16) {
    __nv_bfloat162 m = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&two), __float2bfloat162_rn(128.0f));
    m = __hmin2(__hmax2(m, __float2bfloat162_rn(128.0f)), __float2bfloat162_rn(143.0f));
    r.x = *reinterpret_cast<const uint32_t*>(&m);
    r.y = 0;
  } else {
    __half2 m = __hadd2(*reinterpret_cast<const __half2*>(&two), __float2half2_rn(1024.0f));
    m = __hmin2(__hmax2(m, __float2half2_rn(1024.0f)), __float2half2_rn(1039.0f));
    const __half2 n = __hsub2(m, __float2half2_rn(960.0f));
    r.x = *reinterpret_cast<const uint32_t*>(&m);
    r.y = *reinterpret_cast<const uint32_t*>(&n);
  }
  return r;
}

// A row's scale and the pair constant of its zero, as one word for a shuffle:
// the scale's bits below, the first constant's above.
template <bool BF16>
__device__ __forceinline__ uint32_t pack_scale(uint32_t scale, uint32_t zero, bool zeros) {
  const uint32_t z = zeros ? zero_pair<BF16>(zero).x : (BF16 ? 0x43084308u : 0x64086408u);  // + 8
  return __byte_perm(scale, z, 0x5410);
}

template <bool BF16>
__device__ __forceinline__ void unpack_scale(uint32_t v, float& s, uint2& z) {
  s = w4_float<BF16>(v & 0xFFFFu);
  z.x = __byte_perm(v, v, 0x3232);
  z.y = 0;
  if constexpr (!BF16) {
    const __half2 n = __hsub2(*reinterpret_cast<const __half2*>(&z.x), __float2half2_rn(960.0f));
    z.y = *reinterpret_cast<const uint32_t*>(&n);
  }
}

// Accumulators of one 16 x 8 tile and group.  An mma.sync that adds to the result
// of the one before it waits about 140 cycles for it (a block of eight chained
// ones took 1100 cycles, in two chains of four 534), so a group's mmas go round
// several accumulators, as many as there are registers for.
__host__ __device__ constexpr int w4_accumulators(int nt, int gw) { return nt == 1 && gw > 1 ? 4 : 2; }

template <int NA>
__device__ __forceinline__ float sum_of(const float (&s)[NA][4], int c) {
  return NA == 4 ? (s[0][c] + s[1][c]) + (s[NA - 2][c] + s[NA - 1][c]) : s[0][c] + s[1][c];
}

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  if constexpr (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

}  // namespace sf
