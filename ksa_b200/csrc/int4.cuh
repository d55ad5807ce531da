// Values held in four bits: the format shared by the quantised KV cache (int4_cache.cu, int4_attn.cu) and by weights (int4_linear.cu).
//
// A group of values (32 of a cache row, 32 / 64 / 128 of a weight row along K) has a scale S and an offset O in bf16, and a code c of 0 .. 15
// stands for bf16(S * (1 + c / 16) + O).  1 + c / 16 is what a bf16 becomes when its exponent is that of 1 and the upper four bits of its
// mantissa are the code, so two codes become two values by one shift, one LOP3 and one bf16x2 FMA, which rounds once.  What the
// values are is thereby fixed to the bit: attention and products use the very numbers that reading back returns.
// Eight codes make a 32-bit word, nibbles 0 .. 7 from the lowest being values 0, 2, 4, 6, 1, 3, 5, 7: the same shift leaves a pair of neighbours in
// the two halves of a register, in the order in which mma.sync and 16-byte stores want them.
#pragma once

#include "common.cuh"

namespace ksa {

constexpr int kI4CacheGroup = 32;

// Pair `I` (values 2 I and 2 I + 1) of a word as bf16x2 of 1 + c / 16.
template <int I>
__device__ __forceinline__ uint32_t i4_unit(uint32_t w) {
  const uint32_t x = I == 0 ? w << 3 : w >> (4 * I - 3);
  uint32_t u;                       // (x & 0x00780078) | 0x3F803F80: the compiler makes two operations of the plain form
  asm("lop3.b32 %0, %1, 0x00780078, 0x3F803F80, 0xEA;" : "=r"(u) : "r"(x));
  return u;
}
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// A group's scale and offset (low and high half of a word), each in both halves of a register.
__device__ __forceinline__ uint32_t i4_scale2(uint32_t meta) { return __byte_perm(meta, meta, 0x1010); }
__device__ __forceinline__ uint32_t i4_offset2(uint32_t meta) { return __byte_perm(meta, meta, 0x3232); }
// A word's eight values, neighbours in a register.
__device__ __forceinline__ void i4_values(uint32_t (&v)[4], uint32_t w, uint32_t s2, uint32_t o2) {
  v[0] = fma_bf16x2(i4_unit<0>(w), s2, o2);
  v[1] = fma_bf16x2(i4_unit<1>(w), s2, o2);
  v[2] = fma_bf16x2(i4_unit<2>(w), s2, o2);
  v[3] = fma_bf16x2(i4_unit<3>(w), s2, o2);
}

__device__ __forceinline__ uint32_t min_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("min.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t max_nan_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Sixteen values of each of the `kLanes` neighbouring lanes that hold a group -> this lane's words of codes and the group's scale and offset.
// The codes are those of one IEEE operation after another, c = rint(((x - O) / S) * 16) - 16 (the library is built with approximate division
// otherwise), so that a host computes the same; many values of a coarse grid lie exactly between two codes.  A division costs ten operations a
// value.  Instead t = x - O is multiplied by 16 / S in two terms: an approximation r to 2^-22, and what it leaves, e = (16 - r S) / S to 2^-22 of it.
// RN(t r + RN(t e)) is t * 16 / S to within 2^-43 before the last rounding, and the quotient of 24 bits by 8 bits lies at least 2^-33 from the
// middle between two floats (t - m S is a multiple of 2^-33 t for a middle m of 25 bits, and not zero: m S has more than 24 bits), so that
// the last rounding is the division's.  The range is divided by 15, of four bits, in the same way.
// Magnitudes over 2^126 count as 2^126, which keeps scale and offset finite; a group with an infinity or a NaN becomes NaN as a whole.
template <int kLanes>
__device__ __forceinline__ void i4_quantize(const uint4 (&raw)[2], uint2& words, uint32_t& meta) {
  constexpr float kMost = 8.507059173023462e37f, kLeast = 7.888609052210118e-31f;      // 2^126, 2^-100
  constexpr float kRound = 12582912.f;                           // 1.5 * 2^23: a sum with it has whole numbers in its lowest bits
  const uint32_t u[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
  uint32_t lo2 = u[0], hi2 = u[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) { lo2 = min_bf16x2(lo2, u[i]); hi2 = max_nan_bf16x2(hi2, u[i]); }
#pragma unroll
  for (int d = 1; d < kLanes; d *= 2) {
    lo2 = min_bf16x2(lo2, __shfl_xor_sync(0xffffffffu, lo2, d));
    hi2 = max_nan_bf16x2(hi2, __shfl_xor_sync(0xffffffffu, hi2, d));
  }
  lo2 = min_bf16x2(lo2, __byte_perm(lo2, lo2, 0x1032));
  hi2 = max_nan_bf16x2(hi2, __byte_perm(hi2, hi2, 0x1032));
  const bool bad = (hi2 & 0x7F80u) == 0x7F80u || (lo2 & 0x7F80u) == 0x7F80u;
  const float lo = fminf(fmaxf(__uint_as_float(lo2 << 16), -kMost), kMost), hi = fminf(fmaxf(__uint_as_float(hi2 << 16), -kMost), kMost);
  const float range = __fsub_rn(hi, lo);                         // * 16 / 15
  float s = __bfloat162float(__float2bfloat16_rn(fmaf(range, 1.0666667222976685f, __fmul_rn(range, -5.563100202721216e-08f))));
  if (s < kLeast) s = 0.f;
  const float o = __bfloat162float(__float2bfloat16_rn(__fsub_rn(lo, s)));
  meta = bad ? 0x7FFF7FFFu : pack_bf16x2(s, o);
  words = make_uint2(0, 0);
  if (bad || s == 0.f) return;
  const float down = s > 1.1529215e18f ? 8.6736174e-19f : 1.f;   // 2^60, 2^-60: keeps e normal
  const float to = -o * down, sd = s * down, r = __fdividef(16.f, sd), e = fmaf(-r, sd, 16.f) * (r * 0.0625f);
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float even = 0.f, odd = 0.f;                                 // four codes each, as one number
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t pair = u[h * 4 + i / 2];
      const float x = __uint_as_float(i & 1 ? pair & 0xFFFF0000u : pair << 16), t = fmaf(x, down, to);
      const float y = fminf(fmaxf(fmaf(t, r, __fmul_rn(t, e)), 16.f), 31.f), c = __fsub_rn(__fadd_rn(y, kRound), kRound);
      if (i & 1) odd = fmaf(c, (float)(1 << (i / 2 * 4)), odd);
      else even = fmaf(c, (float)(1 << (i / 2 * 4)), even);
    }
    // 16 * (1 + 16 + 256 + 4096) = 69904 too much each
    w[h] = __byte_perm(__float_as_uint(even + (kRound - 69904.f)), __float_as_uint(odd + (kRound - 69904.f)), 0x5410);
  }
  words = make_uint2(w[0], w[1]);
}

// Each row of an 8 x 8 matrix of 16-bit values lies in four lanes; afterwards each column does.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

}  // namespace ksa
