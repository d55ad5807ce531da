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

// Eight values of each of the `kLanes` neighbouring lanes that hold a group -> this lane's word of codes and the group's scale and offset.
// Every step is one IEEE operation (the library is built with approximate division otherwise), so that a host computes the same codes.
// Magnitudes over 2^126 count as 2^126, which keeps scale and offset finite; a group with an infinity or a NaN becomes NaN as a whole.
template <int kLanes>
__device__ __forceinline__ void i4_quantize(const uint4& raw, uint32_t& word, uint32_t& meta) {
  constexpr float kMost = 8.507059173023462e37f, kLeast = 7.888609052210118e-31f;      // 2^126, 2^-100
  const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
  float f[8], lo = INFINITY, hi = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t bits = i & 1 ? u[i / 2] & 0xFFFF0000u : u[i / 2] << 16;
    bad |= (bits & 0x7F800000u) == 0x7F800000u;
    f[i] = fminf(fmaxf(__uint_as_float(bits), -kMost), kMost);
    lo = fminf(lo, f[i]);
    hi = fmaxf(hi, f[i]);
  }
  if (bad) hi = INFINITY;
#pragma unroll
  for (int d = 1; d < kLanes; d *= 2) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
  }
  float s = __bfloat162float(__float2bfloat16_rn(__fmul_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f), 16.f)));
  if (s < kLeast) s = 0.f;
  const float o = __bfloat162float(__float2bfloat16_rn(__fsub_rn(lo, s)));
  meta = pack_bf16x2(s, o);
  word = 0;
  if (hi == INFINITY) {
    meta = 0x7FFF7FFFu;
  } else if (s > 0.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = rintf(__fmul_rn(__fdiv_rn(__fsub_rn(f[i], o), s), 16.f));
      const uint32_t code = (uint32_t)(int)fminf(fmaxf(c - 16.f, 0.f), 15.f);
      word |= code << ((i & 1) * 16 + (i / 2) * 4);
    }
  }
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
