// MXFP4 codes to BF16 operands, shared by the product kernels.
//
// The low three bits of an E2M1 code, placed at bits 8-6 of a BF16 number, are its magnitude
// times 2^-126 (exponent and mantissa field line up, subnormals included). An integer
// multiplication copies a code there and its sign to bit 15, a mask clears the rest of the
// copies, and one BF16 multiplication by 2^(scale - 127 + 126) gives the value, exactly. A
// register takes code i of a 32-bit word and code i + 4, which lie at the same place of its two
// halves, so the K order of the operand inside each 8 columns is 0, 4, 1, 5, 2, 6, 3, 7; permute_x
// gives the other operand the same one. That is 17 instructions for 8 codes, 9 of them on the
// ALU; looking codes up in natural order with byte permutes takes 15 ALU operations.
#pragma once

#include "ptx.cuh"

namespace ce4b {

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r =
      __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// The factor 2^(scale - 1) of a group, twice in a register. It overflows BF16 from scale 129
// (groups whose largest weight is over 12): mx4_wide_factor stops at 2^127 there, and
// mx4_factor2 holds the rest. Scale 255 is NaN.
__device__ __forceinline__ uint32_t mx4_factor(uint32_t scale) {
  return scale * 0x00800080u + 126u * 0x00800080u;
}

__device__ __forceinline__ uint32_t mx4_wide_factor(uint32_t scale) {
  return scale == 255u ? 0x7FFF7FFFu : min(scale + 126u, 254u) * 0x00800080u;
}

__device__ __forceinline__ uint32_t mx4_factor2(uint32_t scale) {
  return (scale > 128u && scale < 255u ? scale - 1u : 127u) * 0x00800080u;
}

// The two multipliers, kept from the compiler, which would turn a product into shifts and an
// addition: the multiplication runs beside the ALU, which bounds the expansion.
struct Mx4Spread {
  uint32_t even = 0x1040u, odd = 0x0104u;
  __device__ __forceinline__ Mx4Spread() { asm volatile("" : "+r"(even), "+r"(odd)); }
};

// Codes 0..7 of a word as (0, 4), (1, 5), (2, 6), (3, 7).
__device__ __forceinline__ void mx4_expand(uint32_t w, uint32_t factor, const Mx4Spread& m, uint32_t (&v)[4]) {
  const uint32_t w8 = w >> 8;
  v[0] = mul_bf16x2(((w & 0x000F000Fu) * m.even) & 0x81C081C0u, factor);
  v[1] = mul_bf16x2(((w & 0x00F000F0u) * m.odd) & 0x81C081C0u, factor);
  v[2] = mul_bf16x2(((w8 & 0x000F000Fu) * m.even) & 0x81C081C0u, factor);
  v[3] = mul_bf16x2(((w8 & 0x00F000F0u) * m.odd) & 0x81C081C0u, factor);
}

// Codes 0..7 of a word in order. A table of the eight scaled magnitudes is split into low and
// high bytes; a byte permute looks up four codes at once (its selector nibbles are the codes
// themselves), the sign bits are merged into the high bytes, and two more permutes interleave.
__device__ __forceinline__ uint4 mx4_expand_ordered(uint32_t w, uint32_t scale) {
  uint32_t f = scale * 0x00800080u;        // 2^(scale - 127), twice
  if (scale == 0u) f = 0x00400040u;        // subnormal
  if (scale == 255u) f = 0x7FFF7FFFu;      // NaN
  const uint32_t p0 = mul_bf16x2(0x3F000000u, f), p1 = mul_bf16x2(0x3FC03F80u, f);  // 0, 0.5, 1, 1.5
  const uint32_t p2 = mul_bf16x2(0x40404000u, f), p3 = mul_bf16x2(0x40C04080u, f);  // 2, 3, 4, 6
  const uint32_t lo0 = prmt(p0, p1, 0x6420u), lo1 = prmt(p2, p3, 0x6420u);
  const uint32_t hi0 = prmt(p0, p1, 0x7531u), hi1 = prmt(p2, p3, 0x7531u);
  const uint32_t m = w & 0x77777777u, m4 = m >> 16, u = w << 4;
  const uint32_t l0 = prmt(lo0, lo1, m), l1 = prmt(lo0, lo1, m4);
  const uint32_t h0 = prmt(hi0, hi1, m) | (prmt(u, w, 0x5140u) & 0x80808080u);
  const uint32_t h1 = prmt(hi0, hi1, m4) | (prmt(u, w, 0x7362u) & 0x80808080u);
  return make_uint4(prmt(l0, h0, 0x5140u), prmt(l0, h0, 0x7362u), prmt(l1, h1, 0x5140u), prmt(l1, h1, 0x7362u));
}

// Columns 0..7 of a 16-byte chunk of x in the order of mx4_expand.
__device__ __forceinline__ uint4 permute_x(const uint4& v) {
  return make_uint4(prmt(v.x, v.z, 0x5410u), prmt(v.x, v.z, 0x7632u), prmt(v.y, v.w, 0x5410u),
                    prmt(v.y, v.w, 0x7632u));
}

// Weight bytes are read once: they leave the L1 cache to x.
__device__ __forceinline__ uint4 load_stream(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

}  // namespace ce4b
