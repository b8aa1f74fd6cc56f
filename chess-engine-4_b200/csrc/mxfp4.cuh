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
// (groups whose largest weight is over 12): there it is 2^127, and mx4_factor2 holds the rest.
__device__ __forceinline__ uint32_t mx4_factor(uint32_t scale) {
  return scale == 255u ? 0x7FFF7FFFu : min(scale + 126u, 254u) * 0x00800080u;  // 255 is NaN
}

__device__ __forceinline__ uint32_t mx4_factor2(uint32_t scale) {
  return (scale > 128u && scale < 255u ? scale - 1u : 127u) * 0x00800080u;
}

// Codes 0..7 of a word as (0, 4), (1, 5), (2, 6), (3, 7).
__device__ __forceinline__ void mx4_expand(uint32_t w, uint32_t factor, uint32_t (&v)[4]) {
  const uint32_t w8 = w >> 8;
  v[0] = mul_bf16x2(((w & 0x000F000Fu) * 0x1040u) & 0x81C081C0u, factor);
  v[1] = mul_bf16x2(((w & 0x00F000F0u) * 0x0104u) & 0x81C081C0u, factor);
  v[2] = mul_bf16x2(((w8 & 0x000F000Fu) * 0x1040u) & 0x81C081C0u, factor);
  v[3] = mul_bf16x2(((w8 & 0x00F000F0u) * 0x0104u) & 0x81C081C0u, factor);
}

// Columns 0..7 of a 16-byte chunk of x in the order of mx4_expand.
__device__ __forceinline__ uint4 permute_x(const uint4& v) {
  return make_uint4(prmt(v.x, v.z, 0x5410u), prmt(v.x, v.z, 0x7632u), prmt(v.y, v.w, 0x5410u),
                    prmt(v.y, v.w, 0x7632u));
}

}  // namespace ce4b
