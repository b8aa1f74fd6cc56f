// MXFP4 weights (kernel-op API quantize_mxfp4, dequantize_mxfp4):
// E2M1 codes, two to a byte with the even column in the low half, and one E8M0 scale per row
// and 32 columns in the scale tiles of MXFP8 tensors (rows padded to 128).
#include <cuda_fp4.h>

#include <algorithm>

#include "internal.h"
#include "launch.cuh"
#include "mxfp4.cuh"
#include "mxfp8.cuh"
#include "ptx.cuh"

namespace ce4b {

namespace {

// The smallest power of two 2^(code - 127), 2^-39 at least (the floor of the MXFP8 recipe), that
// leaves no magnitude of the group over 6, the largest E2M1 value: 6 * 2^k = 1.5 * 2^(k + 2),
// so the exponent and the comparison of the mantissa with 1.5 decide, without rounding. A
// group that holds a NaN or an infinity gets the scale NaN (255).
__device__ __forceinline__ uint32_t mx4_scale_code(uint32_t amax_bits) {  // of an FP32 magnitude
  const uint32_t e = amax_bits >> 23;
  if (e == 255u) return 255u;
  const uint32_t code = e + ((amax_bits & 0x7FFFFFu) > 0x400000u ? 1u : 0u);
  return code < 88u + 2u ? 88u : code - 2u;
}

// The larger magnitudes of two pairs (of either sign); NaN stays NaN.
__device__ __forceinline__ uint32_t max_abs_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmax2_nan(__habs2(*reinterpret_cast<const __nv_bfloat162*>(&a)),
                                       __habs2(*reinterpret_cast<const __nv_bfloat162*>(&b)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Both kernels take [16 rows][128 columns] tiles with 256 threads, eight columns a thread (16
// bytes of BF16, 4 bytes of codes), and kTiles column tiles at once for loads in flight. Sixteen
// threads hold the four scale bytes of a row in a tile, one 32-bit word. Bound by memory: 8192 x
// 8192 there and back takes 61.5 us, 5.5 TB/s of the bytes in and out and of the 4-bit form
// between them (which the L2 cache mostly holds). No pointer is declared unaliased: the loads would
// become read-only ones, which a kernel may not use for what its predecessor still writes when
// it starts.
constexpr int kTiles = 4;

__global__ void __launch_bounds__(256)
    mx4_quantize_kernel(const bf16* x, uint8_t* codes, uint8_t* scales, int rows, int cols) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 16 + threadIdx.x / 16;
  const int lane = threadIdx.x % 16;
  const int col_tiles = cols / 128;
  grid_dependency_wait();
  grid_launch_dependents();
  const bool live = row < rows;
  uint32_t* const scale_row = reinterpret_cast<uint32_t*>(scales) +
                              (row / 128 * col_tiles) * 128 + (row % 32) * 4 + row / 32 % 4;
  for (int t0 = blockIdx.y * kTiles; t0 < col_tiles; t0 += gridDim.y * kTiles) {
    const uint4* src = reinterpret_cast<const uint4*>(x + row * cols) + t0 * 16 + lane;
    uint32_t* dst = reinterpret_cast<uint32_t*>(codes + row * (cols / 2)) + t0 * 16 + lane;
    uint32_t* scale_dst = scale_row + static_cast<int64_t>(t0) * 128;
    const int here = col_tiles - t0;
    uint4 v[kTiles];
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      v[j] = make_uint4(0u, 0u, 0u, 0u);
      if (live && j < here) v[j] = src[j * 16];
    }
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
      uint32_t top = max_abs_bf16x2(max_abs_bf16x2(w[0], w[1]), max_abs_bf16x2(w[2], w[3]));
      top = max_abs_bf16x2(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max_abs_bf16x2(top, __shfl_xor_sync(0xffffffffu, top, 2)) & 0x7FFF7FFFu;
      const uint32_t code = mx4_scale_code(max(top << 16, top & 0xFFFF0000u));
      // x / scale is exact in BF16 (or far below half the smallest code); 2^(127 - code) is too.
      const uint32_t inv = (254u - code) * 0x00800080u;
      uint32_t q = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack_bf16x2(mul_bf16x2(w[i], inv));
        q |= static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(f, __NV_E2M1, cudaRoundNearest)) << (8 * i);
      }
      if (code == 255u) q = 0;
      uint32_t word = live ? code << (8 * (lane / 4)) : 0u;  // padding rows: 0
      word |= __shfl_xor_sync(0xffffffffu, word, 4);
      word |= __shfl_xor_sync(0xffffffffu, word, 8);
      if (j < here) {
        if (live) dst[j * 16] = q;
        if (lane == 0) scale_dst[j * 128] = word;
      }
    }
  }
}

__global__ void __launch_bounds__(256)
    mx4_dequantize_kernel(const uint8_t* codes, const uint8_t* scales, bf16* out, int rows,
                          int cols) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 16 + threadIdx.x / 16;
  const int lane = threadIdx.x % 16;
  const int col_tiles = cols / 128;
  grid_dependency_wait();
  grid_launch_dependents();
  if (row >= rows) return;
  const uint32_t* const scale_row = reinterpret_cast<const uint32_t*>(scales) +
                                    (row / 128 * col_tiles) * 128 + (row % 32) * 4 + row / 32 % 4;
  for (int t0 = blockIdx.y * kTiles; t0 < col_tiles; t0 += gridDim.y * kTiles) {
    const uint32_t* src = reinterpret_cast<const uint32_t*>(codes + row * (cols / 2)) + t0 * 16 + lane;
    const uint32_t* scale_src = scale_row + static_cast<int64_t>(t0) * 128;
    uint4* dst = reinterpret_cast<uint4*>(out + row * cols) + t0 * 16 + lane;
    const int here = col_tiles - t0;
    uint32_t q[kTiles], s[kTiles];
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      q[j] = j < here ? src[j * 16] : 0u;
      s[j] = j < here ? scale_src[j * 128] : 0u;
    }
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      if (j < here) dst[j * 16] = mx4_expand_ordered(q[j], s[j] >> (8 * (lane / 4)) & 255u);
    }
  }
}

}  // namespace

void mx4_quantize(const bf16* x, uint8_t* codes, uint8_t* scales, int rows, int cols, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(rows) + 127) / 128 * 8),
                  static_cast<unsigned>(std::min((cols / 128 + kTiles - 1) / kTiles, 65535)));
  launch(mx4_quantize_kernel, grid, 256, 0, 0, s, x, codes, scales, rows, cols);
}

void mx4_dequantize(const uint8_t* codes, const uint8_t* scales, bf16* out, int rows, int cols,
                    cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(rows) + 15) / 16),
                  static_cast<unsigned>(std::min((cols / 128 + kTiles - 1) / kTiles, 65535)));
  launch(mx4_dequantize_kernel, grid, 256, 0, 0, s, codes, scales, out, rows, cols);
}

}  // namespace ce4b
