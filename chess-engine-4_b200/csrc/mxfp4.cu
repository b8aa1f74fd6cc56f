// MXFP4 weights (kernel-op API quantize_mxfp4, dequantize_mxfp4):
// E2M1 codes, two to a byte with the even column in the low half, and one E8M0 scale per row
// and 32 columns in the scale tiles of MXFP8 tensors (rows padded to 128).
#include <cuda_fp4.h>

#include <algorithm>

#include "internal.h"
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

__device__ __forceinline__ float mx4_value(uint32_t nibble) {
  const uint32_t m = nibble & 7u;
  const float v = m < 4u ? 0.5f * m : (m == 4u ? 2.0f : (m == 5u ? 3.0f : (m == 6u ? 4.0f : 6.0f)));
  return nibble & 8u ? -v : v;
}

__device__ __forceinline__ float mx4_scale(uint32_t code) {  // 2^(code - 127); NaN for 255
  if (code == 255u) return __uint_as_float(0x7FFFFFFFu);
  return code == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(code << 23);
}

// One thread per (row, 32-column group); rows past the last one zero their scale bytes.
__global__ void mx4_quantize_kernel(const bf16* __restrict__ x, uint8_t* __restrict__ codes,
                                    uint8_t* __restrict__ scales, int rows, int cols) {
  const int groups = cols / 32;
  const int64_t total = static_cast<int64_t>((rows + 127) / 128 * 128) * groups;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int row = static_cast<int>(i / groups);
    const int g = static_cast<int>(i - static_cast<int64_t>(row) * groups);
    uint32_t code = 0;
    if (row < rows) {
      const bf16* src = x + static_cast<size_t>(row) * cols + g * 32;
      uint32_t amax = 0;
      for (int j = 0; j < 32; ++j) {
        amax = max(amax, __float_as_uint(__bfloat162float(src[j])) & 0x7FFFFFFFu);
      }
      code = mx4_scale_code(amax);
      const float inv = code == 255u ? 0.0f : mx_scale_inverse(static_cast<uint8_t>(code));
      uint8_t* dst = codes + static_cast<size_t>(row) * (cols / 2) + g * 16;
      for (int j = 0; j < 16; ++j) {
        const float2 v = make_float2(__bfloat162float(src[2 * j]) * inv, __bfloat162float(src[2 * j + 1]) * inv);
        dst[j] = code == 255u ? 0 : __nv_cvt_float2_to_fp4x2(v, __NV_E2M1, cudaRoundNearest);
      }
    }
    scales[mx_scale_offset(row, g, cols / 128)] = static_cast<uint8_t>(code);
  }
}

__global__ void mx4_dequantize_kernel(const uint8_t* __restrict__ codes,
                                      const uint8_t* __restrict__ scales, bf16* __restrict__ out,
                                      int rows, int cols) {
  const int groups = cols / 32;
  const int64_t total = static_cast<int64_t>(rows) * groups;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int row = static_cast<int>(i / groups);
    const int g = static_cast<int>(i - static_cast<int64_t>(row) * groups);
    const float s = mx4_scale(scales[mx_scale_offset(row, g, cols / 128)]);
    const uint8_t* src = codes + static_cast<size_t>(row) * (cols / 2) + g * 16;
    bf16* dst = out + static_cast<size_t>(row) * cols + g * 32;
    for (int j = 0; j < 16; ++j) {
      dst[2 * j] = __float2bfloat16_rn(mx4_value(src[j] & 15u) * s);
      dst[2 * j + 1] = __float2bfloat16_rn(mx4_value(src[j] >> 4) * s);
    }
  }
}

int grid_for(int64_t work, int threads) {
  return static_cast<int>(std::min<int64_t>((work + threads - 1) / threads, static_cast<int64_t>(sm_count()) * 16));
}

}  // namespace

void mx4_quantize(const bf16* x, uint8_t* codes, uint8_t* scales, int rows, int cols, cudaStream_t s) {
  const int64_t work = static_cast<int64_t>((rows + 127) / 128 * 128) * (cols / 32);
  mx4_quantize_kernel<<<grid_for(work, 256), 256, 0, s>>>(x, codes, scales, rows, cols);
  check_cuda(cudaGetLastError(), "quantize_mxfp4 launch");
}

void mx4_dequantize(const uint8_t* codes, const uint8_t* scales, bf16* out, int rows, int cols,
                    cudaStream_t s) {
  const int64_t work = static_cast<int64_t>(rows) * (cols / 32);
  mx4_dequantize_kernel<<<grid_for(work, 256), 256, 0, s>>>(codes, scales, out, rows, cols);
  check_cuda(cudaGetLastError(), "dequantize_mxfp4 launch");
}

}  // namespace ce4b
