// Residual addition and RMSNorm of rows (kernel-op API add_rmsnorm_forward and
// add_rmsnorm_mxfp8): s = bf16(x + residual), n = bf16(s * (mean(s^2) + eps)^(-1/2) * w), n as
// BF16 or as the MXFP8 codes and scales of that BF16 value.
#include "internal.h"
#include "mxfp8.cuh"
#include "ptx.cuh"

namespace ce4b {

namespace {

// n is the BF16 rounding of the formula's FP32 value: the squares (exact in 64 bits) are summed
// in 64 bits and the factor (mean + eps)^(-1/2) is kept as an FP32 pair hi + lo, so that a row's
// result does not depend on the order of its sum, on the launch shape or on the row's
// neighbours. Every form of the operator gives the same n, and the MXFP8 form quantises
// exactly that value.
struct RowScale {
  float hi, lo;
};

__device__ __forceinline__ RowScale row_scale(double sum, double inv_width, float eps) {
  const double f = rsqrt(fma(sum, inv_width, static_cast<double>(eps)));
  RowScale r;
  r.hi = static_cast<float>(f);
  r.lo = static_cast<float>(f - static_cast<double>(r.hi));
  return r;
}

// s * (hi + lo) * w: q is the FP32 rounding of the product and e the rest, so that q + e is the
// product rounded to FP32 once (about 2^-46 of it is lost before). An overflowing q has no rest.
__device__ __forceinline__ float scale_round(float s, float w, const RowScale& f) {
  const float t = s * f.hi;
  const float te = fmaf(s, f.lo, fmaf(s, f.hi, -t));
  const float q = t * w;
  const float e = fmaf(te, w, fmaf(t, w, -q));
  return bf16_round(fabsf(q) <= 3.0e38f ? q + e : q);
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warps = blockDim.x / 32;
  if ((threadIdx.x & 31) == 0) part[threadIdx.x / 32] = v;
  __syncthreads();
  v = 0.0;
  for (int i = 0; i < warps; ++i) v += part[i];
  return v;
}

// One block per row (rows in blockIdx.x); the row is read again for the second pass.
__global__ void add_rmsnorm_kernel(const bf16* x, const bf16* residual, const bf16* w, bf16* sum,
                                   bf16* out, uint8_t* codes, uint8_t* scales, int rows, int width,
                                   double inv_width, float eps) {
  const int row = blockIdx.x;
  if (row >= rows) {  // padding rows of the last scale tile
    for (int b = threadIdx.x; b < width / 32; b += blockDim.x) scales[mx_scale_offset(row, b, width / 128)] = 0;
    return;
  }
  const size_t at = static_cast<size_t>(row) * width;
  double ss = 0.0;
  for (int c = threadIdx.x; c < width; c += blockDim.x) {
    float s = __bfloat162float(x[at + c]);
    if (residual != nullptr) {
      s = bf16_round(s + __bfloat162float(residual[at + c]));
      sum[at + c] = __float2bfloat16_rn(s);
    }
    ss = fma(static_cast<double>(s), static_cast<double>(s), ss);
  }
  ss = block_sum(ss);
  const RowScale f = row_scale(ss, inv_width, eps);
  const bf16* src = residual != nullptr ? sum : x;
  if (codes == nullptr) {
    for (int c = threadIdx.x; c < width; c += blockDim.x) {
      out[at + c] = __float2bfloat16_rn(
          scale_round(__bfloat162float(src[at + c]), __bfloat162float(w[c]), f));
    }
    return;
  }
  __syncthreads();  // the sum of other threads' columns is read below
  for (int b = threadIdx.x; b < width / 32; b += blockDim.x) {
    float v[32];
    for (int j = 0; j < 32; ++j) {
      v[j] = scale_round(__bfloat162float(src[at + b * 32 + j]), __bfloat162float(w[b * 32 + j]), f);
    }
    uint32_t q[8];
    const uint8_t sc = mx_quantize32(v, q);
    uint32_t* dst = reinterpret_cast<uint32_t*>(codes + at + b * 32);
    for (int j = 0; j < 8; ++j) dst[j] = q[j];
    scales[mx_scale_offset(row, b, width / 128)] = sc;
  }
}

}  // namespace

void add_rmsnorm_rows(const bf16* x, const bf16* residual, const bf16* w, bf16* sum, bf16* out,
                      uint8_t* codes, uint8_t* scales, int rows, int width, float eps,
                      cudaStream_t s) {
  const int grid = codes != nullptr ? (rows + 127) / 128 * 128 : rows;
  add_rmsnorm_kernel<<<grid, 256, 0, s>>>(x, residual, w, sum, out, codes, scales, rows, width,
                                          1.0 / width, eps);
  check_cuda(cudaGetLastError(), "add_rmsnorm launch");
}

}  // namespace ce4b
