// Products of very few BF16 activation rows with an MXFP4 weight (kernel-op API mxfp4_linear,
// mxfp4_swiglu), and the choice between this form and the tcgen05 one.
//
// The time is the weight's 0.53 bytes per element as long as a code costs at most three
// lane operations (an SM takes in about 43 codes a clock at the memory's rate and issues 128
// lane operations), of which expanding it to BF16 takes 2.1 (mxfp4.cuh). With up to 32 rows the
// rest is a warp-level MMA per 8 codes a lane and 8 rows, whose A fragment is made in the very
// registers that the codes were loaded into: no shared memory, no barrier and no hand-over
// between warps until the sums are joined, so that any number of warps hides the memory's
// latency. A warp takes 16 weight rows (SwiGLU: 8 gate rows and their 8 up rows, which meet in
// one thread) and every eighth K block of 128 columns; a lane's 16 bytes of a row are one scale
// group. The eight warps' sums are added in shared memory in a fixed order (deterministic).
#include <algorithm>

#include "internal.h"
#include "launch.cuh"
#include "mxfp4.cuh"

namespace ce4b {

namespace {

constexpr int kWarps = 8;

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Weight bytes are read once: they leave the L1 cache to x.
__device__ __forceinline__ uint4 load_stream(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

template <int NT, int MT, bool SWIGLU>
__global__ void __launch_bounds__(32 * kWarps)
    mx4_vector_kernel(const bf16* x, const uint8_t* codes, const uint8_t* scales,
                      const bf16* residual, bf16* out, int rows, int n, int k) {
  constexpr int kCols = (SWIGLU ? 8 : 16) * MT;  // output columns per CTA
  __shared__ float part[kWarps][8 * NT][16 * MT + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int col0 = blockIdx.x * kCols, row0 = blockIdx.y * 8 * NT;
  const int kblocks = k / 128;
  grid_dependency_wait();
  grid_launch_dependents();

  // Fragment row h of tile m: weight rows past the last one read it again, unused.
  const uint8_t* code_ptr[MT][2];
  const uint8_t* scale_ptr[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int wrow = SWIGLU ? min(col0 + 8 * m + g, n - 1) + h * n : min(col0 + 16 * m + 8 * h + g, n - 1);
      code_ptr[m][h] = codes + static_cast<size_t>(wrow) * (k / 2) + t * 16;
      scale_ptr[m][h] = scales + static_cast<size_t>(wrow / 128) * kblocks * 512 + (wrow % 32) * 16 +
                        (wrow / 32 % 4) * 4 + t;
    }
  }
  const bf16* x_ptr[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    x_ptr[j] = row0 + 8 * j + g < rows ? x + static_cast<size_t>(row0 + 8 * j + g) * k + t * 32 : nullptr;
  }

  float acc[MT][NT][4] = {};
  uint4 q[MT][2];
  uint32_t sc[MT][2];
  auto load = [&](int kb) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        q[m][h] = load_stream(code_ptr[m][h] + kb * 64);
        sc[m][h] = scale_ptr[m][h][static_cast<size_t>(kb) * 512];
      }
    }
  };
  int kb = warp;
  if (kb < kblocks) load(kb);
  while (kb < kblocks) {
    uint4 xv[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        xv[j][i] = x_ptr[j] != nullptr ? *reinterpret_cast<const uint4*>(x_ptr[j] + static_cast<size_t>(kb) * 128 + i * 8)
                                       : make_uint4(0u, 0u, 0u, 0u);
      }
    }
    uint4 c[MT][2];
    uint32_t s[MT][2], f[MT][2], top = 0;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        c[m][h] = q[m][h];
        s[m][h] = sc[m][h];
        f[m][h] = mx4_factor(s[m][h]);
        top = max(top, s[m][h]);
      }
    }
    kb += kWarps;
    if (kb < kblocks) load(kb);
    const bool wide = __any_sync(0xffffffffu, top > 128u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint4 b[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) b[j] = permute_x(xv[j][i]);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        uint32_t a[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mx4_expand(i == 0 ? c[m][h].x : i == 1 ? c[m][h].y : i == 2 ? c[m][h].z : c[m][h].w, f[m][h], a[h]);
          if (wide) {
#pragma unroll
            for (int e = 0; e < 4; ++e) a[h][e] = mul_bf16x2(a[h][e], mx4_factor2(s[m][h]));
          }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          mma_bf16(acc[m][j], a[0][0], a[1][0], a[0][1], a[1][1], b[j].x, b[j].y);
          mma_bf16(acc[m][j], a[0][2], a[1][2], a[0][3], a[1][3], b[j].z, b[j].w);
        }
      }
    }
  }
  // A lane holds weight rows g and g + 8, activation rows 2t and 2t + 1 of each 8.
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) part[warp][8 * j + 2 * t + (e & 1)][16 * m + g + 8 * (e >> 1)] = acc[m][j][e];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 8 * NT * kCols; i += 32 * kWarps) {
    const int r = i / kCols, c = i % kCols;
    if (row0 + r >= rows || col0 + c >= n) continue;
    const int at_part = SWIGLU ? c / 8 * 16 + c % 8 : c;
    float y = 0.0f, u = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      y += part[w][r][at_part];
      if (SWIGLU) u += part[w][r][at_part + 8];
    }
    if (SWIGLU) y = y / (1.0f + expf(-y)) * u;
    const size_t at = static_cast<size_t>(row0 + r) * n + col0 + c;
    if (residual != nullptr) y += __bfloat162float(residual[at]);
    out[at] = __float2bfloat16_rn(y);
  }
}

template <int NT, int MT, bool SWIGLU>
void launch_vector(const bf16* x, const uint8_t* codes, const uint8_t* scales, const bf16* residual,
                   bf16* out, int rows, int n, int k, cudaStream_t s) {
  constexpr int kCols = (SWIGLU ? 8 : 16) * MT;
  const dim3 grid(static_cast<unsigned>((n + kCols - 1) / kCols), static_cast<unsigned>((rows + 8 * NT - 1) / (8 * NT)));
  launch(mx4_vector_kernel<NT, MT, SWIGLU>, grid, 32 * kWarps, 0, 0, s, x, codes, scales, residual, out, rows, n, k);
}

#ifndef VMT
#define VMT 1
#endif
template <bool SWIGLU>
void product(const bf16* x, const uint8_t* codes, const uint8_t* scales, const bf16* residual,
             bf16* out, int rows, int n, int k, cudaStream_t s) {
  if (rows <= 8) {
    launch_vector<1, VMT, SWIGLU>(x, codes, scales, residual, out, rows, n, k, s);
  } else if (rows <= 16) {
    launch_vector<2, VMT, SWIGLU>(x, codes, scales, residual, out, rows, n, k, s);
  } else if (rows <= 32) {
    launch_vector<4, VMT, SWIGLU>(x, codes, scales, residual, out, rows, n, k, s);
  } else {
    mx4_product_tc(x, codes, scales, residual, out, rows, n, k, SWIGLU, s);
  }
}

}  // namespace

void mx4_product(const bf16* x, const uint8_t* codes, const uint8_t* scales, const bf16* residual,
                 bf16* out, int rows, int n, int k, bool swiglu, cudaStream_t s) {
  if (swiglu) {
    product<true>(x, codes, scales, nullptr, out, rows, n, k, s);
  } else {
    product<false>(x, codes, scales, residual, out, rows, n, k, s);
  }
}

}  // namespace ce4b
