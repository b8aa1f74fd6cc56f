// Products of up to 32 BF16 activation rows with an MXFP4 weight (kernel-op API mxfp4_linear,
// mxfp4_swiglu), and the choice between this form and the tcgen05 one.
//
// The time is the weight's 0.53 bytes per element as long as a code costs at most three
// lane operations (an SM takes in about 43 codes a clock at the memory's rate and issues 128
// lane operations), of which expanding it to BF16 takes 2.1 (mxfp4.cuh). The rest is a
// warp-level MMA per 8 codes a lane and 8 rows, whose A fragment is made in the very registers
// that the codes were loaded into: no shared memory, no barrier and no hand-over between warps
// until the sums are joined, so that any number of warps hides the memory's latency. A warp
// takes one or two tiles of 16 weight rows (SwiGLU: 8 gate rows and their 8 up rows, which meet
// in one thread) and every eighth K block of 128 columns; a lane's 16 bytes of a row are one
// scale group. The eight warps' sums are added in shared memory in a fixed order
// (deterministic).
//
// 1 row, n = 512, k = 1536: 2.2 us, of which the launch is 1.5. 7 rows, n = 28672, k = 8192:
// 39.8 us (125 MB of weight, 3.2 TB/s), twice its bytes' time with no unit full: the load pipeline,
// busy 73 %, also takes x's 64-byte pieces, a scale byte for each 16 bytes of codes and the spills
// of the form used there (eight rows, two tiles a warp), which is held to 64 registers for four
// CTAs an SM and spills 72 bytes a thread; one tile's codes are in flight per warp. (x resident in
// shared memory with one CTA of 16 warps per SM and codes by asynchronous copies: 44 us; the
// tensor core's own E2M1 operand, which needs x in 8-bit terms made by a second kernel: 50 us.)
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

// The 64 codes a lane has of a K block (fragment rows g and g + 8 of the tile) times x's
// fragments, which fragment(j, i) gives for n-tile j and word i.
template <int NT, bool WIDE, class Fragment>
__device__ __forceinline__ void multiply_block(const uint4 (&q)[2], const uint32_t (&scale)[2], const Mx4Spread& spread,
                                               Fragment fragment, float (&acc)[NT][4]) {
  uint32_t f[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) f[h] = WIDE ? mx4_wide_factor(scale[h]) : mx4_factor(scale[h]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t a[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mx4_expand(i == 0 ? q[h].x : i == 1 ? q[h].y : i == 2 ? q[h].z : q[h].w, f[h], spread, a[h]);
      if constexpr (WIDE) {
#pragma unroll
        for (int e = 0; e < 4; ++e) a[h][e] = mul_bf16x2(a[h][e], mx4_factor2(scale[h]));
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const uint4 b = fragment(j, i);
      mma_bf16(acc[j], a[0][0], a[1][0], a[0][1], a[1][1], b.x, b.y);
      mma_bf16(acc[j], a[0][2], a[1][2], a[0][3], a[1][3], b.z, b.w);
    }
  }
}

template <int NT, class Fragment>
__device__ __forceinline__ void multiply_block(const uint4 (&q)[2], const uint32_t (&scale)[2], const Mx4Spread& spread,
                                               Fragment fragment, float (&acc)[NT][4]) {
  if (__any_sync(0xffffffffu, max(scale[0], scale[1]) > 128u)) {
    multiply_block<NT, true>(q, scale, spread, fragment, acc);
  } else {
    multiply_block<NT, false>(q, scale, spread, fragment, acc);
  }
}

template <int NT, int MT, bool SWIGLU>
__global__ void __launch_bounds__(32 * kWarps, NT == 1 ? 4 : NT == 2 ? 2 : 1)
    mx4_vector_kernel(const bf16* x, const uint8_t* codes, const uint8_t* scales,
                      const bf16* residual, bf16* out, int rows, int n, int k) {
  constexpr int kTileCols = SWIGLU ? 8 : 16;
  constexpr int kCols = MT * kTileCols;  // output columns per CTA
  __shared__ float part[kWarps][8 * NT][16 * MT + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int col0 = blockIdx.x * kCols, row0 = blockIdx.y * 8 * NT;
  const int kblocks = k / 128;
  grid_dependency_wait();
  grid_launch_dependents();

  // Weight rows past the last one read it again, unused.
  const uint8_t* code_ptr[MT][2];
  const uint8_t* scale_ptr[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int col = col0 + m * kTileCols + g;
      const int wrow = SWIGLU ? min(col, n - 1) + h * n : min(col + 8 * h, n - 1);
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

  const Mx4Spread spread;
  float acc[MT][NT][4] = {};
  uint4 next[2];
  uint32_t next_scale[2];
  auto load = [&](int m, int kb) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      next[h] = load_stream(code_ptr[m][h] + kb * 64);
      next_scale[h] = scale_ptr[m][h][static_cast<size_t>(kb) * 512];
    }
  };
  if (warp < kblocks) load(0, warp);
  for (int kb = warp; kb < kblocks; kb += kWarps) {
    uint4 xv[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        xv[j][i] = x_ptr[j] != nullptr ? permute_x(*reinterpret_cast<const uint4*>(x_ptr[j] + static_cast<size_t>(kb) * 128 + i * 8))
                                       : make_uint4(0u, 0u, 0u, 0u);
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const uint4 q[2] = {next[0], next[1]};
      const uint32_t scale[2] = {next_scale[0], next_scale[1]};
      if (m + 1 < MT) {
        load(m + 1, kb);
      } else if (kb + kWarps < kblocks) {
        load(0, kb + kWarps);
      }
      multiply_block<NT>(q, scale, spread, [&](int j, int i) { return xv[j][i]; }, acc[m]);
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
  const dim3 grid(static_cast<unsigned>((n - 1) / kCols + 1), static_cast<unsigned>((rows - 1) / (8 * NT) + 1));
  launch(mx4_vector_kernel<NT, MT, SWIGLU>, grid, 32 * kWarps, 0, 0, s, x, codes, scales, residual, out, rows, n, k);
}

// Two row tiles a warp read x once for both, which counts as soon as CTAs are many; one tile a
// warp spreads a small weight over more SMs. Measured (us, one tile | two): 7 rows 4096 x 4096
// 6.2 | 7.2, 28672 x 8192 45.2 | 39.7; 16 rows 1024 x 4096 6.6 | 6.9, 4096 x 4096 9.1 | 7.6,
// 28672 x 8192 79.6 | 55.4.
template <int NT, bool SWIGLU>
void choose_tiles(const bf16* x, const uint8_t* codes, const uint8_t* scales, const bf16* residual,
                  bf16* out, int rows, int n, int k, cudaStream_t s) {
  const int tiles = (n - 1) / (SWIGLU ? 8 : 16) + 1;
  if (tiles >= (NT == 1 ? 4 : 1) * sm_count()) {
    launch_vector<NT, 2, SWIGLU>(x, codes, scales, residual, out, rows, n, k, s);
  } else {
    launch_vector<NT, 1, SWIGLU>(x, codes, scales, residual, out, rows, n, k, s);
  }
}

// Up to 16 rows this form is the faster one at every size. With 17 to 32 rows the MMAs and x's
// fragments weigh more than the codes, and the tcgen05 form wins once its fixed 6 us are
// spread over enough codes. us, this form | tcgen05, n x k:
//            512 x 1536  1024 x 2048  2048 x 2048  1024 x 4096  4096 x 4096  28672 x 8192
//   17 rows  3.5 | 6.3   4.2 | 6.2    4.5 | 6.2    6.5 | 6.4    9.1 | 9.1    92 | 53
//   24 rows  3.8 | 6.5   4.7 | 6.2    4.8 | 6.3    6.8 | 6.5    9.6 | 9.2    92 | 53
//   32 rows  4.3 | 6.6   5.2 | 6.6    5.4 | 6.6    8.0 | 6.6    10.4 | 9.5   101 | 53
// The limit is 2^21 codes. Between 2 and 4 million the better form also depends on k (eight warps
// share k here), which the rule leaves out.
template <bool SWIGLU>
void product(const bf16* x, const uint8_t* codes, const uint8_t* scales, const bf16* residual,
             bf16* out, int rows, int n, int k, cudaStream_t s) {
  const int64_t weight = static_cast<int64_t>(n) * k * (SWIGLU ? 2 : 1);
  if (rows > 32 || (rows > 16 && weight > (1 << 21))) {
    mx4_product_tc(x, codes, scales, residual, out, rows, n, k, SWIGLU, s);
  } else if (rows <= 8) {
    choose_tiles<1, SWIGLU>(x, codes, scales, residual, out, rows, n, k, s);
  } else if (rows <= 16) {
    choose_tiles<2, SWIGLU>(x, codes, scales, residual, out, rows, n, k, s);
  } else {
    choose_tiles<4, SWIGLU>(x, codes, scales, residual, out, rows, n, k, s);
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
