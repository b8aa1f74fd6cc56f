// Residual addition and RMSNorm of rows (kernel-op API add_rmsnorm_forward and
// add_rmsnorm_mxfp8): s = bf16(x + residual), n = bf16(s * (mean(s^2) + eps)^(-1/2) * w), n as
// BF16 or as the MXFP8 codes and scales of that BF16 value.
#include <algorithm>

#include "internal.h"
#include "launch.cuh"
#include "mxfp8.cuh"
#include "ptx.cuh"

namespace ce4b {

namespace {

// n is the BF16 rounding of the formula's FP32 value: the squares (exact in 64 bits) are summed
// in 64 bits and the factor (mean + eps)^(-1/2) is kept as an FP32 pair hi + lo. A row's result
// then depends neither on its neighbours nor on the order of its sum, which goes with the launch
// shape, unless the formula's value lies within about 2^-40 (relative) of a border between two
// BF16 values: a 64-bit sum of squares over more than 53 binades rounds too. The MXFP8 form
// quantises the BF16 n.
struct RowScale {
  float power;   // 2^e, about the factor's size
  float hi, lo;  // factor / 2^e = hi + lo, lo >= 0
};

__device__ __forceinline__ RowScale row_scale(double sum, double inv_width, float eps) {
  const double f = rsqrt(fma(sum, inv_width, static_cast<double>(eps)));
  RowScale r;
  if (f > 0.0 && f <= 3.0e300) {
    const int e = min(static_cast<int>((__double2hiint(f) >> 20) & 0x7FF) - 1023, 127);
    const double m = f * __hiloint2double((1023 - e) << 20, 0);
    r.power = static_cast<float>(__hiloint2double((1023 + e) << 20, 0));
    r.hi = __double2float_rz(m);
    // Never 0: a product that overflows stays infinite when multiplied by it.
    r.lo = fmaxf(static_cast<float>(m - static_cast<double>(r.hi)), 0x1p-60f);
  } else {  // 0 beside an infinity, infinite for a row of zeros without eps, NaN
    r.power = static_cast<float>(f);
    r.hi = 1.0f;
    r.lo = 0x1p-60f;
  }
  return r;
}

// s * factor * w rounded to FP32 once. s * 2^e is exact and of the size of s * factor, so its
// product with w (eight bits each: exact) overflows only where the result does; the last FMA
// rounds the exact p * hi plus p * lo. Values under FP32's normal numbers, 2^-126, are the
// exception: s * 2^e and p are multiples of 2^-149 there, so that an s over 2^142 below its row's
// size loses bits and one over 2^150 below counts as 0, however large w is, as in any FP32 form.
__device__ __forceinline__ float scale_product(float s, float w, const RowScale& f) {
  const float p = s * f.power * w;
  return fmaf(p, f.hi, p * f.lo);
}

// Sum over each group of WIDTH lanes.
template <int WIDTH>
__device__ __forceinline__ double lane_sum(double v) {
#pragma unroll
  for (int o = WIDTH / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Elements from..to-1 of a chunk of eight, the others 0.
__device__ __forceinline__ uint4 keep(const uint4& q, int from, int to) {
  uint32_t v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (2 * j < from || 2 * j >= to) v[j] &= 0xFFFF0000u;
    if (2 * j + 1 < from || 2 * j + 1 >= to) v[j] &= 0x0000FFFFu;
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// The chunk of eight BF16 values at p, of which `limit` exist (at least one): a 16-byte load,
// or single elements at the end of the buffer.
__device__ __forceinline__ uint4 load_chunk(const bf16* p, int64_t limit) {
  if (limit >= 8) return *reinterpret_cast<const uint4*>(p);
  uint32_t v[4] = {};
  const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j < limit) v[j / 2] |= static_cast<uint32_t>(u[j]) << (16 * (j % 2));
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// Elements o..o+7 (o = 0..7) of the sixteen of a and b.
__device__ __forceinline__ uint4 window(const uint4& a, const uint4& b, int o) {
  uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int j = 0; j < 6; ++j) v[j] = o & 4 ? v[j + 2] : v[j];
#pragma unroll
  for (int j = 0; j < 5; ++j) v[j] = o & 2 ? v[j + 1] : v[j];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = o & 1 ? __funnelshift_r(v[j], v[j + 1], 16) : v[j];
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// Stores elements from..to-1 of a chunk; a neighbouring row owns the others.
__device__ __forceinline__ void store_chunk(bf16* p, const uint32_t (&v)[4], int from, int to) {
  if (from == 0 && to == 8) {
    *reinterpret_cast<uint4*>(p) = make_uint4(v[0], v[1], v[2], v[3]);
    return;
  }
  uint16_t* u = reinterpret_cast<uint16_t*>(p);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j >= from && j < to) u[j] = static_cast<uint16_t>(v[j / 2] >> (16 * (j % 2)));
  }
}

// A row is held in the registers of TPR threads, V chunks of eight columns each, and read and
// written once. ALIGNED: rows start and end on 16 bytes (width % 8 == 0), and a thread keeps
// its part of w over the rows it takes. Otherwise chunks are the aligned 16 bytes of the
// matrix: the row's first and last one hold elements of its neighbours, which are masked
// after the load and left out of the store, and w is shifted to the row's offset.
//
// Blocks are as small as a row allows, so that their steps interleave: 256 threads for four rows
// of 1021 x 769 took 4.4 us, 128 for one take 3.1; to MXFP8 65536 x 1024 took 83, takes 77.
//
// Bound by memory: 65536 x 1024 takes 85.2 us, 6.3 TB/s of the 6.56 a copy reaches, to MXFP8 77.1
// (6.1 TB/s). Where the MXFP8 form's 28 instructions an element do not hide as well it stays
// below: 16384 x 2048 takes 42.0 us (5.6 TB/s). Rows off 16 bytes pay their ends: 65536 x 769 takes
// 88 us (4.6 TB/s). One row of 512 takes 1.5 us, a launch.
// w too may be what the predecessor writes while this kernel starts, so it takes ordinary loads.
template <int V, int TPR>
constexpr int norm_threads() {
  return TPR > (V >= 2 ? 32 : 64) ? TPR : (V >= 2 ? 32 : 64);
}

template <int V, int TPR, bool ALIGNED, bool MX>
__global__ void __launch_bounds__(norm_threads<V, TPR>())
    add_rmsnorm_kernel(const bf16* x, const bf16* residual, const bf16* w, bf16* sum,
                       bf16* out, uint8_t* codes, uint8_t* scales, int rows, int width,
                       double inv_width, float eps) {
  constexpr int kThreads = norm_threads<V, TPR>();
  constexpr int kRows = kThreads / TPR;  // rows of a block at a time
  constexpr int kWarps = TPR < 32 ? 1 : TPR / 32;  // warps of a row
  __shared__ double part[2][kThreads / 32];
  const int lane = threadIdx.x % TPR;
  grid_dependency_wait();
  grid_launch_dependents();
  // w is loaded ahead of the row's sum, or, where registers are short, at its use.
  constexpr bool kKeepW = V <= 2;
  auto load_w = [&](int c, int shift) {  // columns c - shift .. + 7 of w
    if constexpr (ALIGNED) return *reinterpret_cast<const uint4*>(w + c);
    uint4 a = make_uint4(0u, 0u, 0u, 0u), b = a;
    if (shift > 0 && c > 0) a = load_chunk(w + c - 8, width - c + 8);
    if (c < width) b = load_chunk(w + c, width - c);
    return shift > 0 ? window(a, b, 8 - shift) : b;
  };
  uint4 wv[V];
  if constexpr (ALIGNED && kKeepW) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (i * TPR + lane) * 8;
      wv[i] = c < width ? *reinterpret_cast<const uint4*>(w + c) : make_uint4(0u, 0u, 0u, 0u);
    }
  }
  const int64_t total = static_cast<int64_t>(rows) * width;
  const int last = MX ? (rows + 127) / 128 * 128 : rows;
  int turn = 0;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * kRows; r0 < last;
       r0 += static_cast<int64_t>(gridDim.x) * kRows, turn ^= 1) {
    const int64_t row = r0 + threadIdx.x / TPR;
    const bool live = row < rows;
    // The row's chunks start at element `begin` of the matrix; column 0 is `shift` after it.
    const int64_t first = row * width;
    const int shift = ALIGNED ? 0 : static_cast<int>(first & 7);
    const int64_t begin = first - shift;
    uint4 v[V], r[V];
    auto bounds = [&](int i, int& from, int& to) {
      const int c = (i * TPR + lane) * 8;  // of the chunks' elements
      from = ALIGNED ? 0 : max(shift - c, 0);
      to = ALIGNED ? 8 : min(shift + width - c, 8);
      return live && (ALIGNED ? c < width : c < shift + width);
    };
#pragma unroll
    for (int i = 0; i < V; ++i) {
      int from, to;
      const bool own = bounds(i, from, to);
      const int64_t at = begin + (i * TPR + lane) * 8;
      v[i] = r[i] = make_uint4(0u, 0u, 0u, 0u);
      if constexpr (ALIGNED) {
        if (own) v[i] = *reinterpret_cast<const uint4*>(x + at);
        if (own && residual != nullptr) r[i] = *reinterpret_cast<const uint4*>(residual + at);
      } else if (own) {
        v[i] = load_chunk(x + at, total - at);
        if (residual != nullptr) r[i] = load_chunk(residual + at, total - at);
        if (from > 0 || to < 8) {
          v[i] = keep(v[i], from, to);
          r[i] = keep(r[i], from, to);
        }
      }
    }
    if constexpr (!ALIGNED && kKeepW) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        int from, to;
        wv[i] = make_uint4(0u, 0u, 0u, 0u);
        if (bounds(i, from, to)) wv[i] = load_w((i * TPR + lane) * 8, shift);
      }
    }
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      uint32_t* q = reinterpret_cast<uint32_t*>(&v[i]);
      const uint32_t* p = reinterpret_cast<const uint32_t*>(&r[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 s = unpack_bf16x2(q[j]);
        if (residual != nullptr) {
          const float2 t = unpack_bf16x2(p[j]);
          q[j] = pack_bf16x2(s.x + t.x, s.y + t.y);
          s = unpack_bf16x2(q[j]);
        }
        const double a = s.x, b = s.y;
        ss = fma(a, a, ss);
        ss = fma(b, b, ss);
      }
      int from, to;
      if (residual != nullptr && bounds(i, from, to)) {
        const uint32_t words[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        store_chunk(sum + begin + (i * TPR + lane) * 8, words, from, to);
      }
    }
    ss = lane_sum<TPR < 32 ? TPR : 32>(ss);
    if constexpr (kWarps > 1) {
      const int warp = threadIdx.x / 32;
      if (threadIdx.x % 32 == 0) part[turn][warp] = ss;
      __syncthreads();
      ss = 0.0;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) ss += part[turn][warp / kWarps * kWarps + i];
    }
    const RowScale f = row_scale(ss, inv_width, eps);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      int from, to;
      const bool own = bounds(i, from, to);
      const uint32_t* q = reinterpret_cast<const uint32_t*>(&v[i]);
      const int c = (i * TPR + lane) * 8;
      float n[8];
      uint4 wi = make_uint4(0u, 0u, 0u, 0u);
      if constexpr (kKeepW) {
        wi = wv[i];
      } else if (own) {
        wi = load_w(c, shift);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 s = unpack_bf16x2(q[j]);
        const float2 u = unpack_bf16x2(reinterpret_cast<const uint32_t*>(&wi)[j]);
        n[2 * j] = scale_product(s.x, u.x, f);
        n[2 * j + 1] = scale_product(s.y, u.y, f);
      }
      uint32_t words[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) words[j] = pack_bf16x2(n[2 * j], n[2 * j + 1]);
      if constexpr (!MX) {
        if (own) store_chunk(out + begin + c, words, from, to);
      } else {
        // Four neighbouring threads hold the 32 columns of a scale block.
        float m[8], amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 t = unpack_bf16x2(words[j]);
          m[2 * j] = t.x, m[2 * j + 1] = t.y;
          amax = fmaxf(amax, fmaxf(fabsf(t.x), fabsf(t.y)));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const uint8_t sc = mx_scale_code(amax);
        const float inv = mx_scale_inverse(sc);
        uint2 e;
        e.x = mx_codes4(m[0], m[1], m[2], m[3], inv);
        e.y = mx_codes4(m[4], m[5], m[6], m[7], inv);
        if (own) *reinterpret_cast<uint2*>(codes + first + c) = e;
        if (row < last && c < width && lane % 4 == 0) {
          scales[mx_scale_offset(static_cast<int>(row), c / 32, width / 128)] = live ? sc : 0;
        }
      }
    }
  }
}

// Any width, alignment and form, one block per row (rows in blockIdx.x): rows too wide for the
// registers above, and matrices whose buffers start off 16 bytes. The row's sum is read again
// (from the cache) for the second pass. Columns are counted unsigned: the last one's successors
// pass 2^31.
__global__ void add_rmsnorm_any_kernel(const bf16* x, const bf16* residual, const bf16* w, bf16* sum,
                                       bf16* out, uint8_t* codes, uint8_t* scales, int rows,
                                       uint32_t width, double inv_width, float eps) {
  __shared__ double part[32];
  const int row = blockIdx.x;
  if (row >= rows) {  // padding rows of the last scale tile
    for (uint32_t b = threadIdx.x; b < width / 32; b += blockDim.x) scales[mx_scale_offset(row, b, width / 128)] = 0;
    return;
  }
  const size_t at = static_cast<size_t>(row) * width;
  double ss = 0.0;
  const uint32_t step = blockDim.x;
  for (uint32_t c0 = threadIdx.x; c0 < width; c0 += 4 * step) {
    float s[4], r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t c = c0 + j * step;
      s[j] = c < width ? __bfloat162float(x[at + c]) : 0.0f;
      r[j] = c < width && residual != nullptr ? __bfloat162float(residual[at + c]) : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t c = c0 + j * step;
      if (residual != nullptr && c < width) {
        s[j] = bf16_round(s[j] + r[j]);
        sum[at + c] = __float2bfloat16_rn(s[j]);
      }
      ss = fma(static_cast<double>(s[j]), static_cast<double>(s[j]), ss);
    }
  }
  ss = lane_sum<32>(ss);
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = ss;
  __syncthreads();  // also before the sum of other threads' columns is read below
  ss = 0.0;
  for (int i = 0; i < static_cast<int>(blockDim.x) / 32; ++i) ss += part[i];
  const RowScale f = row_scale(ss, inv_width, eps);
  const bf16* src = residual != nullptr ? sum : x;
  if (codes == nullptr) {
#pragma unroll 4
    for (uint32_t c = threadIdx.x; c < width; c += step) {
      out[at + c] = __float2bfloat16_rn(
          scale_product(__bfloat162float(src[at + c]), __bfloat162float(w[c]), f));
    }
    return;
  }
  for (uint32_t b = threadIdx.x; b < width / 32; b += blockDim.x) {
    float v[32];
    for (int j = 0; j < 32; ++j) {
      v[j] = bf16_round(scale_product(__bfloat162float(src[at + b * 32 + j]), __bfloat162float(w[b * 32 + j]), f));
    }
    uint32_t q[8];
    const uint8_t sc = mx_quantize32(v, q);
    uint32_t* dst = reinterpret_cast<uint32_t*>(codes + at + b * 32);
    for (int j = 0; j < 8; ++j) dst[j] = q[j];
    scales[mx_scale_offset(row, b, width / 128)] = sc;
  }
}

struct NormArgs {
  const bf16 *x, *residual, *w;
  bf16 *sum, *out;
  uint8_t *codes, *scales;
  int rows, width;
  float eps;
  cudaStream_t s;
};

template <int V, int TPR, bool ALIGNED, bool MX>
void launch_norm(const NormArgs& a) {
  constexpr int kThreads = norm_threads<V, TPR>();
  constexpr int kRows = kThreads / TPR;
  const int64_t rows = MX ? (static_cast<int64_t>(a.rows) + 127) / 128 * 128 : a.rows;
  // Blocks that take rows in turn, 2048 threads an SM. The forms for many rows use 54 to 64
  // registers a thread, so that about half of these blocks are on the GPU at once and the others
  // follow as they leave; a block for every row was slower at most sizes.
  const int64_t grid = std::min<int64_t>((rows + kRows - 1) / kRows, static_cast<int64_t>(sm_count()) * (2048 / kThreads));
  launch(add_rmsnorm_kernel<V, TPR, ALIGNED, MX>, dim3(static_cast<unsigned>(grid)), kThreads, 0, 0, a.s,
         a.x, a.residual, a.w, a.sum, a.out, a.codes, a.scales, a.rows, a.width, 1.0 / a.width, a.eps);
}

template <bool ALIGNED, bool MX>
bool launch_rows(const NormArgs& a) {
  const int chunks = ALIGNED ? a.width / 8 : (a.width + 14) / 8;
  // Few rows: as many threads per row as it has chunks, for the shortest chain. Many rows: two
  // chunks a thread, w beside them in registers; the MXFP8 form and rows off 16 bytes, which do
  // more per row and thread, four, w read at its use. us with 1 | 2 | 4 chunks: 16384 x 2048 54.2 |
  // 42.7 | 44.4, to MXFP8 60.8 | 45.8 | 41.5, 10000 x 3001 - | 63.6 | 50.0. Rows wider than 16384 are
  // one block's with eight chunks a thread.
  const bool few = static_cast<int64_t>(a.rows) * chunks <= static_cast<int64_t>(sm_count()) * 2048;
  if (chunks <= 8) return launch_norm<1, 8, ALIGNED, MX>(a), true;
  if (chunks <= 16) return launch_norm<1, 16, ALIGNED, MX>(a), true;
  if (few && chunks <= 1024) {
    if (chunks <= 32) return launch_norm<1, 32, ALIGNED, MX>(a), true;
    if (chunks <= 64) return launch_norm<1, 64, ALIGNED, MX>(a), true;
    if (chunks <= 128) return launch_norm<1, 128, ALIGNED, MX>(a), true;
    if (chunks <= 256) return launch_norm<1, 256, ALIGNED, MX>(a), true;
    if (chunks <= 512) return launch_norm<1, 512, ALIGNED, MX>(a), true;
    return launch_norm<1, 1024, ALIGNED, MX>(a), true;
  }
  if (chunks <= 32) return launch_norm<1, 32, ALIGNED, MX>(a), true;
  if (chunks <= 64) return launch_norm<2, 32, ALIGNED, MX>(a), true;
  if constexpr (ALIGNED && !MX) {
    if (chunks <= 128) return launch_norm<2, 64, ALIGNED, MX>(a), true;
    if (chunks <= 256) return launch_norm<2, 128, ALIGNED, MX>(a), true;
    if (chunks <= 512) return launch_norm<2, 256, ALIGNED, MX>(a), true;
    if (chunks <= 1024) return launch_norm<2, 512, ALIGNED, MX>(a), true;
  } else {
    if (chunks <= 128) return launch_norm<4, 32, ALIGNED, MX>(a), true;
    if (chunks <= 256) return launch_norm<4, 64, ALIGNED, MX>(a), true;
    if (chunks <= 512) return launch_norm<4, 128, ALIGNED, MX>(a), true;
    if (chunks <= 1024) return launch_norm<4, 256, ALIGNED, MX>(a), true;
  }
  if (chunks <= 2048) return launch_norm<2, 1024, ALIGNED, MX>(a), true;
  if (chunks <= 4096) return launch_norm<8, 512, ALIGNED, MX>(a), true;
  return false;
}

}  // namespace

void add_rmsnorm_rows(const bf16* x, const bf16* residual, const bf16* w, bf16* sum, bf16* out,
                      uint8_t* codes, uint8_t* scales, int rows, int width, float eps,
                      cudaStream_t s) {
  const NormArgs a{x, residual, w, sum, out, codes, scales, rows, width, eps, s};
  auto wide = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  const bool mx = codes != nullptr;
  if (wide(x) && wide(residual) && wide(w) && (residual == nullptr || wide(sum)) && (mx || wide(out))) {
    const bool aligned = width % 8 == 0;
    if (mx ? launch_rows<true, true>(a) : aligned ? launch_rows<true, false>(a) : launch_rows<false, false>(a)) {
      return;
    }
  }
  const int grid = mx ? (rows + 127) / 128 * 128 : rows;
  add_rmsnorm_any_kernel<<<grid, width > 4096 ? 1024 : 256, 0, s>>>(x, residual, w, sum, out, codes, scales, rows, width,
                                              1.0 / width, eps);
  check_cuda(cudaGetLastError(), "add_rmsnorm launch");
}

}  // namespace ce4b
