// Products of 17 and more BF16 activation rows with an MXFP4 weight (kernel-op API mxfp4_linear,
// mxfp4_swiglu): y[r, n] = sum_k x[r, k] * code[n, k] * 2^(scale[n, k / 32] - 127).
//
// The weight is the A operand of tcgen05 MMAs (128 weight rows are the 128 lanes of tensor
// memory, up to 64 activation rows the N columns): every code is expanded once, in registers, to
// the BF16 value it stands for (E2M1 times a power of two is exact in BF16), and stored to
// tensor memory, from which the MMA reads A without passing through shared memory, whose
// bandwidth 32 KB per K block in and out would fill. Products are exact, sums are FP32.
//
// A CTA takes 128 weight rows (SwiGLU: 64 gate rows and their 64 up rows) and a slice of K. Four
// warps copy codes and scales asynchronously into a ring, TMA brings x tiles beside them,
// eight warps expand, one thread issues the MMAs. (Codes by TMA come in boxes of 64-byte rows,
// whose requests alone took 33 us at n = 28672, k = 8192.) A cluster of up to eight CTAs shares
// the K blocks of one row tile, so that weights of few rows still occupy the GPU; their FP32
// partial sums are added through distributed shared memory in rank order (deterministic).
//
// Bound, at 64 rows: a launch whose CTAs have four K blocks each takes 6.6 us (n = 1024, k = 512),
// 9.7 with two CTAs on every SM (n = 37888, k = 512); every further K block of an SM 0.43 us of
// expansion, MMA and hand-over, where its bytes take 0.2 (n = 37888, k = 8192: 60.9 us). n = 28672,
// k = 8192 takes 61 us too (125 MB of weight, 2.1 TB/s, 0.49 PFLOP/s), because its 224 row tiles
// fill 76 SMs with two CTAs and leave one to each of the other 72. n = 1024, k = 4096, split over
// clusters of eight, takes 8.1 us.
#include <algorithm>

#include "internal.h"
#include "launch.cuh"
#include "mxfp4.cuh"
#include "ptx.cuh"

namespace ce4b {

namespace {

constexpr int kM = 128;            // weight rows per CTA
constexpr int kKB = 128;           // K elements per ring stage
constexpr int kExpandWarps = 8;
constexpr int kCopyThreads = 128;
constexpr int kThreads = 64 + 32 * kExpandWarps + kCopyThreads;
constexpr int kABuffers = 3;       // expanded K blocks in tensor memory, 64 columns each
constexpr int kACol = 64;          // first column of the A buffers (D before it)
constexpr uint32_t kTmemCols = 256;
constexpr int kMaxSplit = 8;

template <int R>
struct ProductSmem {
  static constexpr int kCodeBytes = kM * kKB / 2;
  static constexpr int kXBytes = R * kKB * 2;
  static constexpr int kSfBytes = 1024;  // four scale bytes a row
  static constexpr int kStageBytes = kCodeBytes + kXBytes + kSfBytes;
  // Two CTAs per SM: while one drains its pipeline the other streams.
  static constexpr int kStages = (113 * 1024 - 2048) / kStageBytes;
  static constexpr int kRingBytes = kStages * kStageBytes;
  static constexpr int kBars = 2 * kStages + 2 * kABuffers + 1;
  static constexpr int kBytes = 1024 + kRingBytes + kBars * 8 + 8;
  static_assert(kStageBytes % 1024 == 0, "stages must stay 1024-byte aligned");
  static_assert(kStages >= 3 && kRingBytes >= R * kM * 4, "the ring holds the partial sums");
  static_assert(kBytes <= 113 * 1024, "two CTAs must fit on an SM");
};

// The 32 codes of one group (16 bytes) as 16 registers of two BF16 values each.
template <bool WIDE>
__device__ __forceinline__ void expand_group(const uint4& q, uint32_t scale, const Mx4Spread& m, uint32_t* out) {
  const uint32_t f = WIDE ? mx4_wide_factor(scale) : mx4_factor(scale);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v[4];
    mx4_expand(w[i], f, m, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) out[4 * i + j] = WIDE ? mul_bf16x2(v[j], mx4_factor2(scale)) : v[j];
  }
}

__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ void copy_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// Arrives on the barrier once this thread's copies so far have landed.
__device__ __forceinline__ void copy_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

template <int R, bool SWIGLU>
__global__ void __launch_bounds__(kThreads, 2)
    mx4_product_kernel(const __grid_constant__ CUtensorMap tm_x, const uint8_t* codes,
                       const uint8_t* scales, const bf16* residual, bf16* out, int rows, int n, int kblocks, int split,
                       int* err) {
  using L = ProductSmem<R>;
  constexpr int NS = L::kStages;
  constexpr int kCols = SWIGLU ? 64 : 128;  // output columns per CTA

  extern __shared__ uint8_t smem_raw[];
  uint32_t base = smem_u32(smem_raw);
  const uint32_t pad = (1024u - (base & 1023u)) & 1023u;
  uint8_t* smem = smem_raw + pad;
  base += pad;
  const uint32_t bars = base + L::kRingBytes;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (NS + s); };
  auto afull_bar = [&](int a) { return bars + 8u * (2 * NS + a); };
  auto aempty_bar = [&](int a) { return bars + 8u * (2 * NS + kABuffers + a); };
  const uint32_t done_bar = bars + 8u * (2 * NS + 2 * kABuffers);
  volatile uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kRingBytes + L::kBars * 8);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % split;
  const int tile = static_cast<int>(blockIdx.x) / split;
  const int row0 = static_cast<int>(blockIdx.y) * R;
  const int kb0 = kblocks * rank / split, kb1 = kblocks * (rank + 1) / split;
  const int w0 = tile * kCols;
  // Weight row of tile row r; rows past the last one (of its half) read it again, unused.
  auto weight_row = [&](int r) {
    return SWIGLU ? min(w0 + r % 64, n - 1) + (r / 64) * n : min(w0 + r, n - 1);
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(full_bar(s), 1 + kCopyThreads);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < kABuffers; ++a) {
      mbar_init(afull_bar(a), 4);
      mbar_init(aempty_bar(a), 1);
    }
    mbar_init(done_bar, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), kTmemCols);
    tmem_relinquish();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dependency_wait();
  grid_launch_dependents();

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&tm_x);
      int it = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int s = it % NS;
        if (!mbar_wait(empty_bar(s), ((it / NS) & 1) ^ 1)) {
          record_error(err, kErrTimeoutProducer);
          ok = false;
          break;
        }
        const uint32_t xs = base + s * L::kStageBytes + L::kCodeBytes;
        mbar_arrive_expect_tx(full_bar(s), L::kXBytes);
        tma_load_2d(xs, &tm_x, full_bar(s), kb * kKB, row0);
        tma_load_2d(xs + L::kXBytes / 2, &tm_x, full_bar(s), kb * kKB + 64, row0);
      }
      if (!ok) {  // the copies in flight land before the CTA may end
        for (int i = max(0, it - NS); i < it; ++i) mbar_wait(full_bar(i % NS), (i / NS) & 1);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_bf16(kM, R);
      int it = 0;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int s = it % NS, a = it % kABuffers;
        // The expanding warps have seen the stage land; this thread reads its x tile.
        if (!mbar_wait(full_bar(s), (it / NS) & 1) || !mbar_wait(afull_bar(a), (it / kABuffers) & 1)) {
          record_error(err, kErrTimeoutMma);
          break;
        }
        tc_fence_after();
        const uint32_t xs = base + s * L::kStageBytes + L::kCodeBytes;
        const uint32_t at = tmem + kACol + 64u * a;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          umma_bf16_ts(tmem, at + 8u * j, sdesc_k128(xs + (j / 4) * (L::kXBytes / 2)) + 2u * (j % 4),
                       idesc, (it | j) != 0 ? 1u : 0u);
        }
        umma_commit(empty_bar(s));
        umma_commit(aempty_bar(a));
      }
      umma_commit(done_bar);
    }
    __syncwarp();
  } else if (warp >= 2 + kExpandWarps) {
    const int ct = threadIdx.x - 64 - 32 * kExpandWarps;
    const uint8_t* src[4];  // 16 bytes (a scale group) of rows ct / 4 + 32 i
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      src[i] = codes + (static_cast<size_t>(weight_row(i * 32 + ct / 4)) * kblocks + kb0) * 64 + ct % 4 * 16;
    }
    const uint32_t dst = (ct / 4) * 64 + (((ct % 4) ^ (ct / 8 & 3)) << 4);
    const int sr = weight_row(ct);
    const uint8_t* scale_src = scales + (static_cast<size_t>(sr / 128) * kblocks + kb0) * 512 + (sr % 32) * 16 + (sr / 32 % 4) * 4;
    for (int it = 0; it < kb1 - kb0; ++it) {
      const int s = it % NS;
      if (!mbar_wait(empty_bar(s), ((it / NS) & 1) ^ 1)) {
        record_error(err, kErrTimeoutProducer);
        break;
      }
      const uint32_t stage = base + s * L::kStageBytes;
#pragma unroll
      for (int i = 0; i < 4; ++i) copy_async16(stage + dst + i * 32 * 64, src[i] + it * 64);
      copy_async4(stage + L::kCodeBytes + L::kXBytes + ct * 4, scale_src + static_cast<size_t>(it) * 512);
      copy_arrive(full_bar(s));
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    // Four warps cover the 128 lanes; the first four expand the even stages, the others the odd.
    const int turn = (warp - 2) / 4;
    const int r = (warp & 3) * 32 + lane;           // weight row in the tile = lane of TMEM
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t sf_off = L::kCodeBytes + L::kXBytes + r * 4;
    const uint32_t swz = (r >> 1) & 3;
    const Mx4Spread spread;
    for (int it = turn; it < kb1 - kb0; it += 2) {
      const int s = it % NS, a = it % kABuffers;
      if (!mbar_wait(full_bar(s), (it / NS) & 1)) {
        record_error(err, kErrTimeoutEpilogue);
        break;
      }
      const uint32_t stage = base + s * L::kStageBytes;
      const uint32_t row = stage + r * 64;
#pragma unroll
      for (int i = 0; i < R * 16 / 128; ++i) {
        const uint32_t at = stage + L::kCodeBytes + (i * 128 + r) * 16;
        st_shared_v4(at, permute_x(ld_shared_v4(at)));
      }
      fence_proxy_async_smem();
      const uint32_t sf = __float_as_uint(ld_shared_f32(stage + sf_off));
      if (!mbar_wait(aempty_bar(a), ((it / kABuffers) & 1) ^ 1)) {
        record_error(err, kErrTimeoutEpilogue);
        break;
      }
      tc_fence_after();
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h) {
        const uint4 q0 = ld_shared_v4(row + (((2u * h) ^ swz) << 4));
        const uint4 q1 = ld_shared_v4(row + (((2u * h + 1u) ^ swz) << 4));
        const uint32_t s0 = (sf >> (16u * h)) & 255u, s1 = (sf >> (16u * h + 8u)) & 255u;
        uint32_t v[32];
        if (__any_sync(0xffffffffu, max(s0, s1) > 128u)) {
          expand_group<true>(q0, s0, spread, v);
          expand_group<true>(q1, s1, spread, v + 16);
        } else {
          expand_group<false>(q0, s0, spread, v);
          expand_group<false>(q1, s1, spread, v + 16);
        }
        tmem_st32(tmem + lane_base + kACol + 64u * a + 32u * h, v);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(afull_bar(a));
    }
    // Partial sums [activation row][weight row] in FP32, over the ring.
    if (turn == 0) {
      if (!mbar_wait(done_bar, 0)) record_error(err, kErrTimeoutEpilogue);
      tc_fence_after();
      float* part = reinterpret_cast<float*>(smem);
#pragma unroll
      for (int c = 0; c < R; c += 16) {
        uint32_t v[16];
        tmem_ld16(tmem + lane_base + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(c + j) * kM + r] = __uint_as_float(v[j]);
      }
      tc_fence_before();
    }
  }

  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
  if (split > 1) cluster_sync_all();
  // Every CTA of the cluster finishes its share of the activation rows, two columns a thread.
  constexpr int kPairs = kCols / 2;
  const int mine = min(R, rows - row0);
  for (int i = threadIdx.x; i < (mine - rank + split - 1) / split * kPairs; i += kThreads) {
    const int b = rank + i / kPairs * split, c = i % kPairs * 2;
    float2 y = make_float2(0.0f, 0.0f), u = make_float2(0.0f, 0.0f);
    for (int p = 0; p < split; ++p) {
      const uint32_t at = split > 1 ? mapa_shared(base, p) : base;
      const float2 v = ld_cluster_f32x2(at + (b * kM + c) * 4);
      y.x += v.x, y.y += v.y;
      if constexpr (SWIGLU) {
        const float2 v2 = ld_cluster_f32x2(at + (b * kM + 64 + c) * 4);
        u.x += v2.x, u.y += v2.y;
      }
    }
    if constexpr (SWIGLU) {
      y.x = y.x / (1.0f + expf(-y.x)) * u.x;
      y.y = y.y / (1.0f + expf(-y.y)) * u.y;
    }
    const int col = w0 + c;
    const size_t at = static_cast<size_t>(row0 + b) * n + col;
    if (residual != nullptr) {
      if (col < n) y.x += __bfloat162float(residual[at]);
      if (col + 1 < n) y.y += __bfloat162float(residual[at + 1]);
    }
    if (col < n) out[at] = __float2bfloat16_rn(y.x);
    if (col + 1 < n) out[at + 1] = __float2bfloat16_rn(y.y);
  }
  if (split > 1) cluster_sync_all();  // a peer may still read this CTA's sums
}

// CTAs per row tile: as many as fit on the GPU at once (two an SM), with at least four K blocks
// each. A launch costs about 5 us beside its blocks (tensor memory, first bytes, join), 0.43 us
// each, so that a second wave never pays: 33 rows, n = 8192 (SwiGLU), k = 2048 takes 13.9 us
// unsplit, 12.9 at 2 and 19.4 at 3, the first split of more CTAs than fit. A whole number of CTAs
// a tile leaves SMs with one CTA beside others with two: with 149 to 295 tiles, unsplit, the time
// is that of 296.
int choose_split(int64_t tiles, int kblocks) {
  const int fit = static_cast<int>(2 * sm_count() / tiles);
  return std::max(1, std::min({kMaxSplit, fit, kblocks / 4}));
}

template <int R, bool SWIGLU>
void launch_product(const bf16* x, const uint8_t* codes, const uint8_t* scales,
                    const bf16* residual, bf16* out, int rows, int n, int k, cudaStream_t s) {
  using L = ProductSmem<R>;
  auto kernel = mx4_product_kernel<R, SWIGLU>;
  ensure_smem(kernel, L::kBytes);
  constexpr int kCols = SWIGLU ? 64 : 128;
  const CUtensorMap tx = make_tmap_bf16(x, rows, k, k, R);
  const int tiles = (n - 1) / kCols + 1, blocks = (rows - 1) / R + 1, kblocks = k / kKB;
  require(blocks <= 65535, "MXFP4 products take at most 65535 blocks of 64 rows");
  const int split = choose_split(static_cast<int64_t>(tiles) * blocks, kblocks);
  const dim3 grid(static_cast<unsigned>(tiles) * split, static_cast<unsigned>(blocks));
  launch(kernel, grid, kThreads, L::kBytes, split > 1 ? split : 0, s, tx, codes, scales, residual, out,
         rows, n, kblocks, split, device_error_word());
}

}  // namespace

void mx4_product_tc(const bf16* x, const uint8_t* codes, const uint8_t* scales,
                    const bf16* residual, bf16* out, int rows, int n, int k, bool swiglu,
                    cudaStream_t s) {
  auto run = [&](auto product, auto swiglu_product) {
    (swiglu ? swiglu_product : product)(x, codes, scales, residual, out, rows, n, k, s);
  };
  if (rows <= 32) {
    run(launch_product<32, false>, launch_product<32, true>);
  } else if (rows <= 48) {
    run(launch_product<48, false>, launch_product<48, true>);
  } else {
    run(launch_product<64, false>, launch_product<64, true>);
  }
}

}  // namespace ce4b
