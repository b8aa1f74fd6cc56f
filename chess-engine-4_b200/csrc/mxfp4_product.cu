// Products of a few BF16 activation rows with an MXFP4 weight (kernel-op API mxfp4_linear,
// mxfp4_swiglu): y[r, n] = sum_k x[r, k] * code[n, k] * 2^(scale[n, k / 32] - 127).
//
// The time is the weight's 0.53 bytes per element, as long as turning codes into operands
// keeps up with them: an SM takes in about 43 codes a clock at the memory's rate and issues
// 128 lane operations, so a code may cost at most three, whatever is done with it. A multiply
// per activation row would spend those on the first few rows. So the weight is the A operand
// of tcgen05 MMAs (128 weight rows are the 128 lanes of tensor memory, up to 64 activation rows
// the N columns): every code is expanded once, in registers, to the BF16 value it stands for
// (E2M1 times a power of two is exact in BF16), and stored to tensor memory, from which the MMA
// reads A without passing through shared memory, whose bandwidth 32 KB per K block in and out
// would fill. Products and activations are exact, sums are FP32.
//
// A CTA takes 128 weight rows (SwiGLU: 64 gate rows and their 64 up rows) and a slice of K. TMA
// brings code tiles, x tiles and scale tiles through a ring; eight warps expand; one thread
// issues the MMAs. A cluster of up to eight CTAs shares the K blocks of one row tile, so that
// weights of few rows still occupy the GPU; their FP32 partial sums are added through
// distributed shared memory in rank order (deterministic).
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
constexpr int kThreads = 64 + 32 * kExpandWarps;
constexpr int kABuffers = 3;       // expanded K blocks in tensor memory, 64 columns each
constexpr int kACol = 64;          // first column of the A buffers (D before it)
constexpr uint32_t kTmemCols = 256;
constexpr int kMaxSplit = 8;

template <int R, bool SWIGLU>
struct ProductSmem {
  static constexpr int kCodeBytes = kM * kKB / 2;
  static constexpr int kXBytes = R * kKB * 2;
  static constexpr int kSfBytes = SWIGLU ? 2048 : 1024;  // 3 or 1 scale tiles of 512 bytes
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
__device__ __forceinline__ void expand_group(const uint4& q, uint32_t scale, uint32_t* out) {
  const uint32_t f = mx4_factor(scale);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v[4];
    mx4_expand(w[i], f, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) out[4 * i + j] = v[j];
  }
  if (__any_sync(0xffffffffu, scale > 128u)) {
    const uint32_t g = mx4_factor2(scale);
#pragma unroll
    for (int i = 0; i < 16; ++i) out[i] = mul_bf16x2(out[i], g);
  }
}

template <int R, bool SWIGLU>
__global__ void __launch_bounds__(kThreads, 2)
    mx4_product_kernel(const __grid_constant__ CUtensorMap tm_codes,
                       const __grid_constant__ CUtensorMap tm_x, const uint8_t* scales,
                       const bf16* residual, bf16* out, int rows, int n, int kblocks, int split,
                       int* err) {
  using L = ProductSmem<R, SWIGLU>;
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
  // First weight rows of the tile (SwiGLU: of its gate half and of its up half).
  const int w0 = tile * kCols;
  const int up0 = n + w0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(full_bar(s), 1);
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
      tma_prefetch_desc(&tm_codes);
      tma_prefetch_desc(&tm_x);
      // Scale tiles of the rows: one, or the gate rows' and the up rows' (which may straddle two).
      const int tiles = ((SWIGLU ? 2 * n : n) + 127) / 128;
      const int t0 = w0 / 128, t1 = up0 / 128, t2 = min(t1 + 1, tiles - 1);
      const uint32_t bytes = L::kCodeBytes + L::kXBytes + (SWIGLU ? 1536u : 512u);
      int it = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int s = it % NS;
        if (!mbar_wait(empty_bar(s), ((it / NS) & 1) ^ 1)) {
          record_error(err, kErrTimeoutProducer);
          ok = false;
          break;
        }
        const uint32_t codes = base + s * L::kStageBytes;
        const uint32_t xs = codes + L::kCodeBytes;
        const uint32_t sf = xs + L::kXBytes;
        mbar_arrive_expect_tx(full_bar(s), bytes);
        if constexpr (SWIGLU) {
          tma_load_2d(codes, &tm_codes, full_bar(s), kb * 64, w0);
          tma_load_2d(codes + L::kCodeBytes / 2, &tm_codes, full_bar(s), kb * 64, up0);
        } else {
          tma_load_2d(codes, &tm_codes, full_bar(s), kb * 64, w0);
        }
        tma_load_2d(xs, &tm_x, full_bar(s), kb * kKB, row0);
        tma_load_2d(xs + L::kXBytes / 2, &tm_x, full_bar(s), kb * kKB + 64, row0);
        bulk_load(sf, scales + (static_cast<size_t>(t0) * kblocks + kb) * 512, 512, full_bar(s));
        if constexpr (SWIGLU) {
          bulk_load(sf + 512, scales + (static_cast<size_t>(t1) * kblocks + kb) * 512, 512, full_bar(s));
          bulk_load(sf + 1024, scales + (static_cast<size_t>(t2) * kblocks + kb) * 512, 512, full_bar(s));
        }
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
  } else {
    // Four warps cover the 128 lanes; the first four expand the even stages, the others the odd.
    const int turn = (warp - 2) / 4;
    const int r = (warp & 3) * 32 + lane;           // weight row in the tile = lane of TMEM
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    // Where the row's four scale bytes of a K block lie in the stage's scale tiles.
    int tile_row = r, area = 0;
    if constexpr (SWIGLU) {
      const int wrow = r < 64 ? w0 + r : up0 + r - 64;
      tile_row = wrow % 128;
      area = r < 64 ? 0 : 1 + (wrow / 128 - up0 / 128);
    }
    const uint32_t sf_off = L::kCodeBytes + L::kXBytes + area * 512 + (tile_row % 32) * 16 + (tile_row / 32) * 4;
    const uint32_t swz = (r >> 1) & 3;
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
        uint32_t v[32];
        expand_group(q0, (sf >> (16u * h)) & 255u, v);
        expand_group(q1, (sf >> (16u * h + 8u)) & 255u, v + 16);
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

// CTAs per row tile. The CTAs of an SM share its issue slots, so a launch takes as long as the
// SM with the most of them: ceil(tiles * split / SMs) times kblocks / split ring stages and a
// fixed part (launch, tensor memory, pipeline fill, join) worth about kFixed stages.
int choose_split(int tiles, int kblocks) {
  constexpr int kFixed = 3;
  const int sms = sm_count();
  int best = 1;
  int64_t best_cost = INT64_MAX;
  for (int split = 1; split <= std::min(kMaxSplit, kblocks); ++split) {
    const int64_t turns = (static_cast<int64_t>(tiles) * split + sms - 1) / sms;
    const int64_t cost = turns * ((kblocks + split - 1) / split + kFixed);
    if (cost < best_cost) best_cost = cost, best = split;
  }
  return best;
}

template <int R, bool SWIGLU>
void launch_product(const bf16* x, const uint8_t* codes, const uint8_t* scales,
                    const bf16* residual, bf16* out, int rows, int n, int k, cudaStream_t s) {
  using L = ProductSmem<R, SWIGLU>;
  auto kernel = mx4_product_kernel<R, SWIGLU>;
  ensure_smem(kernel, L::kBytes);
  constexpr int kCols = SWIGLU ? 64 : 128;
  const int wide = SWIGLU ? 2 * n : n;
  const CUtensorMap tc = make_tmap_u8_sw64(codes, wide, k / 2, k / 2, kCols);
  const CUtensorMap tx = make_tmap_bf16(x, rows, k, k, R);
  const int tiles = (n + kCols - 1) / kCols, kblocks = k / kKB;
  const int split = choose_split(tiles * ((rows + R - 1) / R), kblocks);
  const dim3 grid(static_cast<unsigned>(tiles * split), static_cast<unsigned>((rows + R - 1) / R));
  launch(kernel, grid, kThreads, L::kBytes, split > 1 ? split : 0, s, tc, tx, scales, residual, out,
         rows, n, kblocks, split, device_error_word());
}

}  // namespace

void mx4_product_tc(const bf16* x, const uint8_t* codes, const uint8_t* scales,
                    const bf16* residual, bf16* out, int rows, int n, int k, bool swiglu,
                    cudaStream_t s) {
  if (swiglu) {
    if (rows <= 32) {
      launch_product<32, true>(x, codes, scales, nullptr, out, rows, n, k, s);
    } else {
      launch_product<64, true>(x, codes, scales, nullptr, out, rows, n, k, s);
    }
  } else if (rows <= 32) {
    launch_product<32, false>(x, codes, scales, residual, out, rows, n, k, s);
  } else {
    launch_product<64, false>(x, codes, scales, residual, out, rows, n, k, s);
  }
}

}  // namespace ce4b
