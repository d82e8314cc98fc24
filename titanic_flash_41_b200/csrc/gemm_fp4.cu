// Product of MXFP4 rows and MXFP4 weights for sm_100a:
//
//   C[M, N] = (A * sfa) (B * sfb)^T      A [M, Kp] and B [N, Kp] packed e2m1 (Kp / 2 bytes a row, Kp a multiple of 256), one UE8M0
//                                         scale per (row, 32 k) in units (fp4.cu)
//
// `tcgen05.mma kind::mxf4.block_scale` multiplies 64 k an instruction, in the time that the 8-bit form takes for 32, from
// operands that lie packed in shared memory: half the bytes and half the instructions of the same product with 8-bit rows
// (gemm_mx.cu), whose geometry this kernel shares: a pair of CTAs (`cta_group::2`) works on a tile, the WEIGHTS are
// the M side (256 features, 128 a CTA) and up to 256 rows, 32 at a time, the N side.  A ring stage is 256 k, 128 bytes of
// every operand row, and two units of scales.
//
// Few rows (one tile of at most 64): the weights are the traffic and a feature block a pair leaves SMs idle, so the k range
// is cut over the pairs of a cluster (up to four).  Their sums meet in the first pair's shared memory and are added in the
// order of the k ranges: no workspace, no second launch, the same bits every time.
//
// Persistent clusters; in each CTA:
//   warp 0       TMA producer of the operands (its 128 features, its half of the tile's rows); warp 14 of the scales
//   warp 1       owns the tensor memory; in the first CTA of a pair one thread issues the MMAs of both
//   warps 2-5    scale movers: shared memory -> tensor memory, one per 32-lane quadrant
//   warps 6-13   epilogue: tensor memory -> registers -> bf16 / f16 / f32; a lane is a feature, a register a row
// Sums are fp32 in tensor memory and are rounded once.  Every mbarrier wait is bounded: on a time-out the CTA raises its
// abort flag, reports TF_TIMEOUT, lets copies in flight land, frees its tensor memory and returns.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tc.cuh"
#include "tc_pair.cuh"

namespace {

constexpr int BF = 256, BK = 256;                              // features of a pair's tile, k of a stage
constexpr int kMaxRows = 256;                                  // rows of a tile
constexpr int kMaxStages = 10;
constexpr int kGroupRows = 8;                                  // row tiles walked together
constexpr int kSfwBytes = 512, kSfxBytes = 1024;               // scales of 128 features, of 256 rows, per 128 k
constexpr int kSfBytes = 2 * (kSfwBytes + kSfxBytes);
constexpr int kEpiWarps = 8;
constexpr int kThreads = (2 + 4 + kEpiWarps + 1) * 32;
constexpr int kSfCols = 24;                                    // per stage: 2 x (4 (features) + 8 (rows))
constexpr int kTmemCols = 512;
constexpr int kTailBytes = 512;                                // barriers, tensor-memory address, abort flag
constexpr int kSmemMax = 232448;
constexpr int kSplitRows = 64;                                 // most rows of a tile whose k range is cut
constexpr int kMaxSplit = 4;

struct Fp4GemmParams {
  int M, N, K;               // K: padded
  const uint8_t *sfa, *sfb;  // units [K / 128][units]
  int sfa_units, sfb_units;
  void* C;
  long ldc;
  int out_kind;              // 0 f32, 1 f16, 2 bf16
  int tile_n;                // rows of a tile
  int box_rows;              // rows of one TMA load of A
  int stages, stage_bytes, bufs;
  int splits;                // pairs of a cluster
  TfStatusWord* status;
};

__device__ __forceinline__ void mma_fp4(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
      ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
      : "memory");
}
// A and B e2m1, both K-major, UE8M0 scales, M = 256; + the scale ids (bytes 0-1 or 2-3 of a 32-bit scale column)
__device__ __forceinline__ uint32_t idesc_fp4(uint32_t rows) {
  return (1u << 7) | (1u << 10) | ((rows >> 3) << 17) | (1u << 23) | ((uint32_t)(BF >> 4) << 24);
}

struct Tile {
  int row0, rows, n, f0;     // first row, rows that count, columns of the MMA (a multiple of 32), first feature
};

__global__ void __launch_bounds__(kThreads, 1)
gemm_fp4_kernel(const __grid_constant__ CUtensorMap mapX, const __grid_constant__ CUtensorMap mapW, const Fp4GemmParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = tc::smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;            // swizzled tiles need 1024-byte alignment
  uint8_t* aligned = smem_raw + (base - raw);
  const int stages = p.stages, stage_bytes = p.stage_bytes;
  const uint32_t bar0 = base + stages * stage_bytes;
  auto full = [&](int s) { return bar0 + 8u * s; };                             // of the pair's first CTA: operands of both
  auto empty = [&](int s) { return bar0 + 8u * (kMaxStages + s); };
  auto sc_full = [&](int s) { return bar0 + 8u * (2 * kMaxStages + s); };        // this CTA's scales in shared memory
  auto sf_full = [&](int s) { return bar0 + 8u * (3 * kMaxStages + s); };        // of the first CTA: those of both in tensor memory
  auto tfull = [&](int b) { return bar0 + 8u * (4 * kMaxStages + b); };
  auto tempty = [&](int b) { return bar0 + 8u * (4 * kMaxStages + 2 + b); };     // of the first CTA
  constexpr int kBars = 4 * kMaxStages + 4;
  static_assert(8 * kBars + 8 <= kTailBytes, "");
  uint8_t* tail = aligned + (bar0 - base) + 8 * kBars;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(tail);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int crank = (int)tcp::cluster_rank(), rank = crank & 1, split = crank >> 1;
  const uint32_t lead = (uint32_t)crank & ~1u;             // first CTA of this pair

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      tc::mbar_init(full(s), 1);
      tc::mbar_init(empty(s), 1);
      tc::mbar_init(sc_full(s), 1);
      tc::mbar_init(sf_full(s), 8);
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(tfull(b), 1);
      tc::mbar_init(tempty(b), 2 * kEpiWarps);
    }
    *abort_flag = 0;
    tc::fence_barrier_init();
  }
  if (warp == 1) tcp::tmem_alloc_pair(tc::smem_u32(const_cast<uint32_t*>(tmem_slot)), kTmemCols);
  tc::tc_fence_before();
  __syncthreads();
  tcp::cluster_sync();                                      // the other CTAs' barriers are set up
  tc::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t sf_base = tmem_base + kTmemCols - stages * kSfCols;      // scale columns behind the accumulators
  tf_pdl_sync();
  const int fbs = (p.N + BF - 1) / BF, rt = (p.M + p.tile_n - 1) / p.tile_n, items = rt * fbs;
  const int csize = 2 * p.splits, first = blockIdx.x / csize, step = gridDim.x / csize;
  const int kall = p.K / BK, kb0 = kall * split / p.splits, kb1 = kall * (split + 1) / p.splits;
  // the clusters running at one time share operands: eight row tiles by as many feature blocks as there are clusters
  auto tile_of = [&](int item) {
    Tile t;
    const int g = item / (kGroupRows * fbs), r = item - g * kGroupRows * fbs, gm = min(kGroupRows, rt - g * kGroupRows);
    t.row0 = (g * kGroupRows + r % gm) * p.tile_n;
    t.rows = min(p.tile_n, p.M - t.row0);
    t.n = (t.rows + 31) & ~31;
    t.f0 = r / gm * BF;
    return t;
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer: operand tiles
    if (tc::elect_one()) {
      tc::prefetch_tmap(&mapX);
      tc::prefetch_tmap(&mapW);
      const int box_bytes = p.box_rows * 128;
      const uint32_t first_full = tcp::map_to(full(0), lead);
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int item = first; item < items && ok; item += step) {
        const Tile t = tile_of(item);
        const int half = t.n >> 1, xrow = t.row0 + rank * half, loads = (half + p.box_rows - 1) / p.box_rows;
        const uint32_t tx = 2 * (128 * 128 + loads * box_bytes);          // both CTAs' (parts of a box out of range count too)
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = tc::mbar_wait(empty(s), ph ^ 1, abort_flag))) break;
          // (the second CTA's bytes may come before the first has set its count: the phase cannot end before that arrival,
          // nor can it be an older one, whose MMAs have freed this stage)
          if (rank == 0) tc::mbar_expect_tx(full(s), tx);
          const uint32_t sa = base + s * stage_bytes, sx = sa + 128 * 128, bar = first_full + 8u * s;
          tcp::tma_load_pair(sa, &mapW, kb * 128, t.f0 + rank * 128, bar);
          for (int i = 0; i < loads; ++i) tcp::tma_load_pair(sx + i * box_bytes, &mapX, kb * 128, xrow + i * p.box_rows, bar);
          if (++s == stages) { s = 0; ph ^= 1; }
        }
      }
      // the last commits arrive at this CTA's barriers before it may leave
      for (int i = 0; i < stages && ok; ++i) {
        ok = tc::mbar_wait(empty(s), ph ^ 1, abort_flag);
        if (++s == stages) { s = 0; ph ^= 1; }
      }
      if (!ok) {
        const long long t0 = clock64();
        while (clock64() - t0 < 400000) {}       // copies in flight land before the smem goes back
      }
    }
  } else if (warp == kThreads / 32 - 1) {
    // ------------------------------------------------------------------ TMA producer: scales
    if (tc::elect_one()) {
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int item = first; item < items && ok; item += step) {
        const Tile t = tile_of(item);
        const uint32_t xbytes = t.n * 4;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = tc::mbar_wait(empty(s), ph ^ 1, abort_flag))) break;
          const uint32_t sc = base + (s + 1) * stage_bytes - kSfBytes;
          tc::mbar_expect_tx(sc_full(s), 2 * (kSfwBytes + xbytes));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const long k128 = 2l * kb + h;
            tc::bulk_g2s(sc + h * (kSfwBytes + kSfxBytes), p.sfb + (k128 * p.sfb_units + ((t.f0 + rank * 128) >> 5)) * 128, kSfwBytes, sc_full(s));
            tc::bulk_g2s(sc + h * (kSfwBytes + kSfxBytes) + kSfwBytes, p.sfa + (k128 * p.sfa_units + (t.row0 >> 5)) * 128, xbytes, sc_full(s));
          }
          if (++s == stages) { s = 0; ph ^= 1; }
        }
      }
      if (!ok) {
        const long long t0 = clock64();
        while (clock64() - t0 < 400000) {}
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (rank == 0 && tc::elect_one()) {
      int s = 0, ab = 0;
      uint32_t ph = 0, aph = 0;
      bool ok = true;
      for (int item = first; item < items && ok; item += step) {
        const uint32_t n = (uint32_t)tile_of(item).n, id = idesc_fp4(n);
        const uint32_t td = tmem_base + ab * p.tile_n;
        if (!(ok = tcp::wait_relaxed(tempty(ab), aph ^ 1, abort_flag))) break;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = tcp::wait_relaxed(sf_full(s), ph, abort_flag))) break;
          if (!(ok = tc::mbar_wait(full(s), ph, abort_flag))) break;
          tc::tc_fence_after();
          const uint32_t sa = base + s * stage_bytes;
          const uint64_t da = tc::smem_desc_sw128(sa), db = tc::smem_desc_sw128(sa + 128 * 128);
          const uint32_t sf = sf_base + s * kSfCols;
#pragma unroll
          for (uint32_t k = 0; k < 4; ++k) {
            const uint32_t sfw = sf + (k >> 1) * 12, sel = (k & 1) * 2;
            mma_fp4(td, da + 2 * k, db + 2 * k, id | (sel << 4) | (sel << 29), sfw, sfw + 4, (kb > kb0 || k) ? 1u : 0u);
          }
          tcp::commit_pair(empty(s), lead);  // frees the stage and, with it, the stage's scale columns
          if (++s == stages) { s = 0; ph ^= 1; }
        }
        if (ok) tcp::commit_pair(tfull(ab), lead);
        if (++ab == p.bufs) { ab = 0; aph ^= 1; }
      }
    }
  } else if (warp < 6) {
    // ------------------------------------------------------------------ scale movers
    // When sc_full(s) completes for lap r of the ring, the MMAs that read scale columns s in lap r - 1 are
    // done (the producer refilled the stage only after their commit): the columns are free.
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int item = first; item < items && ok; item += step) {
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = tc::mbar_wait(sc_full(s), ph, abort_flag))) break;
        const uint8_t* sf = aligned + (s + 1) * stage_bytes - kSfBytes;
        const uint32_t t = sf_base + lane_base + s * kSfCols;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t vw[4], vx[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) vw[j] = *reinterpret_cast<const uint32_t*>(sf + j * 128 + lane * 4);
#pragma unroll
          for (int j = 0; j < 8; ++j) vx[j] = *reinterpret_cast<const uint32_t*>(sf + kSfwBytes + j * 128 + lane * 4);
          tcp::tmem_st4(t + 12 * h, vw);
          tcp::tmem_st8(t + 12 * h + 4, vx);
          sf += kSfwBytes + kSfxBytes;
        }
        tcp::tmem_st_wait();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tcp::arrive_at(sf_full(s), lead);
        if (++s == stages) { s = 0; ph ^= 1; }
      }
    }
  } else if (p.splits == 1) {
    // ------------------------------------------------------------------ epilogue warps
    const int quad = warp & 3;                 // TMEM lanes this warp may touch: [32*quad, 32*quad+32)
    const int half = (warp - 6) >> 2;          // which half of the tile's columns
    int ab = 0;
    uint32_t aph = 0;
    bool ok = true;
    for (int item = first; item < items && ok; item += step) {
      const Tile t = tile_of(item);
      const int cols = t.n >> 1, c0 = half * cols;             // a multiple of 16
      const int f = t.f0 + rank * 128 + quad * 32 + lane;      // this lane's feature
      const int live = f < p.N ? min(cols, t.rows - c0) : 0;   // columns of this warp's half that are stored
      const long off = (long)(t.row0 + c0) * p.ldc + f;
      if (!(ok = tc::mbar_wait(tfull(ab), aph, abort_flag))) break;
      tc::tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + ab * p.tile_n + c0;
      auto release = [&]() {
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tcp::arrive_at(tempty(ab), lead);
      };
      if (p.out_kind == 0) {
        float* dst = reinterpret_cast<float*>(p.C) + off;
#pragma unroll 1
        for (int c = 0; c < cols; c += 32) {
          uint32_t v[32];
          tcp::tmem_ld16(taddr + c, v);
          if (c + 16 < cols) tcp::tmem_ld16(taddr + c + 16, v + 16);
          tc::tmem_ld_wait();
          if (c + 32 >= cols) release();
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (c + i < live) *dst = __uint_as_float(v[i]);
            dst += p.ldc;
          }
        }
      } else {
        uint16_t* dst = reinterpret_cast<uint16_t*>(p.C) + off;
        const bool half16 = p.out_kind == 1;
        uint32_t pk[64];
#pragma unroll
        for (int c = 0; c < 128; c += 32) {
          if (c < cols) {
            uint32_t v[32];
            tcp::tmem_ld16(taddr + c, v);
            if (c + 16 < cols) tcp::tmem_ld16(taddr + c + 16, v + 16);
            tc::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float a = __uint_as_float(v[2 * i]), b = __uint_as_float(v[2 * i + 1]);
              const __nv_bfloat162 hb = __floats2bfloat162_rn(a, b);
              const __half2 hh = __floats2half2_rn(a, b);
              pk[c / 2 + i] = half16 ? *reinterpret_cast<const uint32_t*>(&hh) : *reinterpret_cast<const uint32_t*>(&hb);
            }
          }
        }
        release();
#pragma unroll
        for (int c = 0; c < 128; c += 2) {
          if (c < live) dst[0] = (uint16_t)pk[c / 2];
          if (c + 1 < live) dst[p.ldc] = (uint16_t)(pk[c / 2] >> 16);
          dst += 2 * p.ldc;
        }
      }
      if (++ab == p.bufs) { ab = 0; aph ^= 1; }
    }
  } else if (first < items) {
    // ------------------------------------------------------------------ k range cut over the cluster's pairs: this pair's sums are there
    tc::mbar_wait(tfull(0), 0, abort_flag);
    tc::tc_fence_after();
  }
  if (p.splits > 1) {
    // Once every pair is done the rings are free: the later pairs leave their sums in the first pair's, which adds them in order.
    tc::tc_fence_before();
    __syncthreads();
    tcp::cluster_sync();
    tc::tc_fence_after();
    const int quad = warp & 3, half = (warp - 6) >> 2;
    const bool epi = warp >= 6 && warp < 6 + kEpiWarps && first < items;
    const Tile t = tile_of(first < items ? first : 0);
    const int cols = t.n >> 1, c0 = half * cols;
    const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + c0;
    const int lane_f = quad * 32 + lane;                     // this lane's feature of the CTA's 128
    uint32_t v[32];
    if (epi) {
      tcp::tmem_ld16(taddr, v);
      if (cols > 16) tcp::tmem_ld16(taddr + 16, v + 16);
      tc::tmem_ld_wait();
      if (split) {
        // [split - 1][row][feature] fp32
        const uint32_t dst = tcp::map_to(base + (uint32_t)(((split - 1) * kSplitRows + c0) * 128 + lane_f) * 4u, (uint32_t)rank);
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i < cols) tcp::st_cluster(dst + i * 512u, v[i]);
      }
    }
    tc::tc_fence_before();
    __syncthreads();
    tcp::cluster_sync();
    if (epi && !split) {
      const int f = t.f0 + rank * 128 + lane_f;
      const float* got = reinterpret_cast<const float*>(aligned) + c0 * 128 + lane_f;
      const int live = f < p.N ? min(cols, t.rows - c0) : 0;
      const long off = (long)(t.row0 + c0) * p.ldc + f;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        if (i < live) {
          float a = __uint_as_float(v[i]);
          for (int k = 1; k < p.splits; ++k) a += got[((k - 1) * kSplitRows + i) * 128];
          const long o = off + i * p.ldc;
          if (p.out_kind == 0) reinterpret_cast<float*>(p.C)[o] = a;
          else if (p.out_kind == 1) reinterpret_cast<__half*>(p.C)[o] = __float2half(a);
          else reinterpret_cast<__nv_bfloat16*>(p.C)[o] = __float2bfloat16(a);
        }
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0) tf_report(p.status, TF_TIMEOUT, 184, blockIdx.x, 0);
  __syncwarp();
  tcp::cluster_sync();                         // nobody leaves while another CTA may still arrive at its barriers
  if (warp == 1) {
    tc::tc_fence_after();
    tcp::tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

int g_sms = 0;

// Rows of the tiles: the least estimated time over the tile widths.  Per 256 k a tile takes its MMAs (2 cycles a row, 184 at least)
// or its L2 bytes (128 features + its rows / 2, 128 bytes each, at 64 bytes a cycle), whichever is longer, and the tiles
// run in waves of one per pair.
int tile_rows(int M, int fbs, int pairs) {
  int best = 32;
  long best_cost = 0;
  for (int n = 32; n <= kMaxRows; n += 32) {
    const long tiles = (long)((M + n - 1) / n) * fbs, waves = (tiles + pairs - 1) / pairs;
    const long mma = 2 * n > 184 ? 2 * n : 184, l2 = 256 + n;
    const long cost = waves * (mma > l2 ? mma : l2);
    if (n == 32 || cost <= best_cost) {
      best = n;
      best_cost = cost;
    }
    if (n >= M) break;
  }
  return best;
}

}  // namespace

// C [M, N] (out_kind 0 f32, 1 f16, 2 bf16; row pitch ldc elements) = A [M, Kp / 2] x B [N, Kp / 2]^T, both packed e2m1 with unit-layout
// scales: sfa_units >= M / 32 and sfb_units >= N / 32 units per 128 k, the latter in whole 256-feature blocks.  Kp a multiple of 256.
TF_API int tf_gemm_fp4(const void* A, const void* sfa, int sfa_units, const void* B, const void* sfb, int sfb_units, void* C, long ldc,
                       int out_kind, int M, int N, int Kp, void* status, cudaStream_t st) {
  if (M <= 0 || N <= 0 || Kp <= 0 || Kp % BK || out_kind < 0 || out_kind > 2 || ldc < N) return -1;
  if (!A || !B || !sfa || !sfb || !C) return -1;
  if (sfa_units < (M + 31) / 32 || sfb_units < (N + BF - 1) / BF * (BF / 32)) return -1;
  if ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(B) | reinterpret_cast<uintptr_t>(sfa) | reinterpret_cast<uintptr_t>(sfb)) & 15)
    return -1;
  if (reinterpret_cast<uintptr_t>(C) & (out_kind == 0 ? 3 : 1)) return -1;
  if (!g_sms) {
    int dev = 0, n = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    g_sms = n;
  }
  static unsigned long long limit_set = 0;
  if (tf_smem_limit((const void*)gemm_fp4_kernel, kSmemMax, &limit_set) != cudaSuccess) return -2;
  Fp4GemmParams p = {};
  const int pairs = g_sms / 2, fbs = (N + BF - 1) / BF;
  p.tile_n = tile_rows(M, fbs, pairs);
  const int rt = (M + p.tile_n - 1) / p.tile_n;
  const long items = (long)rt * fbs;
  p.splits = 1;
  if (p.tile_n <= kSplitRows)
    while (p.splits < kMaxSplit && items * p.splits * 2 <= pairs && Kp / BK >= 4 * p.splits) p.splits *= 2;
  p.box_rows = p.tile_n / 2;
  const int x_rows = (p.tile_n / 2 + 31) / 32 * 32;      // (what a swizzled tile behind it needs: whole groups of eight rows)
  p.stage_bytes = 128 * 128 + x_rows * 128 + (kSfBytes + 1023) / 1024 * 1024;
  const int room = kSmemMax - 1024 - kTailBytes;
  p.stages = room / p.stage_bytes < kMaxStages ? room / p.stage_bytes : kMaxStages;
  p.bufs = 2 * p.tile_n + p.stages * kSfCols <= kTmemCols ? 2 : 1;
  CUtensorMap mX, mW;
  if (!tc::make_map_2d(&mX, A, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, M, Kp / 2, Kp / 2, p.box_rows)) return -4;
  if (!tc::make_map_2d(&mW, B, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, N, Kp / 2, Kp / 2, 128)) return -4;
  p.M = M; p.N = N; p.K = Kp;
  p.sfa = (const uint8_t*)sfa; p.sfb = (const uint8_t*)sfb;
  p.sfa_units = sfa_units; p.sfb_units = sfb_units;
  p.C = C; p.ldc = ldc; p.out_kind = out_kind;
  p.status = (TfStatusWord*)status;
  const int csize = 2 * p.splits;
  const long clusters = p.splits > 1 ? items : (items < pairs ? items : pairs);
  return tcp::launch_cluster(gemm_fp4_kernel, dim3((unsigned)(clusters * csize)), dim3(kThreads), kSmemMax, csize, st, mX, mW, p);
}
