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
// Few tiles: the weights are the traffic and a tile a pair leaves SMs idle, so the k range is cut over the pairs of a
// cluster (up to four).  Their sums meet in the first pair's shared memory and are added in the
// order of the k ranges: no workspace, no second launch, the same bits every time.
//
// Persistent clusters; in each CTA:
//   warp 0       TMA producer of the operands (its 128 features, its half of the tile's rows); warp 14 of the scales
//   warp 1       owns the tensor memory; in the first CTA of a pair one thread issues the MMAs of both
//   warps 2-5    scale movers: shared memory -> tensor memory, one per 32-lane quadrant
//   warps 6-13   epilogue: tensor memory -> registers -> bf16 / f16 / f32; a lane is a feature, a register a row
// Measured: 16384 x 9984 x 4096 250 us, 5.4 PFLOP/s (70 % of the tensor pipe's cycles; the clock falls at the power cap in longer runs).
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
constexpr int kSfwBytes = 512, kSfxBytes = 1024;               // scales of 128 features, of up to 256 rows, per 128 k
constexpr int kSfBytes = 2 * (kSfwBytes + kSfxBytes);
constexpr int kEpiWarps = 8;
constexpr int kThreads = (2 + 4 + kEpiWarps + 1) * 32;
constexpr int kBatch = 3;                                      // stages whose scales are announced together, at most
constexpr int kSfCols = 24;                                    // per stage: 2 x (4 (features) + 8 (rows))
constexpr int kTmemCols = 512;
constexpr int kOutBytes = kEpiWarps * 1024;                    // a warp's 16 rows x 32 features on their way out
constexpr int kTailBytes = 512;                                // barriers, tensor-memory address, abort flag
constexpr int kSmemMax = 232448;
constexpr int kSplitRows = 192;                                // most rows of sums (128 features each) that the later pairs leave: 96 KB
constexpr int kMaxSplit = 4;

struct Fp4GemmParams {
  int M, N, K;               // K: padded
  void* C;
  long ldc;
  int vec;                   // 16-bit rows of C start on 16-byte boundaries
  int tile_n;                // rows of a tile
  int box_rows;              // rows of one TMA load of A
  int stages, stage_bytes, bufs;
  int splits, cluster_shift; // pairs of a cluster (1, 2 or 4), log2 of its CTAs
  int fbs, rt;               // feature blocks, row tiles
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

__device__ __forceinline__ void sts16(uint32_t a, uint16_t v) { asm volatile("st.shared.b16 [%0], %1;" ::"r"(a), "h"(v) : "memory"); }
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

struct Tile {
  int row0, rows, n, f0;     // first row, rows that count, columns of the MMA (a multiple of 32), first feature
};

template <int OUT>                                              // 0 f32, 1 f16, 2 bf16
__global__ void __launch_bounds__(kThreads, 1)
gemm_fp4_kernel(const __grid_constant__ CUtensorMap mapX, const __grid_constant__ CUtensorMap mapW, const __grid_constant__ CUtensorMap mapSX,
                const __grid_constant__ CUtensorMap mapSW, const Fp4GemmParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = tc::smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;            // swizzled tiles need 1024-byte alignment
  uint8_t* aligned = smem_raw + (base - raw);
  const int stages = p.stages, stage_bytes = p.stage_bytes;
  const uint32_t stage_out = base + stages * stage_bytes, bar0 = stage_out + kOutBytes;
  auto full = [&](int s) { return bar0 + 8u * s; };                             // of the pair's first CTA: operands of both, scales in tensor memory
  auto empty = [&](int s) { return bar0 + 8u * (kMaxStages + s); };
  auto sc_full = [&](int s) { return bar0 + 8u * (2 * kMaxStages + s); };        // this CTA's scales in shared memory
  auto tfull = [&](int b) { return bar0 + 8u * (3 * kMaxStages + b); };
  auto tempty = [&](int b) { return bar0 + 8u * (3 * kMaxStages + 2 + b); };     // of the first CTA
  constexpr int kBars = 3 * kMaxStages + 4;
  static_assert(8 * kBars + 8 <= kTailBytes, "");
  uint8_t* tail = aligned + (bar0 - base) + 8 * kBars;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(tail);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int crank = (int)tcp::cluster_rank(), rank = crank & 1, split = crank >> 1;
  const uint32_t lead = (uint32_t)crank & ~1u;             // first CTA of this pair

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      tc::mbar_init(full(s), 1 + 8);
      tc::mbar_init(empty(s), 1);
      tc::mbar_init(sc_full(s), 1);
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
  tcp::cluster_sync_relaxed();                              // the other CTAs' barriers are set up
  tc::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t sf_base = tmem_base + kTmemCols - stages * kSfCols;      // scale columns behind the accumulators
  tf_pdl_sync();
  const int fbs = p.fbs, rt = p.rt, items = rt * fbs;
  const int first = blockIdx.x >> p.cluster_shift, step = gridDim.x >> p.cluster_shift;
  const int kall = p.K / BK, kb0 = (kall * split) >> (p.cluster_shift - 1), kb1 = (kall * (split + 1)) >> (p.cluster_shift - 1);
  // the clusters running at one time share operands: eight row tiles by as many feature blocks as there are clusters
  auto tile_of = [&](int item) {
    Tile t;
    int g = 0, r = item, gm = rt, fb = item;
    if (rt > 1) {
      g = item / (kGroupRows * fbs);
      r = item - g * kGroupRows * fbs;
      gm = min(kGroupRows, rt - g * kGroupRows);
      fb = r / gm;
      r -= fb * gm;
    } else {
      r = 0;
    }
    t.row0 = (g * kGroupRows + r) * p.tile_n;
    t.rows = min(p.tile_n, p.M - t.row0);
    t.n = (t.rows + 31) & ~31;
    t.f0 = fb * BF;
    return t;
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer: operand tiles
    // (The whole warp waits and one thread, elected once, issues: a loop that one thread runs by itself takes 200 cycles more a
    // wait, since the compiler then guards every copy or MMA behind a branch for lanes that might have left.)
    const bool one = tc::elect_one();
    if (one) {
      tc::prefetch_tmap(&mapX);
      tc::prefetch_tmap(&mapW);
    }
    const uint32_t tx = 2 * (128 * 128 + p.box_rows * 128);               // both CTAs' (parts of a box out of range count too)
    const uint32_t first_full = tcp::map_to(full(0), lead);
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int item = first; item < items && ok; item += step) {
      const Tile t = tile_of(item);
      const int xrow = t.row0 + rank * (t.n >> 1);         // (a box has half of a tile's rows; the last tile's boxes reach over their half and the matrix's end)
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = tc::mbar_wait(empty(s), ph ^ 1, abort_flag))) break;
        if (one) {
          // (the second CTA's bytes may come before the first has set its count: the phase cannot end before that arrival,
          // nor can it be an older one, whose MMAs have freed this stage)
          if (rank == 0) tc::mbar_expect_tx(full(s), tx);
          const uint32_t sa = base + s * stage_bytes, bar = first_full + 8u * s;
          tcp::tma_load_pair(sa, &mapW, kb * 128, t.f0 + rank * 128, bar);
          tcp::tma_load_pair(sa + 128 * 128, &mapX, kb * 128, xrow, bar);
        }
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
      while (clock64() - t0 < 400000) {}         // copies in flight land before the smem goes back
    }
  } else if (warp == kThreads / 32 - 1) {
    // ------------------------------------------------------------------ TMA producer: scales
    const bool one = tc::elect_one();
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int item = first; item < items && ok; item += step) {
      const Tile t = tile_of(item);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = tc::mbar_wait(empty(s), ph ^ 1, abort_flag))) break;
        if (one) {
          // two units of 128 k each, one copy an operand
          const uint32_t sc = base + (s + 1) * stage_bytes - kSfBytes;
          tc::mbar_expect_tx(sc_full(s), 2 * (kSfwBytes + p.tile_n * 4));
          tc::tma_load_2d(sc, &mapSW, t.f0 + rank * 128, 2 * kb, sc_full(s));
          tc::tma_load_2d(sc + 2 * kSfwBytes, &mapSX, t.row0, 2 * kb, sc_full(s));
        }
        if (++s == stages) { s = 0; ph ^= 1; }
      }
    }
    if (!ok) {
      const long long t0 = clock64();
      while (clock64() - t0 < 400000) {}
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (rank == 0) {
      const bool one = tc::elect_one();
      int s = 0, ab = 0;
      uint32_t ph = 0, aph = 0;
      bool ok = true;
      for (int item = first; item < items && ok; item += step) {
        const uint32_t n = (uint32_t)tile_of(item).n, id = idesc_fp4(n);
        const uint32_t td = tmem_base + ab * p.tile_n;
        if (!(ok = tcp::wait_relaxed(tempty(ab), aph ^ 1, abort_flag))) break;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = tc::mbar_wait(full(s), ph, abort_flag))) break;
          tc::tc_fence_after();
          if (one) {
            const uint32_t sa = base + s * stage_bytes;
            const uint64_t da = tc::smem_desc_sw128(sa), db = tc::smem_desc_sw128(sa + 128 * 128);
            const uint32_t sf = sf_base + s * kSfCols;
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
              const uint32_t sfw = sf + (k >> 1) * 12, sel = (k & 1) * 2;
              mma_fp4(td, da + 2 * k, db + 2 * k, id | (sel << 4) | (sel << 29), sfw, sfw + 4, (kb > kb0 || k) ? 1u : 0u);
            }
            tcp::commit_pair(empty(s), lead);            // frees the stage and, with it, the stage's scale columns
            if (kb + 1 == kb1) tcp::commit_pair(tfull(ab), lead);
          }
          if (++s == stages) { s = 0; ph ^= 1; }
        }
        if (++ab == p.bufs) { ab = 0; aph ^= 1; }
      }
    }
  } else if (warp < 6) {
    // ------------------------------------------------------------------ scale movers
    // When sc_full(s) completes for lap r of the ring, the MMAs that read scale columns s in lap r - 1 are
    // done (the producer refilled the stage only after their commit): the columns are free.
    // Up to kBatch stages are written before they are waited for and announced together: the wait for tcgen05.st is some 400
    // cycles, and stage by stage it took longer than the MMAs.  A stage that is not there yet ends the batch.
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16, first_sf = tcp::map_to(full(0), lead);
    int s = 0, first_s = 0, batch = 0;
    uint32_t ph = 0;
    bool ok = true;
    auto announce = [&]() {
      tcp::tmem_st_wait();
      tc::tc_fence_before();
      __syncwarp();
      if (lane < batch) tcp::arrive_mapped(first_sf + 8u * (first_s + lane < stages ? first_s + lane : first_s + lane - stages));
      batch = 0;
      first_s = s;
    };
    for (int item = first; item < items && ok; item += step) {
      const int nx = tile_of(item).n >> 5;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!__all_sync(0xffffffffu, tc::mbar_try(sc_full(s), ph))) {
          if (batch) announce();
          if (!(ok = tc::mbar_wait(sc_full(s), ph, abort_flag))) break;
        } else if (batch == kBatch) {
          announce();
        }
        const uint8_t* sf = aligned + (s + 1) * stage_bytes - kSfBytes + lane * 4;
        const uint32_t t = sf_base + lane_base + s * kSfCols;
        uint32_t v[24];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int j = 0; j < 4; ++j) v[12 * h + j] = *reinterpret_cast<const uint32_t*>(sf + h * kSfwBytes + j * 128);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            v[12 * h + 4 + j] = j < nx ? *reinterpret_cast<const uint32_t*>(sf + 2 * kSfwBytes + h * p.tile_n * 4 + j * 128) : 0u;
        }
        tcp::tmem_st16(t, v);
        tcp::tmem_st8(t + 16, v + 16);
        ++batch;
        if (++s == stages) { s = 0; ph ^= 1; }
      }
    }
    if (batch) announce();
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
      if (OUT == 0) {
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
              if (OUT == 1) {
                const __half2 h = __floats2half2_rn(a, b);
                pk[c / 2 + i] = *reinterpret_cast<const uint32_t*>(&h);
              } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
                pk[c / 2 + i] = *reinterpret_cast<const uint32_t*>(&h);
              }
            }
          }
        }
        release();
        if (p.vec && t.f0 + rank * 128 + quad * 32 + 32 <= p.N) {
          // 16 rows at a time through shared memory, so that a lane stores eight features: two bytes a lane took longer than a tile's MMAs
          const uint32_t mine = stage_out + (warp - 6) * 1024;
          uint8_t* base_row = reinterpret_cast<uint8_t*>(p.C) + ((long)(t.row0 + c0) * p.ldc + t.f0 + rank * 128 + quad * 32) * 2 + (lane & 3) * 16;
          const int rows = min(cols, t.rows - c0);
#pragma unroll
          for (int c = 0; c < 128; c += 16) {
            if (c < rows) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                sts16(mine + (2 * i) * 64 + lane * 2, (uint16_t)pk[c / 2 + i]);
                sts16(mine + (2 * i + 1) * 64 + lane * 2, (uint16_t)(pk[c / 2 + i] >> 16));
              }
              __syncwarp();
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const int r = c + 8 * i + (lane >> 2);
                const uint4 w = lds128(mine + i * 512 + lane * 16);
                if (r < rows) *reinterpret_cast<uint4*>(base_row + (long)r * p.ldc * 2) = w;
              }
              __syncwarp();
            }
          }
        } else {
#pragma unroll
          for (int c = 0; c < 128; c += 2) {
            if (c < live) dst[0] = (uint16_t)pk[c / 2];
            if (c + 1 < live) dst[p.ldc] = (uint16_t)(pk[c / 2] >> 16);
            dst += 2 * p.ldc;
          }
        }
      }
      if (++ab == p.bufs) { ab = 0; aph ^= 1; }
    }
  } else {
    // ------------------------------------------------------------------ k range cut over the cluster's pairs: this pair's sums are there
    tc::mbar_wait(tfull(0), 0, abort_flag);
    tc::tc_fence_after();
  }
  if (p.splits > 1) {
    // Once every pair is done the rings are free: the later pairs leave their sums in the first pair's, which adds them in order.
    const int quad = warp & 3, half = (warp - 6) >> 2;
    const bool epi = warp >= 6 && warp < 6 + kEpiWarps;
    const Tile t = tile_of(first);
    const int cols = t.n >> 1, c0 = half * cols, live = min(cols, t.rows - c0);      // columns of this warp, those that count
    const int lane_f = quad * 32 + lane;                     // this lane's feature of the CTA's 128
    const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + c0;
    __syncthreads();
    tcp::cluster_sync_relaxed();
    if (epi && split) {
      // [split - 1][row][feature] fp32
      const uint32_t dst = tcp::map_to(base + (uint32_t)(((split - 1) * p.tile_n + c0) * 128 + lane_f) * 4u, (uint32_t)rank);
#pragma unroll 1
      for (int c = 0; c < live; c += 16) {
        uint32_t v[16];
        tcp::tmem_ld16(taddr + c, v);
        tc::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (c + i < live) tcp::st_cluster(dst + (c + i) * 512u, v[i]);
      }
    }
    __syncwarp();
    tcp::cluster_sync();
    const int f = t.f0 + rank * 128 + lane_f;
    if (epi && !split) {
      const float* got = reinterpret_cast<const float*>(aligned) + c0 * 128 + lane_f;
      const long off = (long)(t.row0 + c0) * p.ldc + f;
#pragma unroll 1
      for (int c = 0; c < live; c += 16) {
        uint32_t v[16];
        tcp::tmem_ld16(taddr + c, v);
        float a[kMaxSplit - 1][16];
#pragma unroll
        for (int k = 0; k < kMaxSplit - 1; ++k)
#pragma unroll
          for (int i = 0; i < 16; ++i) a[k][i] = k + 1 < p.splits && c + i < live ? got[(k * p.tile_n + c + i) * 128] : 0.f;
        tc::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (c + i >= live || f >= p.N) break;
          const float x = ((__uint_as_float(v[i]) + a[0][i]) + a[1][i]) + a[2][i];
          const long o = off + (c + i) * p.ldc;
          if (OUT == 0) reinterpret_cast<float*>(p.C)[o] = x;
          else if (OUT == 1) reinterpret_cast<__half*>(p.C)[o] = __float2half(x);
          else reinterpret_cast<__nv_bfloat16*>(p.C)[o] = __float2bfloat16(x);
        }
        __syncwarp();
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0) tf_report(p.status, TF_TIMEOUT, 184, blockIdx.x, 0);
  __syncwarp();
  tcp::cluster_sync_relaxed();                 // nobody leaves while another CTA may still arrive at its barriers
  if (warp == 1) {
    tc::tc_fence_after();
    tcp::tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

int g_sms = 0;

// Scales [K / 128][units][128 bytes] as rows of 32-bit words (the four scales of a row): a box is `rows` rows of two units.
bool make_map_scales(CUtensorMap* map, const void* base, uint64_t k128, uint64_t units, uint32_t rows) {
  auto fn = tc::encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {units * 32, k128};
  cuuint64_t strides[1] = {units * 128};
  cuuint32_t box[2] = {rows, 2};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Rows of the tiles and pairs that share a tile's k range: the least estimated time, in cycles.  A stage (256 k) takes its MMAs
// (2 a row), its L2 bytes (128 features + half of the rows, 128 bytes each, at 64 a cycle) or what its waits and scale columns
// take in a row (480), whichever is longest; a tile its drain (5 a row) too, and a cut one the exchange of sums.  The later
// pairs' sums have to fit the ring.  197 x 4096 x 8192: one tile of 224 rows on 16 pairs 18.7 us, two of 128 cut in two 15 (warm).
void plan(int M, int fbs, int pairs, int kall, int* rows, int* splits) {
  long best = 0;
  for (int n = 32; n <= kMaxRows; n += 32) {
    const long tiles = (long)((M + n - 1) / n) * fbs;
    for (int s = 1; s <= kMaxSplit; s *= 2) {
      if (s > 1 && (tiles * s > pairs || kall < 2 * s || (s - 1) * n > kSplitRows)) break;
      const long waves = s > 1 ? 1 : (tiles + pairs - 1) / pairs;
      const long stage = 2 * n > 480 ? 2 * n : 480, l2 = 256 + n;
      const long cost = waves * ((kall + s - 1) / s * (stage > l2 ? stage : l2) + 5 * n) + (s > 1 ? 2500 + 10 * n : 0);
      if (!best || cost < best || (cost == best && s == *splits)) {
        best = cost;
        *rows = n;
        *splits = s;
      }
    }
    if (n >= M) break;
  }
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
  auto kernel = out_kind == 0 ? gemm_fp4_kernel<0> : out_kind == 1 ? gemm_fp4_kernel<1> : gemm_fp4_kernel<2>;
  static unsigned long long limit_set[3] = {0, 0, 0};
  if (tf_smem_limit((const void*)kernel, kSmemMax, &limit_set[out_kind]) != cudaSuccess) return -2;
  Fp4GemmParams p = {};
  const int pairs = g_sms / 2, fbs = (N + BF - 1) / BF;
  plan(M, fbs, pairs, Kp / BK, &p.tile_n, &p.splits);
  const int rt = (M + p.tile_n - 1) / p.tile_n;
  const long items = (long)rt * fbs;
  p.box_rows = p.tile_n / 2;
  const int x_rows = (p.tile_n / 2 + 31) / 32 * 32;      // (what a swizzled tile behind it needs: whole groups of eight rows)
  p.stage_bytes = 128 * 128 + x_rows * 128 + (kSfBytes + 1023) / 1024 * 1024;
  const int room = kSmemMax - 1024 - kOutBytes - kTailBytes;
  p.stages = room / p.stage_bytes < kMaxStages ? room / p.stage_bytes : kMaxStages;
  p.bufs = 2 * p.tile_n + p.stages * kSfCols <= kTmemCols ? 2 : 1;
  CUtensorMap mX, mW, mSX, mSW;
  if (!make_map_scales(&mSX, sfa, Kp / 128, sfa_units, p.tile_n) || !make_map_scales(&mSW, sfb, Kp / 128, sfb_units, 128)) return -4;
  if (!tc::make_map_2d(&mX, A, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, M, Kp / 2, Kp / 2, p.box_rows)) return -4;
  if (!tc::make_map_2d(&mW, B, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, N, Kp / 2, Kp / 2, 128)) return -4;
  p.M = M; p.N = N; p.K = Kp;
  p.C = C; p.ldc = ldc;
  p.vec = out_kind && ldc % 8 == 0 && !(reinterpret_cast<uintptr_t>(C) & 15);
  p.status = (TfStatusWord*)status;
  const int csize = 2 * p.splits;
  p.cluster_shift = p.splits == 1 ? 1 : p.splits == 2 ? 2 : 3;
  p.fbs = fbs; p.rt = rt;
  const long clusters = p.splits > 1 ? items : (items < pairs ? items : pairs);
  return tcp::launch_cluster(kernel, dim3((unsigned)(clusters * csize)), dim3(kThreads), kSmemMax, csize, st, mX, mW, mSX, mSW, p);
}
