// Attention of many query rows a sequence (prompts, long follow-ups) over the paged 4-bit cache, on the tcgen05 tensor cores; the
// formula and the few-row form are in paged_attn.cu.
//
//   S[row, key]  = Q[row, :] . K[key, :]          A = 128 rows of Q, f16          B = 128 keys, f16, both K-major in shared memory
//   O[row, :]   += P[row, key] V[key, :]          A = P, f16, in tensor memory    B = V transposed: [channel][token], K-major
//
// A row is a (token, query head) pair of one kv head, so the heads that share keys share a tile.  A CTA takes 256 rows, two
// tiles that lag each other: while the softmax warps of one work, the MMAs of the other run.  Scores and probabilities never
// leave tensor memory (S 128 columns a tile, P over S, O D columns a tile).  Keys and values are taken apart once per 256 rows:
// four warps turn packed keys into the swizzled f16 tile, three the values.  The page layout has two tokens of a channel in a byte,
// so a value word of the transposed tile is one cvt and one multiplication, and a warp's store is one 128-byte row of it.
// Keys that no row of the sequence sees are stored as zeros, whatever their pages hold.
//
// A softmax thread owns a row.  The reference maximum is the first tile's and moves (O and the sum rescaled in tensor memory) only
// when a score exceeds it by 2^8.  Registers are moved from the unpacking warps to the softmax warps (a row of S is 128 of them).
// QK of the next keys waits for the PV that reads P, whose columns it overwrites.
// Few items (a short prompt over a long prefix): the keys of an item are cut over several CTAs, whose partial results
// paged_tc_merge_kernel joins in order.
//
// Every mbarrier wait is bounded: on a time-out the CTA raises its abort flag, reports TF_TIMEOUT, frees its tensor memory and returns.
#include "paged_tc.h"

#include "paged.cuh"
#include "tc.cuh"

namespace {

using namespace paged;

constexpr int kRows = 256, kKeys = 128;                  // rows of a CTA, keys of a tile
constexpr int kThreads = 512;                            // warps 0-7 softmax, 8-11 keys, 12 MMA, 13-15 values
constexpr int kMoreRegs = 184, kLessRegs = 72;           // 256 threads each: 65,536 in all, as launched
constexpr float kNone = -3e38f;

struct TcParams : AttnCall {
  int splits;                                            // CTAs of an item; `work` holds [items][splits][kRows][D + 4] where there are several
};

struct Item {
  int seq, h, blk, n, row0, end, len, key0, lo, hi;      // key0: first key that a row of the block sees; lo, hi: this block's keys
};
// the item of a CTA: row blocks of the sequences one after another, the last (longest) block of a sequence first, kv heads inside
__device__ __forceinline__ bool item_of(const TcParams& p, long index, Item* it) {
  const int lane = threadIdx.x & 31;
  long base = 0;
  for (int s0 = 0; s0 < p.r.seqs; s0 += 32) {
    long w = 0;
    if (s0 + lane < p.r.seqs) {
      const int n = p.r.cu ? p.r.cu[s0 + lane + 1] - p.r.cu[s0 + lane] : 1;
      w = ((long)max(n, 0) * p.group + kRows - 1) / kRows * p.c.kv;
    }
    long incl = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    incl += base;
    const unsigned hit = __ballot_sync(0xffffffffu, incl > index);
    if (hit) {
      const int l = __ffs(hit) - 1;
      const long before = __shfl_sync(0xffffffffu, incl - w, l), count = __shfl_sync(0xffffffffu, w, l);
      const long i = count - 1 - (index - before);
      it->seq = s0 + l;
      it->h = (int)(i % p.c.kv);
      it->blk = (int)(i / p.c.kv);
      it->row0 = p.r.cu ? p.r.cu[it->seq] : it->seq;
      it->end = p.r.cu ? p.r.cu[it->seq + 1] : it->seq + 1;
      it->n = it->end - it->row0;
      it->len = p.r.lengths[it->seq];
      const int tok0 = it->blk * kRows / p.group, tok1 = min(((it->blk + 1) * kRows - 1) / p.group, it->n - 1);
      const int pos0 = it->len - it->n + tok0, pos1 = it->len - it->n + tok1;
      it->key0 = max(p.first ? p.first[it->seq] : 0, 0);
      if (p.window) it->key0 = max(it->key0, pos0 - p.window + 1);
      it->lo = it->key0 & ~(kKeys - 1);
      it->hi = max((int)min((long)pos1 + 1, (long)p.r.width << p.c.shift), it->lo);
      return true;
    }
    base = __shfl_sync(0xffffffffu, incl, 31);
  }
  return false;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint64_t pair64(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t v[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
      "%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D[tmem] (+)= A[tmem] * B[smem]: row i of A is lane i, two f16 per 32-bit column; ONE thread issues
__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void sts32(uint32_t a, uint32_t x) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(a), "r"(x) : "memory"); }

// 64 f16 of a row: the 128 swizzled bytes of a K-major tile; 16-byte piece c of row r
__device__ __forceinline__ uint32_t piece(uint32_t tile, int r, int c) { return tile + r * 128 + ((c ^ (r & 7)) << 4); }

template <int D>
struct TcShape {
  static constexpr int kTile = 128 * D * 2;              // bytes of a tile of 128 rows (Q, K) or of a transposed value tile
  static constexpr int kBytes = 6 * kTile + 1024 + 256;  // two tiles of Q, two stages of K and V, barriers
};

// rows of a block relative to their maximum -> out and lse (one thread a row; `o` holds 32 channels from c0 on)
template <typename T>
__device__ __forceinline__ void store32(T* dst, const float* o, float f) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    *reinterpret_cast<uint4*>(dst + 8 * i) = make_uint4(pack<T>(o[8 * i] * f, o[8 * i + 1] * f), pack<T>(o[8 * i + 2] * f, o[8 * i + 3] * f),
                                                        pack<T>(o[8 * i + 4] * f, o[8 * i + 5] * f), pack<T>(o[8 * i + 6] * f, o[8 * i + 7] * f));
}

template <int D, typename T>
__global__ void __launch_bounds__(kThreads, 1) paged_tc_kernel(const TcParams p) {
  using S = TcShape<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = tc::smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* tail = smem_raw + (base - raw) + 6 * S::kTile;
  const uint32_t q_s = base, k_s = base + 2 * S::kTile, v_s = base + 4 * S::kTile, bar0 = base + 6 * S::kTile;
  const uint32_t q_ready = bar0;
  auto k_full = [&](int s) { return bar0 + 8u + 8u * s; };
  auto k_empty = [&](int s) { return bar0 + 24u + 8u * s; };
  auto v_full = [&](int s) { return bar0 + 40u + 8u * s; };
  auto v_empty = [&](int s) { return bar0 + 56u + 8u * s; };
  auto s_ready = [&](int t) { return bar0 + 72u + 8u * t; };
  auto p_ready = [&](int t) { return bar0 + 88u + 8u * t; };
  auto pv_done = [&](int t) { return bar0 + 104u + 8u * t; };
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(tail + 128);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 136);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  tf_pdl_sync();
  Item it;
  const int split = blockIdx.x % p.splits;
  if (!item_of(p, blockIdx.x / p.splits, &it)) return;
  if (threadIdx.x == 0) {
    tc::mbar_init(q_ready, 8);
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(k_full(s), 4);
      tc::mbar_init(k_empty(s), 1);
      tc::mbar_init(v_full(s), 3);
      tc::mbar_init(v_empty(s), 1);
      tc::mbar_init(s_ready(s), 1);
      tc::mbar_init(p_ready(s), 4);
      tc::mbar_init(pv_done(s), 1);
    }
    *abort_flag = 0;
    tc::fence_barrier_init();
  }
  if (warp == 12) tc::tmem_alloc(tc::smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto tS = [&](int t) { return tmem + 128u * t; };
  auto tO = [&](int t) { return tmem + 256u + (uint32_t)D * t; };
  // this CTA's tiles of the item's keys
  const int all = (it.hi - it.lo + kKeys - 1) / kKeys;
  const int j0 = (int)((long)all * split / p.splits), tiles = (int)((long)all * (split + 1) / p.splits) - j0;
  const int tok0 = it.lo + j0 * kKeys;
  const bool two = it.blk * kRows + 128 < it.n * p.group;      // the second tile has rows

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLessRegs));
    const int* tab = p.r.table + (long)it.seq * p.r.width;
    const int shift = p.c.shift, values = (D >> 1) << shift, mask = (1 << shift) - 1;
    auto page_at = [&](int tok) { return tok >= it.key0 && tok < it.hi ? __ldg(tab + (tok >> shift)) : -2; };
    // offset of the head's blocks in a page; a page that is none counts as zeros
    auto block_at = [&](int pg) -> long {
      if (pg >= 0 && pg < p.c.pages) return ((long)pg * p.c.kv + it.h) * p.c.block;
      if (pg != -2) tf_report(p.st, TF_BAD_INDEX, 185, it.seq, pg);
      return -1;
    };
    if (warp < 12) {
      // ---------------------------------------------------------------- keys: a thread takes 32 channels of a token
      constexpr int LR = D / 32, RW = 32 / LR, N = 128 / RW / 4;     // lanes of a row, rows of a warp's item, items of a warp
      const int w = warp - 8, sub = lane % LR;
      uint4 d[N];
      uint16_t sc[N];
      int pg[N];
      auto row_of = [&](int i) { return (w + 4 * i) * RW + lane / LR; };
      auto pages = [&](int j) {
#pragma unroll
        for (int i = 0; i < N; ++i) pg[i] = j < tiles ? page_at(tok0 + j * kKeys + row_of(i)) : -2;
      };
      auto load = [&](int j) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const long off = block_at(pg[i]);
          d[i] = make_uint4(0u, 0u, 0u, 0u);
          sc[i] = 0;
          if (off >= 0) {
            const uint8_t* b = p.c.k + off;
            const int slot = (tok0 + j * kKeys + row_of(i)) & mask;
            d[i] = *reinterpret_cast<const uint4*>(b + slot * (D / 2) + sub * 16);
            sc[i] = *reinterpret_cast<const uint16_t*>(b + values + slot * (D / 16) + sub * 2);
          }
        }
      };
      pages(0);
      load(0);
      pages(1);
      for (int j = 0; j < tiles; ++j) {
        const int s = j & 1;
        if (!tc::mbar_wait(k_empty(s), ((j >> 1) & 1) ^ 1, abort_flag)) break;
        const uint32_t tile = k_s + s * S::kTile + (sub >> 1) * (128 * 128);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int r = row_of(i);
          const uint32_t ss = e4m3x2_to_h2(sc[i]);
          const uint32_t x[4] = {d[i].x, d[i].y, d[i].z, d[i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            // (lanes whose pieces would fall on the same banks take theirs in another order)
            const int c = e ^ (LR == 4 ? (sub >> 1) * 2 : 0);
            const uint32_t wd = c == 0 ? x[0] : c == 1 ? x[1] : c == 2 ? x[2] : x[3];
            const uint32_t f = __byte_perm(ss, 0, c < 2 ? 0x1010 : 0x3232);
            uint32_t h[4];
            fp4::e2m1x8_to_h2x4(wd, h);
            sts128(piece(tile, r, (sub & 1) * 4 + c), fp4::hmul2(h[0], f), fp4::hmul2(h[1], f), fp4::hmul2(h[2], f), fp4::hmul2(h[3], f));
          }
        }
        load(j + 1);
        pages(j + 2);
        tc::fence_proxy_async();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(k_full(s));
      }
    } else if (warp > 12) {
      // ---------------------------------------------------------------- values: a thread takes 32 channels of a pair of tokens
      constexpr int ITEMS = D / 16, N = (ITEMS + 2) / 3;
      const int w = warp - 13;
      uint4 d[N][2];
      uint32_t sc[N];
      int pg[N];
      // item x: 32 pairs from 32 (x & 1) on, channels 32 (x >> 1) ..
      auto pages = [&](int j) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int x = w + 3 * i;
          pg[i] = -2;
          if (x < ITEMS && j < tiles) {
            const int tok = tok0 + j * kKeys + 2 * (32 * (x & 1) + lane);
            pg[i] = page_at(tok);
            if (pg[i] == -2) pg[i] = page_at(tok + 1);
          }
        }
      };
      auto load = [&](int j) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int x = w + 3 * i, tok = tok0 + j * kKeys + 2 * (32 * (x & 1) + lane);
          const long off = block_at(pg[i]);
          d[i][0] = d[i][1] = make_uint4(0u, 0u, 0u, 0u);
          sc[i] = 0;
          if (off >= 0) {
            const uint8_t* b = p.c.v + off;
            const int pair = (tok & mask) >> 1;
            const uint4* src = reinterpret_cast<const uint4*>(b + pair * D + (x >> 1) * 32);
            d[i][0] = src[0];
            d[i][1] = src[1];
            sc[i] = *reinterpret_cast<const uint32_t*>(b + values + pair * (D / 8) + (x >> 1) * 4);
            if (tok < it.key0 || tok >= it.hi) sc[i] &= 0xff00ff00u;
            if (tok + 1 < it.key0 || tok + 1 >= it.hi) sc[i] &= 0x00ff00ffu;
          }
        }
      };
      pages(0);
      load(0);
      pages(1);
      for (int j = 0; j < tiles; ++j) {
        const int s = j & 1;
        if (!tc::mbar_wait(v_empty(s), ((j >> 1) & 1) ^ 1, abort_flag)) break;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int x = w + 3 * i;
          if (x >= ITEMS) continue;
          const uint32_t tile = v_s + s * S::kTile + (x & 1) * (D * 128);      // 64 tokens: [D][128 bytes]
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const uint32_t f = e4m3x2_to_h2((uint16_t)(sc[i] >> 16 * b));
            const uint32_t y[4] = {d[i][b].x, d[i][b].y, d[i][b].z, d[i][b].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t h[4];
              fp4::e2m1x8_to_h2x4(y[e], h);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                sts32(piece(tile, (x >> 1) * 32 + b * 16 + e * 4 + k, lane >> 2) + (lane & 3) * 4, fp4::hmul2(h[k], f));
            }
          }
        }
        load(j + 1);
        pages(j + 2);
        tc::fence_proxy_async();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(v_full(s));
      }
    } else if (tc::elect_one()) {
      // ---------------------------------------------------------------- MMA issuer
      constexpr uint32_t id_qk = tc::instr_desc(0, 0, 128, 128), id_pv = tc::instr_desc(0, 0, 128, D);
      auto qk = [&](int t, int j) {
        const uint32_t q0 = q_s + t * S::kTile, k0 = k_s + (j & 1) * S::kTile;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          tc::mma_f16(tS(t), tc::smem_desc_sw128(q0 + (k >> 2) * 16384) + 2 * (k & 3), tc::smem_desc_sw128(k0 + (k >> 2) * 16384) + 2 * (k & 3),
                      id_qk, k ? 1u : 0u);
        tc::mma_commit(s_ready(t));
      };
      auto pv = [&](int t, int j) {
        const uint32_t v0 = v_s + (j & 1) * S::kTile;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          mma_ts(tO(t), tS(t) + 8 * k, tc::smem_desc_sw128(v0 + (k >> 2) * (D * 128)) + 2 * (k & 3), id_pv, (j | k) ? 1u : 0u);
        tc::mma_commit(pv_done(t));
      };
      bool ok = tiles > 0 && tc::mbar_wait(q_ready, 0, abort_flag) && tc::mbar_wait(k_full(0), 0, abort_flag);
      if (ok) {
        tc::tc_fence_after();
        qk(0, 0);
        if (two) qk(1, 0);
        tc::mma_commit(k_empty(0));
      }
      for (int j = 0; j < tiles && ok; ++j) {
        const uint32_t ph = j & 1, rph = (j >> 1) & 1;
        if (!(ok = tc::mbar_wait(p_ready(0), ph, abort_flag) && tc::mbar_wait(v_full(ph), rph, abort_flag))) break;
        tc::tc_fence_after();
        pv(0, j);
        if (!two) tc::mma_commit(v_empty(ph));
        if (j + 1 < tiles) {
          if (!(ok = tc::mbar_wait(k_full(ph ^ 1), ((j + 1) >> 1) & 1, abort_flag) && tc::mbar_wait(pv_done(0), ph, abort_flag))) break;
          tc::tc_fence_after();
          qk(0, j + 1);
          if (!two) tc::mma_commit(k_empty(ph ^ 1));
        }
        if (two) {
          if (!(ok = tc::mbar_wait(p_ready(1), ph, abort_flag))) break;
          tc::tc_fence_after();
          pv(1, j);
          tc::mma_commit(v_empty(ph));
          if (j + 1 < tiles) {
            if (!(ok = tc::mbar_wait(pv_done(1), ph, abort_flag))) break;
            tc::tc_fence_after();
            qk(1, j + 1);
            tc::mma_commit(k_empty(ph ^ 1));
          }
        }
      }
      // the last commit arrives at this CTA's barrier before it may leave
      if (ok && tiles) ok = tc::mbar_wait(v_empty((tiles - 1) & 1), ((tiles - 1) >> 1) & 1, abort_flag);
      if (*abort_flag) {
        const long long t0 = clock64();
        while (clock64() - t0 < 400000) {}       // MMAs in flight end
      }
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMoreRegs));
    // ------------------------------------------------------------------ softmax: one row per thread
    const int t = warp >> 2, r = (warp & 3) * 32 + lane, fr = it.blk * kRows + t * 128 + r;
    const int tok = fr / p.group, head = it.h * p.group + fr - tok * p.group, row = it.row0 + tok;
    const bool live = tok < it.n && row >= 0 && row < p.r.total;
    const int pos = it.len - it.n + tok;
    int klo = max(p.first ? p.first[it.seq] : 0, 0);
    if (p.window) klo = max(klo, pos - p.window + 1);
    const int khi = min(pos + 1, it.hi);
    float fac = 0.f;
    {
      // the row's query: a power of two brings its largest element into [1, 2), f16 keeps what matters
      const T* src = (const T*)p.q + (live ? (long)row * p.q_row + (long)head * p.q_head : 0l);
      float am = 0.f;
#pragma unroll 4
      for (int c = 0; c < D / 8; ++c) {
        const uint4 v = live ? *reinterpret_cast<const uint4*>(src + 8 * c) : make_uint4(0u, 0u, 0u, 0u);
        const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = paged::two<T>(x[e]);
          am = fmaxf(am, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      const int ex = am > 0.f && am < INFINITY ? (int)(__float_as_uint(am) >> 23) - 127 : 0;
      const float down = __uint_as_float((uint32_t)(127 - min(ex, 126)) << 23);
      fac = ldexpf(p.scale2, min(ex, 126));
#pragma unroll 4
      for (int c = 0; c < D / 8; ++c) {
        const uint4 v = live ? *reinterpret_cast<const uint4*>(src + 8 * c) : make_uint4(0u, 0u, 0u, 0u);
        const uint32_t x[4] = {v.x, v.y, v.z, v.w};
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = paged::two<T>(x[e]);
          o[e] = pack<__half>(f.x * down, f.y * down);
        }
        sts128(piece(q_s + t * S::kTile + (c >> 3) * 16384, r, c & 7), o[0], o[1], o[2], o[3]);
      }
      tc::fence_proxy_async();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(q_ready);
    }
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    bool fail = false;
    // after a time-out the warp stops waiting and runs out its loop: the launch's result is void
    auto wait = [&](uint32_t bar, uint32_t parity) {
      if (!fail && !tc::mbar_wait(bar, parity, abort_flag)) fail = true;
      __syncwarp();
    };
    float m = kNone, l = 0.f;
    // keys that all rows of the warp see
    int in_lo = live ? klo : 0, in_hi = live ? khi : 0x7fffffff;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      in_lo = max(in_lo, __shfl_xor_sync(0xffffffffu, in_lo, o));
      in_hi = min(in_hi, __shfl_xor_sync(0xffffffffu, in_hi, o));
    }
    if (t == 0 || two) {
      for (int j = 0; j < tiles; ++j) {
        const int key = tok0 + j * kKeys;
        wait(s_ready(t), j & 1);
        tc::tc_fence_after();
        uint32_t v[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tc::tmem_ld32(tS(t) + lanes + c * 32, v + c * 32);
        tc::tmem_ld_wait();
        if (key < in_lo || key + kKeys > in_hi) {
          const int a = klo - key, b = khi - key;
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (i < a || i >= b) v[i] = 0xff800000u;
        }
        float c0 = __uint_as_float(v[0]), c1 = __uint_as_float(v[1]), c2 = __uint_as_float(v[2]), c3 = __uint_as_float(v[3]);
#pragma unroll
        for (int i = 4; i < 124; i += 8) {
          c0 = fmaxf(c0, fmaxf(__uint_as_float(v[i]), __uint_as_float(v[i + 1])));
          c1 = fmaxf(c1, fmaxf(__uint_as_float(v[i + 2]), __uint_as_float(v[i + 3])));
          c2 = fmaxf(c2, fmaxf(__uint_as_float(v[i + 4]), __uint_as_float(v[i + 5])));
          c3 = fmaxf(c3, fmaxf(__uint_as_float(v[i + 6]), __uint_as_float(v[i + 7])));
        }
        c0 = fmaxf(c0, fmaxf(__uint_as_float(v[124]), __uint_as_float(v[125])));
        c1 = fmaxf(c1, fmaxf(__uint_as_float(v[126]), __uint_as_float(v[127])));
        const float cm = fmaxf(fmaxf(c0, c1), fmaxf(c2, c3)) * fac;
        if (__any_sync(0xffffffffu, cm > m + 8.f)) {
          // The maximum moves; rare behind the first tiles.  (The PV before is done: QK of this tile has waited for it.)
          const float nm = fmaxf(m, cm), f = ex2(m - nm);
          m = nm;
          l *= f;
          if (j) {
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t o[16];
              asm volatile(
                  "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                  : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]), "=r"(o[4]), "=r"(o[5]), "=r"(o[6]), "=r"(o[7]), "=r"(o[8]),
                    "=r"(o[9]), "=r"(o[10]), "=r"(o[11]), "=r"(o[12]), "=r"(o[13]), "=r"(o[14]), "=r"(o[15])
                  : "r"(tO(t) + lanes + c)
                  : "memory");
              tc::tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              asm volatile(
                  "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(tO(t) + lanes + c),
                  "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7]), "r"(o[8]), "r"(o[9]), "r"(o[10]),
                  "r"(o[11]), "r"(o[12]), "r"(o[13]), "r"(o[14]), "r"(o[15])
                  : "memory");
            }
          }
        }
        // s fac - m is one fma, whose product is not rounded as m was: where an ulp of m is a matter of powers of two, round it
        float ff = fac;
        if (__any_sync(0xffffffffu, fabsf(m) > 1048576.f && m != kNone)) {
#pragma unroll
          for (int i = 0; i < 128; ++i) v[i] = __float_as_uint(__fmul_rn(__uint_as_float(v[i]), fac));
          ff = 1.f;
        }
        const uint64_t f2 = pair64(ff, ff), m2 = pair64(-m, -m);
        uint64_t l0 = pair64(0.f, 0.f), l1 = l0;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int x = c * 64 + 2 * i;
            const float2 z = unpair(fma2(pair64(__uint_as_float(v[x]), __uint_as_float(v[x + 1])), f2, m2));
            const float a = ex2(z.x), b = ex2(z.y);
            if (i & 1) l1 = add2(l1, pair64(a, b));
            else l0 = add2(l0, pair64(a, b));
            pk[i] = pack<__half>(a, b);
          }
          tmem_st32(tS(t) + lanes + c * 32, pk);
        }
        const float2 s = unpair(add2(l0, l1));
        l += s.x + s.y;
        tmem_st_done();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(p_ready(t));
      }
      if (tiles) wait(pv_done(t), (tiles - 1) & 1);
      tc::tc_fence_after();
    }
    // ---- the row's result
    const bool mine = live && (t == 0 || two);
    float f = 1.f;
    if (p.splits == 1) {
      if (p.sink && live) {
        const float s2 = p.sink[head] * 1.4426950408889634f, nm = fmaxf(m, s2);
        f = ex2(m - nm);
        l = l * f + ex2(s2 - nm);
        m = nm;
      }
      f = l == 0.f ? 0.f : f / l;                        // no key and no sink: zeros
      if (mine && p.lse) p.lse[(long)row * p.heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
    }
    float* part = p.work + ((long)blockIdx.x * kRows + t * 128 + r) * (D + 4);
    T* dst = (T*)p.out + (mine ? (long)row * p.o_row + (long)head * p.o_head : 0l);
#pragma unroll 1
    for (int c = 0; c < D; c += 32) {
      uint32_t o[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = 0u;
      if (tiles && (t == 0 || two)) {
        tc::tmem_ld32(tO(t) + lanes + c, o);
        tc::tmem_ld_wait();
      }
      if (!mine) continue;
      if (p.splits == 1) {
        store32<T>(dst + c, reinterpret_cast<const float*>(o), f);
      } else {
#pragma unroll
        for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(part + c + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
      }
    }
    if (mine && p.splits > 1) *reinterpret_cast<float2*>(part + D) = make_float2(m, l);
  }
  tc::tc_fence_before();
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0) tf_report(p.st, TF_TIMEOUT, 186, blockIdx.x, it.seq);
  if (warp == 12) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// Joins the partial results of an item's CTAs in their order: one warp a row, D / 32 channels a thread.
template <int D, typename T>
__global__ void __launch_bounds__(256) paged_tc_merge_kernel(const TcParams p) {
  tf_pdl_sync();
  Item it;
  if (!item_of(p, blockIdx.x, &it)) return;
  constexpr int C = D / 32;
  const int r = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, fr = it.blk * kRows + r;
  const int tok = fr / p.group, head = it.h * p.group + fr - tok * p.group, row = it.row0 + tok;
  if (tok >= it.n || row < 0 || row >= p.r.total) return;
  float m = kNone, l = 0.f, o[C];
#pragma unroll
  for (int i = 0; i < C; ++i) o[i] = 0.f;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float* src = p.work + (((long)blockIdx.x * p.splits + s) * kRows + r) * (D + 4);
    const float2 ml = *reinterpret_cast<const float2*>(src + D);
    float v[C];
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = src[lane * C + i];
    const float nm = fmaxf(m, ml.x), f0 = ex2(m - nm), f1 = ex2(ml.x - nm);
    m = nm;
    l = l * f0 + ml.y * f1;
#pragma unroll
    for (int i = 0; i < C; ++i) o[i] = o[i] * f0 + v[i] * f1;
  }
  float f = 1.f;
  if (p.sink) {
    const float s2 = p.sink[head] * 1.4426950408889634f, nm = fmaxf(m, s2);
    f = ex2(m - nm);
    l = l * f + ex2(s2 - nm);
    m = nm;
  }
  f = l == 0.f ? 0.f : f / l;
  T* dst = (T*)p.out + (long)row * p.o_row + (long)head * p.o_head + lane * C;
#pragma unroll
  for (int i = 0; i < C; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pack<T>(o[i] * f, o[i + 1] * f);
  if (p.lse && lane == 0) p.lse[(long)row * p.heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

template <int D, typename T>
int launch_tc(const TcParams& p, long items, cudaStream_t st) {
  static unsigned long long limit_set = 0;
  if (tf_smem_limit((const void*)paged_tc_kernel<D, T>, TcShape<D>::kBytes, &limit_set) != cudaSuccess) return -2;
  tf_launch(paged_tc_kernel<D, T>, dim3((unsigned)(items * p.splits)), dim3(kThreads), TcShape<D>::kBytes, st, p);
  if (p.splits > 1) tf_launch(paged_tc_merge_kernel<D, T>, dim3((unsigned)items, kRows / 8), dim3(256), 0, st, p);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

long items_of(int total, int seqs, int group, int kv) { return ((long)total * group / kRows + seqs) * kv; }
// CTAs of an item: as many as fill the machine, where every one keeps at least four tiles of a full-length sequence
int splits_of(long items, long keys, int sms) {
  const long room = sms / items, most = keys / (4 * kKeys);
  const long n = room < most ? room : most;
  return n < 1 ? 1 : n > 64 ? 64 : (int)n;
}

}  // namespace

long paged_tc_workspace(int total, int seqs, int heads, int kv, int D, long keys, int sms) {
  const long items = items_of(total, seqs, heads / kv, kv);
  const int n = splits_of(items, keys, sms);
  return n > 1 ? items * n * kRows * (D + 4) : 0;
}

int paged_tc_attention(const paged::AttnCall& a, int sms, cudaStream_t st) {
  TcParams p = {};
  static_cast<AttnCall&>(p) = a;
  const long items = items_of(a.r.total, a.r.seqs, a.group, a.c.kv);
  p.splits = splits_of(items, (long)a.r.width << a.c.shift, sms);
  if (items * p.splits > 0x7fffffffl) return -1;
  if (a.c.D == 128) return a.kind == 1 ? launch_tc<128, __half>(p, items, st) : launch_tc<128, __nv_bfloat16>(p, items, st);
  return a.kind == 1 ? launch_tc<64, __half>(p, items, st) : launch_tc<64, __nv_bfloat16>(p, items, st);
}
