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
// Keys that no row sees are masked in S, and their values are stored as zeros, whatever their pages hold.
//
// A block of 128 rows or fewer lets both tiles have its rows and take the tiles of keys in turn; their results are joined in the end
// (4 x 8 rows x 8 heads over 32,768 tokens: 208 -> 154 us; 64 rows x 8 heads over 65,536: 245 -> 163).
//
// The unpacking warps bring their pages in by bulk copies, the next tile's as soon as this one's are in registers, and are small
// loops: a warp of each role is on every scheduler, and laid out in full (or with more registers than they have, 72) they were
// what everything waited for (4,097 rows x 8 heads at 4,096 tokens: 901 -> 836 us; PV in halves, below, -> 803).
//
// A softmax thread owns a row.  The reference maximum is the first tile's and moves (O and the sum rescaled in tensor memory) only
// when a score exceeds it by 2^8.  Registers are moved from the unpacking warps to the softmax warps (a row of S is 128 of them).
// QK of the next keys waits for the PV that reads P, whose columns it overwrites: the chain QK, softmax, PV of a row tile is what
// bounds the kernel (47 % of the tensor pipe, 48 % of the exponentials' rate).  PV of the first 64 keys runs under the softmax of the others.
// Few items (a short prompt over a long prefix): the keys of an item are cut over several CTAs, whose partial results
// paged_tc_merge_kernel joins in order.
//
// Every mbarrier wait is bounded: on a time-out the CTA raises its abort flag, reports TF_TIMEOUT, frees its tensor memory and returns.
#include "paged_tc.h"
#include "tc.cuh"

namespace {

using namespace paged;

constexpr int kRows = 256;                               // rows of a CTA
constexpr int kThreads = 512;                            // warps 0-7 softmax, 8-11 keys, 12 MMA, 13-15 values
constexpr int kMoreRegs = 184, kLessRegs = 72;           // 256 threads each: 65,536 in all, as launched

constexpr int kKeys = 128;                               // keys of a tile
constexpr float kNone = -3e38f;                          // the maximum of a row that has seen no key

struct TcParams : AttnCall {
  int cut;                                               // 1: the keys of an item are cut over CTAs; `work` holds [CTAs][rows of an item][D + 4]
};

struct Seq {
  int n, row0, pos0, key0, hi, blocks, tiles;            // rows, first row, its position; first key, last key + 1, row blocks, most key tiles of one
};
__device__ __forceinline__ Seq seq_of(const TcParams& p, int s) {
  Seq q;
  q.n = rows_of(p.r, s, &q.row0, &q.pos0);
  q.blocks = (int)(((long)q.n * p.group + kRows - 1) / kRows);
  q.key0 = first_key(p, s, q.pos0);
  q.hi = (int)min((long)p.r.lengths[s], (long)p.r.width << p.c.shift);
  q.tiles = max((q.hi - (min(q.key0, max(q.hi, 0)) & ~(kKeys - 1)) + kKeys - 1) / kKeys, 1);
  return q;
}
__device__ __forceinline__ long scan(long v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}
// Cut items: every part of an item has at most `quota` tiles, so that the parts of all items are no more than the CTAs.
__device__ __forceinline__ long quota_of(const TcParams& p, int ctas) {
  long items = 0, tiles = 0;
  for (int s0 = 0; s0 < p.r.seqs; s0 += 32) {
    const int s = s0 + (threadIdx.x & 31);
    if (s < p.r.seqs) {
      const Seq q = seq_of(p, s);
      items += (long)q.blocks * p.c.kv;
      tiles += (long)q.blocks * p.c.kv * q.tiles;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    items += __shfl_xor_sync(0xffffffffu, items, o);
    tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
  }
  const long room = max(ctas - items, 1l);
  return max((tiles + room - 1) / room, 4l);
}
struct Item {
  int seq, h, blk, n, row0, pos0, key0, lo, hi;          // key0: first key that a row of the block sees; lo, hi: this block's keys
  int part, parts;                                       // of its tiles
  long first;                                            // CTA of part 0 (cut items), or the item's own
};
// The item of CTA `index` (by_item: the index counts items): row blocks of the sequences one after another, the last (longest)
// block of a sequence first, kv heads inside, an item's parts next to each other.
__device__ __forceinline__ bool item_of(const TcParams& p, long index, long quota, bool by_item, Item* it) {
  const int lane = threadIdx.x & 31;
  long base = 0, ctas = 0;
  for (int s0 = 0; s0 < p.r.seqs; s0 += 32) {
    long w = 0;
    int parts = 1;
    if (s0 + lane < p.r.seqs) {
      const Seq q = seq_of(p, s0 + lane);
      if (quota) parts = (int)((q.tiles + quota - 1) / quota);
      w = (long)q.blocks * p.c.kv;
    }
    const long own = by_item ? w : w * parts, incl = scan(own) + base, incl_c = scan(w * parts) + ctas;
    const unsigned hit = __ballot_sync(0xffffffffu, incl > index);
    if (hit) {
      const int l = __ffs(hit) - 1;
      const long before = __shfl_sync(0xffffffffu, incl - own, l), before_c = __shfl_sync(0xffffffffu, incl_c - w * parts, l);
      const long count = __shfl_sync(0xffffffffu, w, l);
      it->parts = __shfl_sync(0xffffffffu, parts, l);
      const long at = index - before, nth = by_item ? at : at / it->parts;
      it->part = by_item ? 0 : (int)(at - nth * it->parts);
      it->first = before_c + nth * it->parts;
      const long i = count - 1 - nth;
      it->seq = s0 + l;
      it->h = (int)(i % p.c.kv);
      it->blk = (int)(i / p.c.kv);
      const Seq q = seq_of(p, it->seq);
      it->row0 = q.row0;
      it->n = q.n;
      it->pos0 = q.pos0;
      const int tok0 = it->blk * kRows / p.group, tok1 = min(((it->blk + 1) * kRows - 1) / p.group, it->n - 1);
      it->key0 = first_key(p, it->seq, q.pos0 + tok0);
      it->lo = min(it->key0, max(q.hi, 0)) & ~(kKeys - 1);
      it->hi = max((int)min((long)q.pos0 + tok1 + 1, (long)p.r.width << p.c.shift), it->lo);
      return true;
    }
    base = __shfl_sync(0xffffffffu, incl, 31);
    ctas = __shfl_sync(0xffffffffu, incl_c, 31);
  }
  return false;
}

// Joins the partial results of an item's CTAs in their order: one warp a row, D / 32 channels a thread.
template <int D, typename T>
__global__ void __launch_bounds__(256) paged_tc_merge_kernel(const TcParams p, int ctas) {
  tf_pdl_sync();
  Item it;
  if (!item_of(p, blockIdx.x, quota_of(p, ctas), true, &it) || it.parts == 1) return;
  constexpr int C = D / 32;
  const int r = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, fr = it.blk * kRows + r;
  const int tok = fr / p.group, head = it.h * p.group + fr - tok * p.group, row = it.row0 + tok;
  if (tok >= it.n) return;
  float m = kNone, l = 0.f, o[C];
#pragma unroll
  for (int i = 0; i < C; ++i) o[i] = 0.f;
  // eight parts at a time: their loads are one latency, and their sums do not wait for each other's maxima
  for (int s = 0; s < it.parts; s += 8) {
    float2 ml[8];
    float v[8][C];
    float nm = m;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      ml[k] = make_float2(kNone, 0.f);
#pragma unroll
      for (int i = 0; i < C; ++i) v[k][i] = 0.f;
      if (s + k < it.parts) {
        const float* src = p.work + ((it.first + s + k) * kRows + r) * (D + 4);
        ml[k] = *reinterpret_cast<const float2*>(src + D);
#pragma unroll
        for (int i = 0; i < C; ++i) v[k][i] = src[lane * C + i];
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) nm = fmaxf(nm, ml[k].x);
    const float f0 = ex2(m - nm);
    m = nm;
    l *= f0;
#pragma unroll
    for (int i = 0; i < C; ++i) o[i] *= f0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float f = ex2(ml[k].x - nm);
      l = fmaf(ml[k].y, f, l);
#pragma unroll
      for (int i = 0; i < C; ++i) o[i] = fmaf(v[k][i], f, o[i]);
    }
  }
  float f = 1.f, lse = row_lse(m, l);
  if (p.sink) f = take_sink(p.sink[head], m, &l, &lse);
  f = l == 0.f ? 0.f : f / l;
  T* dst = (T*)p.out + (long)row * p.o_row + (long)head * p.o_head + lane * C;
#pragma unroll
  for (int i = 0; i < C; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pack<T>(o[i] * f, o[i + 1] * f);
  if (p.lse && lane == 0) p.lse[(long)row * p.heads + head] = lse;
}

long items_of(int total, int seqs, int group, int kv) { return ((long)total * group / kRows + seqs) * kv; }
// The keys of an item are cut over CTAs where the items leave half of the SMs idle and one may have keys for two parts.
bool cut_of(long items, long keys, int sms) { return 2 * items <= sms && keys > 8 * kKeys; }

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
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void sts32(uint32_t a, uint32_t x) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(a), "r"(x) : "memory"); }
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint16_t lds16(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(a) : "memory");
  return v;
}
// 64 f16 of a row: the 128 swizzled bytes of a K-major tile; 16-byte piece c of row r
__device__ __forceinline__ uint32_t piece(uint32_t tile, int r, int c) { return tile + r * 128 + ((c ^ (r & 7)) << 4); }
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t v[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
      "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
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
// Packed keys or values of `span` tokens a lane (lanes below `count`) come into shared memory by bulk copies.  A page that no row sees is
// left out (its scores are masked, its values' scales zeroed where they are taken apart), one that cannot be read is zeros.
template <int D>
struct Pages {
  const int* table;
  const uint8_t* base;
  long page_bytes;
  int pages, shift, span, count, key0, hi, seq;
  TfStatusWord* st;
  __device__ __forceinline__ Pages(const TcParams& p, const Item& it, const uint8_t* cache, int tokens)
      : table(p.r.table + (long)it.seq * p.r.width), base(cache + it.h * p.c.block), page_bytes(p.c.kv * p.c.block), pages(p.c.pages),
        shift(p.c.shift), span(min(tokens, 1 << p.c.shift)), count(tokens / span), key0(it.key0), hi(it.hi), seq(it.seq), st(p.st) {}
  // page of the lane's tokens, -2 where no row sees one
  __device__ __forceinline__ int find(int tok0, bool more) const {
    const int lane = threadIdx.x & 31, tok = tok0 + lane * span;
    return more && lane < count && tok < hi && tok + span > key0 ? __ldg(table + (tok >> shift)) : -2;
  }
  // `data` holds the tokens' codes, then their scales; all lanes of a warp
  __device__ __forceinline__ void copy(int pg, int tok0, uint32_t data, uint32_t scales, uint32_t full) const {
    const int lane = threadIdx.x & 31, at = (tok0 + lane * span) & ((1 << shift) - 1);
    const bool ok = (unsigned)pg < (unsigned)pages;
    data += lane * span * (D / 2);
    scales += lane * span * (D / 16);
    if (!ok && pg != -2) {
      for (int i = 0; i < span * (D / 2); i += 16) sts128(data + i, 0u, 0u, 0u, 0u);
      for (int i = 0; i < span * (D / 16); i += 16) sts128(scales + i, 0u, 0u, 0u, 0u);
      tc::fence_proxy_async();
      tf_report(st, TF_BAD_INDEX, 185, seq, pg);
    }
    __syncwarp();
    const int n = __popc(__ballot_sync(0xffffffffu, ok));
    if (lane == 0) tc::mbar_expect_tx(full, n * span * (D / 2 + D / 16));
    __syncwarp();
    if (ok) {
      const uint8_t* src = base + pg * page_bytes;
      tc::bulk_g2s(data, src + at * (D / 2), span * (D / 2), full);
      tc::bulk_g2s(scales, src + ((D >> 1) << shift) + at * (D / 16), span * (D / 16), full);
    }
  }
};
// a copy that nobody waits for any more lands before the CTA leaves
__device__ __forceinline__ void drain(uint32_t full, uint32_t parity) {
  const long long t0 = clock64();
  while (!tc::mbar_try(full, parity) && clock64() - t0 < 2000000000ll) {}
}

// Keys: warp w of four has 32 tokens of a tile, in its own part of `staged`, and a thread takes 32 channels of one.  What it has read into
// registers makes room for the next tile's.
template <int D>
__device__ __forceinline__ void unpack_keys(const Pages<D> s, int w, int tok0, int tiles, uint32_t staged, uint32_t filled, uint32_t tiles_at,
                                            uint32_t full, uint32_t empty, volatile int* abort_flag) {
  constexpr int LR = D / 32, RW = 32 / LR, N = 32 / RW;  // lanes of a row, rows of an item, items
  const int lane = threadIdx.x & 31, sub = lane % LR, row = lane / LR;
  const uint32_t codes = staged + w * 32 * (D / 2 + D / 16), scales = codes + 16 * D;
  const bool swap = LR == 4 && (sub & 2);                // (lanes whose pieces would fall on the same banks store theirs in another order)
  const uint32_t at = (32 * w + row) * 128 + (((((sub & 1) * 4) | (swap ? 2 : 0)) ^ (row & 7)) << 4) + (sub >> 1) * (128 * 128);
  tok0 += 32 * w;
  if (tiles > 0) s.copy(s.find(tok0, true), tok0, codes, scales, filled);
  int pg = s.find(tok0 + kKeys, tiles > 1);
  for (int j = 0; j < tiles; ++j) {
    if (!tc::mbar_wait(filled, j & 1, abort_flag)) return drain(filled, j & 1);
    const int b = j & 1, next = tok0 + (j + 1) * kKeys;
    if (!tc::mbar_wait(empty + 8 * b, ((j >> 1) & 1) ^ 1, abort_flag)) return;
    uint32_t src = codes + lane * 16, ssc = scales + row * (D / 16) + sub * 2, tile = tiles_at + b * (256 * D) + at;
    uint4 d = lds128(src);
    uint32_t sc = lds16(ssc);
    // (a loop: the SM's warps run four programs, and what is laid out in full is fetched from afar every time)
#pragma unroll 1
    for (int i = 0; i < N; ++i, tile += RW * 128) {
      const uint32_t ss = e4m3x2_to_h2((uint16_t)sc), s0 = __byte_perm(ss, 0, swap ? 0x3232 : 0x1010), s1 = __byte_perm(ss, 0, swap ? 0x1010 : 0x3232);
      const uint32_t y[4] = {swap ? d.z : d.x, swap ? d.w : d.y, swap ? d.x : d.z, swap ? d.y : d.w};
      if (i + 1 < N) {
        d = lds128(src += 512);
        sc = lds16(ssc += RW * (D / 16));
      } else {
        __syncwarp();
        if (j + 1 < tiles) s.copy(pg, next, codes, scales, filled);
        pg = s.find(next + kKeys, j + 2 < tiles);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t f = e < 2 ? s0 : s1;
        uint32_t h[4];
        fp4::e2m1x8_to_h2x4(y[e], h);
        sts128(tile ^ (e << 4), fp4::hmul2(h[0], f), fp4::hmul2(h[1], f), fp4::hmul2(h[2], f), fp4::hmul2(h[3], f));
      }
    }
    tc::fence_proxy_async();
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(full + 8 * b);
  }
}

// Values: three warps share a tile's 64 pairs of tokens, and a thread takes 16 channels of one at a time.  The lanes of a warp take their
// channels from different ones on: the same channels of 32 pairs would all be read from the same banks.
template <int D>
__device__ __forceinline__ void unpack_values(const Pages<D> s, int w, int tok0, int tiles, uint32_t staged, uint32_t filled, uint32_t taken,
                                              uint32_t tiles_at, uint32_t full, uint32_t empty, volatile int* abort_flag) {
  constexpr int C = D / 16;                              // blocks of channels; an item x is one of 32 pairs from 32 (x & 1) on
  const int lane = threadIdx.x & 31, turn = D == 128 ? lane : lane >> 1;
  const uint32_t scales = staged + 64 * D, at = ((lane >> 2) << 4) + (lane & 3) * 4;
  const uint32_t src = staged + lane * D, ssc = scales + lane * (D / 8);
  int pg = -2;
  if (w == 0) {
    if (tiles > 0) s.copy(s.find(tok0, true), tok0, staged, scales, filled);
    pg = s.find(tok0 + kKeys, tiles > 1);
  }
  for (int j = 0; j < tiles; ++j) {
    const int b = j & 1;
    if (!tc::mbar_wait(filled, j & 1, abort_flag)) return drain(filled, j & 1);
    if (!tc::mbar_wait(empty + 8 * b, ((j >> 1) & 1) ^ 1, abort_flag)) return;
    const uint32_t tile = tiles_at + b * (256 * D) + at;
    const int first = tok0 + j * kKeys + 2 * lane;
    int c = (turn + (w >> 1)) & (C - 1);
    uint4 d = lds128(src + (w & 1) * (32 * D) + c * 16);
    uint32_t sc = lds16(ssc + (w & 1) * (4 * D) + c * 2);
#pragma unroll 1
    for (int x = w; x < 2 * C; x += 3) {
      const int tok = first + 64 * (x & 1);
      const uint32_t seen = (tok >= s.key0 && tok < s.hi ? 0xffu : 0u) | (tok + 1 >= s.key0 && tok + 1 < s.hi ? 0xff00u : 0u);
      // 64 tokens: [D][128 bytes]; eight rows in a row take the eight orders of the swizzle
      const uint32_t f = e4m3x2_to_h2((uint16_t)(sc & seen)), to = tile + (x & 1) * (D * 128) + c * (16 * 128);
      const uint32_t y[4] = {d.x, d.y, d.z, d.w};
      const int n = x + 3;
      if (n < 2 * C) {
        c = (turn + (n >> 1)) & (C - 1);
        d = lds128(src + (n & 1) * (32 * D) + c * 16);
        sc = lds16(ssc + (n & 1) * (4 * D) + c * 2);
      } else {
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(taken);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t h[4];
        fp4::e2m1x8_to_h2x4(y[e], h);
#pragma unroll
        for (int k = 0; k < 4; ++k) sts32((to ^ (((4 * e + k) & 7) << 4)) + (4 * e + k) * 128, fp4::hmul2(h[k], f));
      }
    }
    if (w == 0 && j + 1 < tiles) {
      const int next = tok0 + (j + 1) * kKeys;
      if (!tc::mbar_wait(taken, j & 1, abort_flag)) return;
      s.copy(pg, next, staged, scales, filled);
      pg = s.find(next + kKeys, j + 2 < tiles);
    }
    tc::fence_proxy_async();
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(full + 8 * b);
  }
}

template <int D>
struct TcShape {
  static constexpr int kTile = 128 * D * 2;              // bytes of a tile of 128 rows (Q, K) or of a transposed value tile
  static constexpr int kPacked = 128 * (D / 2 + D / 16);                // keys or values of a tile as the pages have them
  static constexpr int kBytes = 6 * kTile + 2 * kPacked + 1024 + 256;   // two tiles of Q, two stages of K and V, packed ones, barriers
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
  uint8_t* tail = smem_raw + (base - raw) + 6 * S::kTile + 2 * S::kPacked;
  const uint32_t q_s = base, k_s = base + 2 * S::kTile, v_s = base + 4 * S::kTile;
  const uint32_t staged = base + 6 * S::kTile, bar0 = staged + 2 * S::kPacked;
  const uint32_t q_ready = bar0;
  auto k_full = [&](int s) { return bar0 + 8u + 8u * s; };
  auto k_empty = [&](int s) { return bar0 + 24u + 8u * s; };
  auto v_full = [&](int s) { return bar0 + 40u + 8u * s; };
  auto v_empty = [&](int s) { return bar0 + 56u + 8u * s; };
  auto s_ready = [&](int t) { return bar0 + 72u + 8u * t; };
  auto p_ready = [&](int t) { return bar0 + 88u + 8u * t; };
  auto pv_done = [&](int t) { return bar0 + 104u + 8u * t; };
  auto p_half = [&](int t) { return bar0 + 168u + 8u * t; };            // P of the first 64 keys
  const uint32_t filled = bar0 + 120u, taken = bar0 + 160u;             // packed keys of the four warps, values; values read
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(tail + 184);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 192);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  tf_pdl_sync();
  Item it;
  if (!item_of(p, blockIdx.x, p.cut ? quota_of(p, gridDim.x) : 0, false, &it)) return;
  if (threadIdx.x == 0) {
    tc::mbar_init(q_ready, 8);
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(k_full(s), 4);
      tc::mbar_init(k_empty(s), 1);
      tc::mbar_init(v_full(s), 3);
      tc::mbar_init(v_empty(s), 1);
      tc::mbar_init(s_ready(s), 1);
      tc::mbar_init(p_ready(s), 4);
      tc::mbar_init(p_half(s), 4);
      tc::mbar_init(pv_done(s), 1);
    }
    for (int s = 0; s < 5; ++s) tc::mbar_init(filled + 8 * s, 1);
    tc::mbar_init(taken, 3);
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
  const int j0 = (int)((long)all * it.part / it.parts), tiles = (int)((long)all * (it.part + 1) / it.parts) - j0;
  const int tok0 = it.lo + j0 * kKeys;
  // The block has rows for both tiles; with one, the two take turns at the key tiles with the same rows, and their results are joined.
  const bool two = it.blk * kRows + 128 < it.n * p.group;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLessRegs));
    if (warp < 12) {
      const int w = warp - 8;
      unpack_keys<D>(Pages<D>(p, it, p.c.k, 32), w, tok0, tiles, staged, filled + 8 * w, k_s, k_full(0), k_empty(0), abort_flag);
    } else if (warp > 12) {
      unpack_values<D>(Pages<D>(p, it, p.c.v, kKeys), warp - 13, tok0, tiles, staged + S::kPacked, filled + 32, taken, v_s, v_full(0), v_empty(0),
                       abort_flag);
    } else {
      // ---------------------------------------------------------------- MMA issuer (the warp waits, one thread issues)
      constexpr uint32_t id_qk = tc::instr_desc(0, 0, 128, 128), id_pv = tc::instr_desc(0, 0, 128, D);
      const bool one = tc::elect_one();
      auto qk = [&](int t, int j) {
        const uint32_t q0 = q_s + t * S::kTile, k0 = k_s + (j & 1) * S::kTile;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          tc::mma_f16(tS(t), tc::smem_desc_sw128(q0 + (k >> 2) * 16384) + 2 * (k & 3), tc::smem_desc_sw128(k0 + (k >> 2) * 16384) + 2 * (k & 3),
                      id_qk, k ? 1u : 0u);
        tc::mma_commit(s_ready(t));
      };
      // (64 keys at a time: the first half runs while the softmax warps are at the second)
      auto pv = [&](int t, int j, int half, bool more) {
        const uint32_t v0 = v_s + (j & 1) * S::kTile + half * (D * 128);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_ts(tO(t), tS(t) + 32 * half + 8 * k, tc::smem_desc_sw128(v0) + 2 * k, id_pv, (more || k || half) ? 1u : 0u);
        if (half) tc::mma_commit(pv_done(t));
      };
      auto wait = [&](uint32_t bar, uint32_t parity) { return tc::mbar_wait(bar, parity, abort_flag); };
      bool ok = wait(q_ready, 0);
      if (two) {
        if (ok && tiles && (ok = wait(k_full(0), 0))) {
          tc::tc_fence_after();
          if (one) {
            qk(0, 0);
            qk(1, 0);
            tc::mma_commit(k_empty(0));
          }
        }
        for (int j = 0; j < tiles && ok; ++j) {
          const uint32_t ph = j & 1, rph = (j >> 1) & 1;
          const bool next = j + 1 < tiles;
          if (!(ok = wait(v_full(ph), rph) && wait(p_half(0), ph))) break;
          tc::tc_fence_after();
          if (one) pv(0, j, 0, j > 0);
          if (!(ok = wait(p_ready(0), ph))) break;
          tc::tc_fence_after();
          if (one) pv(0, j, 1, true);
          if (next) {
            if (!(ok = wait(k_full(ph ^ 1), ((j + 1) >> 1) & 1) && wait(pv_done(0), ph))) break;
            tc::tc_fence_after();
            if (one) qk(0, j + 1);
          }
          if (!(ok = wait(p_half(1), ph))) break;
          tc::tc_fence_after();
          if (one) pv(1, j, 0, j > 0);
          if (!(ok = wait(p_ready(1), ph))) break;
          tc::tc_fence_after();
          if (one) {
            pv(1, j, 1, true);
            tc::mma_commit(v_empty(ph));
          }
          if (next) {
            if (!(ok = wait(pv_done(1), ph))) break;
            tc::tc_fence_after();
            if (one) {
              qk(1, j + 1);
              tc::mma_commit(k_empty(ph ^ 1));
            }
          }
        }
      } else {
        for (int j = 0; j < 2 && j < tiles && ok; ++j) {
          if (!(ok = wait(k_full(j), 0))) break;
          tc::tc_fence_after();
          if (one) {
            qk(j, j);
            tc::mma_commit(k_empty(j));
          }
        }
        for (int j = 0; j < tiles && ok; ++j) {
          const int t = j & 1;
          const uint32_t ph = (j >> 1) & 1;
          if (!(ok = wait(v_full(t), ph) && wait(p_half(t), ph))) break;
          tc::tc_fence_after();
          if (one) pv(t, j, 0, j > 1);
          if (!(ok = wait(p_ready(t), ph))) break;
          tc::tc_fence_after();
          if (one) {
            pv(t, j, 1, true);
            tc::mma_commit(v_empty(t));
          }
          if (j + 2 < tiles) {
            if (!(ok = wait(k_full(t), ph ^ 1) && wait(pv_done(t), ph))) break;
            tc::tc_fence_after();
            if (one) {
              qk(t, j + 2);
              tc::mma_commit(k_empty(t));
            }
          }
        }
      }
      // the last commits arrive at this CTA's barriers before it may leave
      for (int j = max(tiles - 2, 0); j < tiles && ok; ++j) ok = wait(v_empty(j & 1), (j >> 1) & 1);
      if (*abort_flag) {
        const long long t0 = clock64();
        while (clock64() - t0 < 400000) {}       // MMAs in flight end
      }
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMoreRegs));
    // ------------------------------------------------------------------ softmax: one row per thread
    // (one tile of rows: the second takes them 64 lanes on, so that few rows are on two of the SM's four schedulers)
    const int t = warp >> 2, r = (warp & 3) * 32 + lane, fr = it.blk * kRows + (two ? t * 128 + r : t ? (r + 64) & 127 : r);
    const int tok = fr / p.group, head = it.h * p.group + fr - tok * p.group, row = it.row0 + tok;
    const bool live = tok < it.n;
    const int pos = it.pos0 + tok, klo = first_key(p, it.seq, pos);
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
      fac = fmaxf(ldexpf(p.scale2, min(ex, 126)), 1.17549435e-38f);      // (a zero would make NaN of masked scores; logits are below 2^-100 either way)
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
    const bool any = __any_sync(0xffffffffu, live);
    const int step = two ? 1 : 2;
    int done = 0;                                        // tiles that this warp has done
    for (int j = two ? 0 : t; j < tiles; j += step, ++done) {
      {
        const int key = tok0 + j * kKeys;
        wait(s_ready(t), done & 1);
        tc::tc_fence_after();
        if (!any) {
          // no rows: whatever stands there as P stays in rows that nobody stores
          __syncwarp();
          if (lane == 0) {
            tc::mbar_arrive(p_half(t));
            tc::mbar_arrive(p_ready(t));
          }
          continue;
        }
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
        float most[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) most[i] = fmaxf(__uint_as_float(v[i]), __uint_as_float(v[8 + i]));
#pragma unroll
        for (int i = 16; i < 128; i += 16)
#pragma unroll
          for (int c = 0; c < 8; ++c) most[c] = fmaxf(fmaxf(most[c], __uint_as_float(v[i + 2 * c])), __uint_as_float(v[i + 2 * c + 1]));
        const float cm = fmaxf(fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])), fmaxf(fmaxf(most[4], most[5]), fmaxf(most[6], most[7]))) * fac;
        if (__any_sync(0xffffffffu, cm > m + 8.f)) {
          // The maximum moves; rare behind the first tiles.  (The PV before is done: QK of this tile has waited for it.)
          const float nm = fmaxf(m, cm), f = ex2(m - nm);
          m = nm;
          l *= f;
          if (done) {
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
              tmem_st16(tO(t) + lanes + c, o);
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
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int x = c * 32 + 2 * i;
            const float2 z = unpair(fma2(pair64(__uint_as_float(v[x]), __uint_as_float(v[x + 1])), f2, m2));
            const float a = ex2(z.x), b = ex2(z.y);
            if (i & 1) l1 = add2(l1, pair64(a, b));
            else l0 = add2(l0, pair64(a, b));
            pk[i] = pack<__half>(a, b);
          }
          tmem_st16(tS(t) + lanes + c * 16, pk);
          if (c & 1) {
            tmem_st_done();
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(c == 1 ? p_half(t) : p_ready(t));
          }
        }
        const float2 s = unpair(add2(l0, l1));
        l += s.x + s.y;
      }
    }
    if (done) wait(pv_done(t), (done - 1) & 1);
    tc::tc_fence_after();
    float* half = reinterpret_cast<float*>(smem_raw + (k_s - raw));      // [128][D + 4]: the tiles of K and V are no longer read
    if (!two) {
      // the second tile's results go to the first one's threads
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (t && any) {
        float* dst = half + (fr - it.blk * kRows) * (D + 4);
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
          __syncwarp();                                  // (a load of tensor memory is one of the whole warp)
          if (done) {
            tc::tmem_ld32(tO(t) + lanes + c, o);
            tc::tmem_ld_wait();
          }
          if (live) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(dst + c + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
        if (live) *reinterpret_cast<float2*>(dst + D) = make_float2(m, l);
        __syncwarp();
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
    }
    // ---- the row's result
    const bool mine = live && (t == 0 || two);
    float f = 1.f, g = 0.f;
    const float* other = half + r * (D + 4);
    if (!two && mine) {
      const float2 ml = *reinterpret_cast<const float2*>(other + D);
      const float nm = fmaxf(m, ml.x);
      f = ex2(m - nm);
      g = ex2(ml.x - nm);
      l = l * f + ml.y * g;
      m = nm;
    }
    const bool whole = it.parts == 1;
    if (whole) {
      float w = 1.f, lse = row_lse(m, l);
      if (p.sink && live) w = take_sink(p.sink[head], m, &l, &lse);
      w = l == 0.f ? 0.f : w / l;                        // no key and no sink: zeros
      f *= w;
      g *= w;
      if (mine && p.lse) p.lse[(long)row * p.heads + head] = lse;
    }
    float* part = p.work + ((long)blockIdx.x * kRows + (two ? t * 128 : 0) + r) * (D + 4);
    T* dst = (T*)p.out + (mine ? (long)row * p.o_row + (long)head * p.o_head : 0l);
#pragma unroll 1
    for (int c = 0; c < D; c += 32) {
      uint32_t o[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = 0u;
      __syncwarp();
      if (done && any) {
        tc::tmem_ld32(tO(t) + lanes + c, o);
        tc::tmem_ld_wait();
      }
      if (mine) {
        float* x = reinterpret_cast<float*>(o);
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] *= f;
        if (!two) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 y = *reinterpret_cast<const float4*>(other + c + i);
            x[i] = fmaf(y.x, g, x[i]);
            x[i + 1] = fmaf(y.y, g, x[i + 1]);
            x[i + 2] = fmaf(y.z, g, x[i + 2]);
            x[i + 3] = fmaf(y.w, g, x[i + 3]);
          }
        }
        if (whole) {
          store32<T>(dst + c, x, 1.f);
        } else {
#pragma unroll
          for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(part + c + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
      }
    }
    if (mine && !whole) *reinterpret_cast<float2*>(part + D) = make_float2(m, l);
  }
  tc::tc_fence_before();
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0) tf_report(p.st, TF_TIMEOUT, 186, blockIdx.x, it.seq);
  if (warp == 12) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

template <int D, typename T>
int launch_tc(const TcParams& p, long items, int sms, cudaStream_t st) {
  static unsigned long long limit_set = 0;
  if (tf_smem_limit((const void*)paged_tc_kernel<D, T>, TcShape<D>::kBytes, &limit_set) != cudaSuccess) return -2;
  tf_launch(paged_tc_kernel<D, T>, dim3((unsigned)(p.cut ? sms : items)), dim3(kThreads), TcShape<D>::kBytes, st, p);
  // (rows of an item: at most those of the call)
  const int rows = (int)((long)p.r.total * p.group < kRows ? (long)p.r.total * p.group : kRows);
  if (p.cut) tf_launch(paged_tc_merge_kernel<D, T>, dim3((unsigned)items, (rows + 7) / 8), dim3(256), 0, st, p, sms);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace

long paged_tc_workspace(int total, int seqs, int heads, int kv, int D, long keys, int sms) {
  return cut_of(items_of(total, seqs, heads / kv, kv), keys, sms) ? (long)sms * kRows * (D + 4) : 0;
}

int paged_tc_attention(const paged::AttnCall& a, int sms, cudaStream_t st) {
  TcParams p = {};
  static_cast<AttnCall&>(p) = a;
  const long items = items_of(a.r.total, a.r.seqs, a.group, a.c.kv);
  if (items > 0x7fffffffl) return -1;
  p.cut = cut_of(items, (long)a.r.width << a.c.shift, sms);
  if (a.c.D == 128) return a.kind == 1 ? launch_tc<128, __half>(p, items, sms, st) : launch_tc<128, __nv_bfloat16>(p, items, sms, st);
  return a.kind == 1 ? launch_tc<64, __half>(p, items, sms, st) : launch_tc<64, __nv_bfloat16>(p, items, sms, st);
}
