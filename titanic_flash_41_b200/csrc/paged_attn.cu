// Attention of a few query rows a sequence over the paged 4-bit cache (decode steps, verification blocks); rows of longer
// prompts take paged_tc.cu.
//
//   o[i, h] = sum_j p_ij v_j / (sum_j p_ij + e^sink_h),  p_ij = exp(scale q_ih . k_j)     max(first, pos_i - window + 1) <= j <= pos_i
//
// Bound by HBM: a token's keys and values of one head are 144 bytes at 128 channels, read once for all query heads that share
// them and all rows of a block.  What stands against the bytes is taking the nibbles apart: 4,096 values per 16 tokens and
// head.  So both products have the CACHE on the M side of `mma.sync.m16n8k16` and the query rows (8 a column tile) on the N side:
//   S^T[16 tokens, rows] = K[tokens, D] Q^T       A = keys: a thread's 16 bytes of a key row are its fragments of D / 16 steps
//   O^T[16 channels, rows] += V^T P^T             A = values: a byte is one channel of two tokens, a register of the fragment
// One cvt turns a byte into a register and one multiplication applies its scale, with nothing moved between threads; the
// order of the channels inside a step and of the channels in the M tiles is chosen to suit (sums and outputs do not mind).
// The probabilities, tokens by rows, become the B operand by `movmatrix`.  Queries on the M side would waste half of
// every MMA at eight heads a key head.
//
// The cache streams through a ring per warp (bulk copies, 32 or 64 tokens a stage; a warp waits for its own copies only).  The work
// of a launch, (sequence, kv head, row block) x units of a stage, is laid end to end and cut into equal ranges, one a CTA, so that
// ragged sequences and few heads still fill the machine; a range that begins or ends inside an item leaves a partial result
// (fp32, with its maximum and sum) that paged_merge_kernel joins in the order of the ranges.
// Sums, maxima and O are fp32; the keys' and values' numbers are exact in f16; q is exact up to 2^-24 of its row's maximum (a
// power of two per row brings it into f16's range); p is rounded to f16 (2^-11: below
// the rounding of a bf16 output, as much as an f16 one's).
// Measured: 4 sequences of 131,072 tokens x 8 heads of 128, one row of 64 heads each, 125 - 134 us, 4.5 - 4.8 TB/s (0.7 of the copy rate); four rows each
// of three ragged ones, 97 us: there the MMAs, 38 % busy, wait for two warps a scheduler.
#include "paged_tc.h"
#include "tc.cuh"

namespace {

using namespace paged;

constexpr float kNone = -3e38f;                          // the maximum of a row that has seen no key

struct AttnParams : AttnCall {
  int whole;                                             // 1: an item is never cut; `work` holds [2 * CTAs][RB][D + 4] otherwise
};

template <int D, int NT>
struct Shape {
  static constexpr int RB = 8 * NT;                      // rows of a block
  // Tokens of a ring stage, and those whose scores a warp holds at a time.  With stages of 64 tokens a page of 64 is two copies, and the loop
  // around the MMAs, a fifth of the instructions of 32 tokens, runs half as often: 4 x 131,072 tokens of 8 heads of 128, one row, 143 -> 134
  // us (the copies of 32 alone took 127); two rows of one 67 -> 61; 4 x 32,768 of 64 channels 41 -> 37.
  static constexpr int kUnit = D == 128 || NT == 1 ? 64 : 32, kOwn = D == 64 ? kUnit : 32;
  // Warps that keep O (D / 4 x NT registers a thread) without spilling.  With ring stages of 32 tokens, 16 rows at 128 channels: two CTAs
  // of 6 warps 69 us over 131,072 tokens of 8 heads, of 8 warps (128 registers, spilled) 83; 32 rows at 64 channels: 77 us so, one CTA of
  // 8 85.
  static constexpr int kWarps = D * NT == 256 || (D == 128 && NT == 1) ? 6 : 8;
  static constexpr int kKeys = kUnit * D / 2, kScales = kUnit * D / 16;
  static constexpr int kStage = 2 * kKeys + 2 * kScales; // as in a page: keys, their scales, values, their scales
  static constexpr int kSK = kKeys, kV = kKeys + kScales, kSV = kV + kKeys;
  static constexpr int kCtas = D * NT <= 256 ? 2 : 1;          // CTAs of an SM (registers)
  static constexpr int kStages = kUnit * D == 64 * 128 ? (NT <= 2 ? 2 : 3) : kUnit * D == 32 * 64 ? 6 : 3;
  static constexpr int kQ = NT > 1 ? 32 * 8 * NT * (D / 16) : 0;      // queries in shared memory: uint2 [step][tile][lane]
  static constexpr int kRowF = D + 4;
  static constexpr int kJoin = kWarps * RB * (kRowF + 2) * 4;
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kBytes = (kRing > kJoin ? kRing : kJoin) + kQ + RB * 8 + kWarps * kStages * 8 + 16;
};

struct Seq {
  int n, row0, pos0, key0, lo, hi, units, blocks;        // rows, first row, its position, first key, its unit, last key + 1, units, row blocks
};
template <typename S>
__device__ __forceinline__ Seq seq_of(const AttnParams& p, int s) {
  Seq q;
  q.n = rows_of(p.r, s, &q.row0, &q.pos0);
  q.key0 = first_key(p, s, q.pos0);
  q.hi = (int)min((long)p.r.lengths[s], (long)p.r.width << p.c.shift);
  q.lo = min(q.key0, max(q.hi, 0)) & ~(S::kUnit - 1);
  q.units = max((q.hi - q.lo + S::kUnit - 1) / S::kUnit, 1);   // (a sequence without keys still gets its rows written)
  q.blocks = (q.n * p.group + S::RB - 1) / S::RB;
  return q;
}
__device__ __forceinline__ long warp_scan(long v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}
// Walks the sequences until the running total of `weight` passes `target`: the sequence, and the total before it.  Returns
// false (and the grand total) when it never does.
template <typename S, bool UNITS>
__device__ __forceinline__ bool locate(const AttnParams& p, long target, int* seq, long* before) {
  if (!UNITS && !p.r.cu) {
    // a row a sequence: no walk (1,024 of 300 tokens x 8 heads of 64: 371 us with it, 164 so)
    const int each = (p.group + S::RB - 1) / S::RB * p.c.kv;
    if (target >= (long)each * min(p.r.total, p.r.seqs)) return false;
    *seq = (int)(target / each);
    *before = (long)*seq * each;
    return true;
  }
  const int lane = threadIdx.x & 31;
  long base = 0;
  for (int s0 = 0; s0 < p.r.seqs; s0 += 32) {
    long w = 0;
    if (s0 + lane < p.r.seqs) {
      const Seq q = seq_of<S>(p, s0 + lane);
      w = (long)q.blocks * p.c.kv * (UNITS ? q.units : 1);
    }
    const long incl = warp_scan(w) + base;
    const unsigned hit = __ballot_sync(0xffffffffu, incl > target);
    if (hit) {
      const int l = __ffs(hit) - 1;
      *seq = s0 + l;
      *before = __shfl_sync(0xffffffffu, incl - w, l);
      return true;
    }
    base = __shfl_sync(0xffffffffu, incl, 31);
  }
  *before = base;
  return false;
}

__device__ __forceinline__ uint32_t trans8x8(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2(uint16_t v) { return e4m3x2_to_h2(v); }

// rows of a block: maximum, sum and weighted values, already relative to the row's maximum -> out and lse
template <typename T>
__device__ __forceinline__ void finish4(const AttnParams& p, const Seq& q, int h, int fr, int c, float M, float L, float4 o) {
  const int tok = fr / p.group, head = h * p.group + fr - tok * p.group, row = q.row0 + tok;
  if (tok >= q.n) return;
  float lse = row_lse(M, L);
  if (p.sink) {
    const float f = take_sink(p.sink[head], M, &L, &lse);
    o.x *= f; o.y *= f; o.z *= f; o.w *= f;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;            // no key and no sink: zeros
  uint2 w = make_uint2(pack<T>(o.x * inv, o.y * inv), pack<T>(o.z * inv, o.w * inv));
  *reinterpret_cast<uint2*>((T*)p.out + (long)row * p.o_row + (long)head * p.o_head + c) = w;
  if (p.lse && c == 0) p.lse[(long)row * p.heads + head] = lse;
}

template <int D, int NT, typename T>
__global__ void __launch_bounds__(Shape<D, NT>::kWarps * 32, Shape<D, NT>::kCtas) paged_attn_kernel(const AttnParams p) {
  using S = Shape<D, NT>;
  constexpr int RB = S::RB, KS = D / 16, KW = D / 32;    // 16-channel steps, words a thread has of a key row
  constexpr int CH = D / 8;                              // channels a thread has of a value row
  constexpr int TI = S::kOwn / 16, PIECES = S::kUnit / 16;             // tiles of 16 tokens at a time; most pages of a stage
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t* tail = smem + (S::kRing > S::kJoin ? S::kRing : S::kJoin);
  uint2* sq = reinterpret_cast<uint2*>(tail);
  int2* range = reinterpret_cast<int2*>(tail + S::kQ);   // keys of every row of the block
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + S::kQ + RB * 8);
  tf_pdl_sync();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  int seq;
  long before, total;
  long u, u_end, quota = 0;
  if (p.whole) {
    // one item a CTA
    if (!locate<S, false>(p, blockIdx.x, &seq, &before)) return;
    u = 0;
    u_end = 1;
  } else {
    locate<S, true>(p, 0x7fffffffffffffffl, &seq, &total);
    quota = max((total + gridDim.x - 1) / gridDim.x, (long)2 * S::kWarps);
    u = blockIdx.x * quota;
    u_end = min(u + quota, total);
    if (u >= u_end) return;
  }
  const long u_begin = u;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * S::kStages * S::kStage;
  uint8_t* ring_p = smem + warp * S::kStages * S::kStage;
  const uint32_t bars = tc::smem_u32(tail) + S::kQ + RB * 8 + 16 + warp * S::kStages * 8;
  if (threadIdx.x == 0) *abort_flag = 0;
  if (lane == 0) {
    for (int i = 0; i < S::kStages; ++i) tc::mbar_init(bars + 8 * i, 1);
    tc::fence_barrier_init();
  }
  __syncwarp();
  int stage = 0, ahead = 0;                              // ring stage that is read next, and that is filled next
  uint32_t phase = 0;
  bool ok = true;
  while (u < u_end) {
    long item;
    int ua, ub;                                          // units of the item that are done here
    if (p.whole) {
      item = blockIdx.x - before;
    } else {
      locate<S, true>(p, u, &seq, &before);
    }
    const Seq q = seq_of<S>(p, seq);
    if (p.whole) {
      ua = 0;
      ub = q.units;
    } else {
      item = (u - before) / q.units;
      ua = (int)(u - before - item * q.units);
      ub = (int)min((long)q.units, ua + (u_end - u));
    }
    const int h = (int)(item % p.c.kv), blk = (int)(item / p.c.kv);
    // ---- the block's queries and key ranges
    uint32_t qf[NT > 1 ? 1 : KS][2];
    float fac[NT][2];
    int in_lo = 0, in_hi = 0x7fffffff;                   // keys that every row of the block sees
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int fr = blk * RB + nt * 8 + g, tok = fr / p.group, head = h * p.group + fr - tok * p.group, row = q.row0 + tok;
      const bool live = tok < q.n;
      uint4 raw[D / 32];
      float am = 0.f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        raw[i] = make_uint4(0u, 0u, 0u, 0u);
        if (live) raw[i] = *reinterpret_cast<const uint4*>((const T*)p.q + (long)row * p.q_row + (long)head * p.q_head + t * (D / 4) + i * 8);
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = two<T>(w[e]);
          am = fmaxf(am, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 1));
      am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 2));
      // a power of two brings the row's largest element into [1, 2)
      const int ex = am > 0.f && am < INFINITY ? (int)(__float_as_uint(am) >> 23) - 127 : 0;
      const float down = __uint_as_float((uint32_t)(127 - min(ex, 126)) << 23);
      const float up = ldexpf(p.scale2, min(ex, 126));
      fac[nt][0] = __shfl_sync(0xffffffffu, up, (2 * t) * 4);
      fac[nt][1] = __shfl_sync(0xffffffffu, up, (2 * t + 1) * 4);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = two<T>(w[e]);
          o[e] = pack<__half>(f.x * down, f.y * down);
        }
        if (NT == 1) {
          qf[NT > 1 ? 0 : 2 * i][0] = o[0];
          qf[NT > 1 ? 0 : 2 * i][1] = o[1];
          qf[NT > 1 ? 0 : 2 * i + 1][0] = o[2];
          qf[NT > 1 ? 0 : 2 * i + 1][1] = o[3];
        } else if (warp == 0) {
          sq[((2 * i) * NT + nt) * 32 + lane] = make_uint2(o[0], o[1]);
          sq[((2 * i + 1) * NT + nt) * 32 + lane] = make_uint2(o[2], o[3]);
        }
      }
      const int pos = q.pos0 + tok, klo = first_key(p, seq, pos);
      const int khi = min(pos + 1, q.hi);
      if (warp == 0 && t == 0) range[nt * 8 + g] = live ? make_int2(klo, khi) : make_int2(0, 0);
      if (live) {
        in_lo = max(in_lo, klo);
        in_hi = min(in_hi, khi);
      }
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      in_lo = max(in_lo, __shfl_xor_sync(0xffffffffu, in_lo, o));
      in_hi = min(in_hi, __shfl_xor_sync(0xffffffffu, in_hi, o));
    }
    __syncthreads();                                     // queries and ranges are in shared memory

    float O[KS][NT][4];
#pragma unroll
    for (int j = 0; j < KS; ++j)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) O[j][nt][c] = 0.f;
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = kNone;
      l[nt][0] = l[nt][1] = 0.f;
    }
    // ---- the ring
    const int* tab = p.r.table + (long)seq * p.r.width;
    const int shift = p.c.shift, values = (D >> 1) << shift, mask = (1 << shift) - 1;
    const int mine = max(ub - ua - warp + S::kWarps - 1, 0) / S::kWarps;       // units of this warp
    auto token0 = [&](int k) { return q.lo + (ua + warp + k * S::kWarps) * S::kUnit; };
    // Pages are looked up for 32 units at a time, a unit a lane, the pages of its tokens one after another.  -2: no key there that a row sees.
    int cur[PIECES], next[PIECES];
    auto look_up = [&](int k0) {
      const int k = k0 + lane, span = min(S::kUnit, 1 << shift), pieces = S::kUnit / span;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int tok = token0(k) + i * span;
        next[i] = i < pieces && k < mine && tok < q.hi && tok + span > q.key0 ? __ldg(tab + (tok >> shift)) : -2;
      }
    };
    auto issue = [&](int k) {
      if (k >= mine) return;
      if (!(k & 31)) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) cur[i] = next[i];
      }
      if ((k & 31) == 16) look_up((k & ~31) + 32);
      const uint32_t dst = ring + ahead * S::kStage, bar = bars + ahead * 8;
      const int page = __shfl_sync(0xffffffffu, cur[0], k & 31);
      if (1 << shift >= S::kUnit && (unsigned)page < (unsigned)p.c.pages) {
        // the usual case: all tokens of one page
        if (lane == 0) {
          const int slot = token0(k) & mask;
          const long off = ((long)page * p.c.kv + h) * p.c.block + slot * (D / 2), so = off - slot * (D / 2) + values + slot * (D / 16);
          tc::mbar_expect_tx(bar, S::kStage);
          if (1 << shift == S::kUnit) {
            tc::bulk_g2s(dst, p.c.k + off, S::kV, bar);
            tc::bulk_g2s(dst + S::kV, p.c.v + off, S::kV, bar);
          } else {
            tc::bulk_g2s(dst, p.c.k + off, S::kKeys, bar);
            tc::bulk_g2s(dst + S::kSK, p.c.k + so, S::kScales, bar);
            tc::bulk_g2s(dst + S::kV, p.c.v + off, S::kKeys, bar);
            tc::bulk_g2s(dst + S::kSV, p.c.v + so, S::kScales, bar);
          }
        }
      } else {
        const int span = min(S::kUnit, 1 << shift), pieces = S::kUnit / span;
        uint32_t there = 0;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          if (i >= pieces) continue;
          const int pg = __shfl_sync(0xffffffffu, cur[i], k & 31);
          if ((unsigned)pg < (unsigned)p.c.pages) {
            there |= 1u << i;
          } else if (pg != -2) {                         // (-2: masked below, whatever lies in the ring)
            if (lane == 0) tf_report(p.st, TF_BAD_INDEX, 183, seq, pg);
            uint8_t* z = ring_p + ahead * S::kStage + i * span * (D / 2);
            uint8_t* zs = ring_p + ahead * S::kStage + S::kSK + i * span * (D / 16);
            for (int o = lane * 16; o < span * (D / 2); o += 512) {
              *reinterpret_cast<uint4*>(z + o) = make_uint4(0u, 0u, 0u, 0u);
              *reinterpret_cast<uint4*>(z + S::kV + o) = make_uint4(0u, 0u, 0u, 0u);
            }
            if (lane < span * (D / 16) / 16) {
              *reinterpret_cast<uint4*>(zs + lane * 16) = make_uint4(0u, 0u, 0u, 0u);
              *reinterpret_cast<uint4*>(zs + S::kV + lane * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
          }
        }
        if (lane == 0) tc::mbar_expect_tx(bar, __popc(there) * (S::kStage / pieces));
        __syncwarp();
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const int pg = __shfl_sync(0xffffffffu, cur[i], k & 31);
          if (!(there >> i & 1) || lane) continue;
          const int sl = (token0(k) + i * span) & mask, at = i * span * (D / 2), sat = i * span * (D / 16);
          const long base = ((long)pg * p.c.kv + h) * p.c.block, off = base + sl * (D / 2), so = base + values + sl * (D / 16);
          tc::bulk_g2s(dst + at, p.c.k + off, span * (D / 2), bar);
          tc::bulk_g2s(dst + S::kSK + sat, p.c.k + so, span * (D / 16), bar);
          tc::bulk_g2s(dst + S::kV + at, p.c.v + off, span * (D / 2), bar);
          tc::bulk_g2s(dst + S::kSV + sat, p.c.v + so, span * (D / 16), bar);
        }
      }
      if (++ahead == S::kStages) ahead = 0;
    };
    if (lane == 0) tc::fence_proxy_async();              // (the ring held the joined results of the item before)
    look_up(0);
#pragma unroll 1
    for (int k = 0; k < S::kStages - 1; ++k) issue(k);
    for (int k = 0; k < mine; ++k) {
      // stage k - 1 is read by all lanes: it is filled again
      __syncwarp();
      issue(k + S::kStages - 1);
      if (ok) ok = tc::mbar_wait(bars + stage * 8, phase, abort_flag);
      __syncwarp();
      const uint8_t* st = ring_p + stage * S::kStage;
      if (++stage == S::kStages) {
        stage = 0;
        phase ^= 1;
      }
#pragma unroll 1
      for (int own = 0; own < S::kUnit; own += S::kOwn) {
        const int tok = token0(k) + own;
        const bool inside = tok >= in_lo && tok + S::kOwn <= in_hi;
        // ---- S^T
        float s[TI][NT][4];
#pragma unroll
        for (int i = 0; i < TI; ++i) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[i][nt][c] = 0.f;
          uint32_t ka[2][KW], sc[2][2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = own + i * 16 + e * 8 + g;
            if (D == 128) {
              const uint4 v = *reinterpret_cast<const uint4*>(st + row * 64 + t * 16);
              ka[e][0] = v.x; ka[e][1] = v.y; ka[e][KW - 2] = v.z; ka[e][KW - 1] = v.w;
              const uint32_t two_s = e4m3x2(*reinterpret_cast<const uint16_t*>(st + S::kSK + row * 8 + t * 2));
              sc[e][0] = __byte_perm(two_s, 0, 0x1010);
              sc[e][1] = __byte_perm(two_s, 0, 0x3232);
            } else {
              const uint2 v = *reinterpret_cast<const uint2*>(st + row * 32 + t * 8);
              ka[e][0] = v.x; ka[e][KW - 1] = v.y;
              const uint32_t one_s = e4m3x2(st[S::kSK + row * 4 + t]);
              sc[e][0] = sc[e][1] = __byte_perm(one_s, 0, 0x1010);
            }
          }
#pragma unroll
          for (int w = 0; w < KW; ++w) {
            uint32_t a0[4], a1[4];
            fp4::e2m1x8_to_h2x4(ka[0][w], a0);
            fp4::e2m1x8_to_h2x4(ka[1][w], a1);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              a0[e] = fp4::hmul2(a0[e], sc[0][w / 2]);
              a1[e] = fp4::hmul2(a1[e], sc[1][w / 2]);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t a[4] = {a0[2 * e], a1[2 * e], a0[2 * e + 1], a1[2 * e + 1]};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                if (NT == 1) {
                  mma_f16_16816(s[i][nt], a, qf[NT > 1 ? 0 : 2 * w + e]);
                } else {
                  const uint2 b2 = sq[((2 * w + e) * NT + nt) * 32 + lane];
                  const uint32_t b[2] = {b2.x, b2.y};
                  mma_f16_16816(s[i][nt], a, b);
                }
              }
            }
          }
        }
        // ---- softmax over the tokens (rows g and g + 8 of every tile), columns 2t and 2t + 1
        bool more = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float f = fac[nt][c];
#pragma unroll
            for (int i = 0; i < TI; ++i) {
              s[i][nt][c] *= f;
              s[i][nt][c + 2] *= f;
            }
            if (!inside) {
              const int2 r = range[nt * 8 + 2 * t + c];
#pragma unroll
              for (int i = 0; i < TI; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int key = tok + i * 16 + e * 8 + g;
                  if (key < r.x || key >= r.y) s[i][nt][c + 2 * e] = -INFINITY;
                }
            }
            const float top = m[nt][c] + 8.f;
            float x = fmaxf(s[0][nt][c], s[0][nt][c + 2]);
#pragma unroll
            for (int i = 1; i < TI; ++i) x = fmaxf(x, fmaxf(s[i][nt][c], s[i][nt][c + 2]));
            more |= x > top;
          }
        }
        if (__any_sync(0xffffffffu, more)) {
          // the maximum moves (rare behind the first tiles)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float x = fmaxf(s[0][nt][c], s[0][nt][c + 2]);
#pragma unroll
              for (int i = 1; i < TI; ++i) x = fmaxf(x, fmaxf(s[i][nt][c], s[i][nt][c + 2]));
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
              const float nm = fmaxf(m[nt][c], x), f = ex2(m[nt][c] - nm);
              m[nt][c] = nm;
              l[nt][c] *= f;
#pragma unroll
              for (int j = 0; j < KS; ++j) {
                O[j][nt][c] *= f;
                O[j][nt][c + 2] *= f;
              }
            }
        }
        uint32_t pb[TI][NT][2];
#pragma unroll
        for (int i = 0; i < TI; ++i)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              s[i][nt][c] = ex2(s[i][nt][c] - m[nt][c]);
              s[i][nt][c + 2] = ex2(s[i][nt][c + 2] - m[nt][c]);
              l[nt][c] += s[i][nt][c] + s[i][nt][c + 2];
            }
            pb[i][nt][0] = trans8x8(pack<__half>(s[i][nt][0], s[i][nt][1]));
            pb[i][nt][1] = trans8x8(pack<__half>(s[i][nt][2], s[i][nt][3]));
          }
        // ---- O^T
#pragma unroll
        for (int i = 0; i < TI; ++i) {
          uint32_t va[2][CH / 4], sv[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int pair = own / 2 + i * 8 + e * 4 + t;
            const uint8_t* src = st + S::kV + pair * D + g * CH;
            if (D == 128) {
              const uint4 v = *reinterpret_cast<const uint4*>(src);
              va[e][0] = v.x; va[e][1] = v.y; va[e][CH / 4 - 2] = v.z; va[e][CH / 4 - 1] = v.w;
            } else {
              const uint2 v = *reinterpret_cast<const uint2*>(src);
              va[e][0] = v.x; va[e][CH / 4 - 1] = v.y;
            }
            sv[e] = e4m3x2(*reinterpret_cast<const uint16_t*>(st + S::kSV + pair * (D / 8) + (g * CH / 16) * 2));
            if (!inside) {
              // keys that nobody sees may lie outside the sequence, where the page holds anything: zero times NaN
              const int key = tok - own + 2 * pair;
              if (key >= q.hi || key < q.key0) sv[e] &= 0xffff0000u;
              if (key + 1 >= q.hi || key + 1 < q.key0) sv[e] &= 0x0000ffffu;
            }
          }
#pragma unroll
          for (int w = 0; w < CH / 4; ++w) {
            uint32_t a0[4], a1[4];
            fp4::e2m1x8_to_h2x4(va[0][w], a0);
            fp4::e2m1x8_to_h2x4(va[1][w], a1);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              a0[e] = fp4::hmul2(a0[e], sv[0]);
              a1[e] = fp4::hmul2(a1[e], sv[1]);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t a[4] = {a0[2 * e], a0[2 * e + 1], a1[2 * e], a1[2 * e + 1]};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_f16_16816(O[2 * w + e][nt], a, pb[i][nt]);
            }
          }
        }
      }
    }
    // ---- the warps' results together
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], o);
    __syncthreads();
    float* jo = reinterpret_cast<float*>(smem);
    float2* jm = reinterpret_cast<float2*>(smem + S::kWarps * RB * S::kRowF * 4);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = nt * 8 + 2 * t + c;
        if (g == 0) jm[warp * RB + r] = make_float2(m[nt][c], l[nt][c]);
        float* dst = jo + (warp * RB + r) * S::kRowF + g * CH;
        // (a thread's pieces in an order of its own: neighbours in g lie 16 words apart)
#pragma unroll
        for (int x = 0; x < CH / 4; ++x)
          *reinterpret_cast<float4*>(dst + 4 * x) = make_float4(O[2 * x][nt][c], O[2 * x][nt][c + 2], O[2 * x + 1][nt][c], O[2 * x + 1][nt][c + 2]);
      }
    __syncthreads();
    const bool complete = ua == 0 && ub == q.units;
    const long slot = 2 * (long)blockIdx.x + (u > u_begin ? 1 : 0);
    for (int x = threadIdx.x; x < RB * D / 4; x += S::kWarps * 32) {
      const int r = x / (D / 4), c = x % (D / 4) * 4;
      float M = kNone;
#pragma unroll
      for (int w = 0; w < S::kWarps; ++w) M = fmaxf(M, jm[w * RB + r].x);
      float L = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < S::kWarps; ++w) {
        const float2 ml = jm[w * RB + r];
        const float f = ex2(ml.x - M);
        const float4 v = *reinterpret_cast<const float4*>(jo + (w * RB + r) * S::kRowF + c);
        L = fmaf(ml.y, f, L);
        o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y); o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w);
      }
      if (complete) {
        finish4<T>(p, q, h, blk * RB + r, c, M, L, o);
      } else {
        float* dst = p.work + (slot * RB + r) * (D + 4);
        *reinterpret_cast<float4*>(dst + c) = o;
        if (c == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(M, L);
      }
    }
    __syncthreads();                                     // shared memory is used again
    u += ub - ua;
    if (p.whole) break;
  }
  if (*abort_flag) {
    const long long t0 = clock64();
    while (clock64() - t0 < 400000) {}                   // copies in flight land before the shared memory goes back
    if (threadIdx.x == 0) tf_report(p.st, TF_TIMEOUT, 183, blockIdx.x, 0);
  }
}

// Joins the partial results of the items that lay in more than one CTA's range, in the order of the ranges.  A CTA takes some rows of one item;
// `lanes` groups of threads share a row's parts, a thread four channels.  Few items: CTA x looks at item x.  Many: at the one that begins in range
// x and ends behind it, of which there is one at most (256 sequences of 600 tokens x 2 heads, attention and this: by items 140 us, so 54).
template <int D, int NT, typename T>
__global__ void __launch_bounds__(256) paged_merge_kernel(const AttnParams p, int ctas, int by_item, int lanes) {
  using S = Shape<D, NT>;
  constexpr int RB = S::RB, PG = 256 / (D / 4);
  __shared__ float4 so[PG][D / 4];
  __shared__ float2 sm[PG];
  tf_pdl_sync();
  int seq;
  long before, total, a, item;
  locate<S, true>(p, 0x7fffffffffffffffl, &seq, &total);
  const long quota = max((total + ctas - 1) / ctas, (long)2 * S::kWarps);
  if (by_item) {
    if (!locate<S, false>(p, blockIdx.x, &seq, &before)) return;
    item = blockIdx.x - before;
    // units before the sequence: what locate would give for a unit of it
    a = 0;
    const int lane = threadIdx.x & 31;
    for (int s0 = 0; s0 < seq; s0 += 32) {
      long w = 0;
      if (s0 + lane < seq) {
        const Seq x = seq_of<S>(p, s0 + lane);
        w = (long)x.blocks * p.c.kv * x.units;
      }
      a += __shfl_sync(0xffffffffu, warp_scan(w), 31);
    }
  } else {
    const long last = (blockIdx.x + 1) * quota - 1;
    if (last + 1 >= total || !locate<S, true>(p, last, &seq, &a)) return;
    item = -1;
  }
  const Seq q = seq_of<S>(p, seq);
  if (item < 0) item = ((blockIdx.x + 1) * quota - 1 - a) / q.units;
  a += item * q.units;
  const long c0 = a / quota, c1 = (a + q.units - 1) / quota;
  if (c0 == c1 || (!by_item && c0 != blockIdx.x)) return;        // done where it was computed, or begun in an earlier range
  const int h = (int)(item % p.c.kv), blk = (int)(item / p.c.kv);
  const int x = threadIdx.x % (D / 4), pg = threadIdx.x / (D / 4), r = blockIdx.y * (PG / lanes) + pg / lanes, part = pg % lanes;
  float M = kNone, L = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  // eight parts at a time: their loads are one latency, and their sums do not wait for each other's maxima
  if (blk * RB + r < q.n * p.group) {
    for (long c = c0 + part; c <= c1; c += 8 * lanes) {
      float4 v[8];
      float2 ml[8];
      float nm = M;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const long n = c + i * lanes;
        v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        ml[i] = make_float2(kNone, 0.f);
        if (n <= c1) {
          const float* src = p.work + ((2 * n + (a > n * quota ? 1 : 0)) * RB + r) * (D + 4);
          v[i] = *reinterpret_cast<const float4*>(src + 4 * x);
          ml[i] = *reinterpret_cast<const float2*>(src + D);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) nm = fmaxf(nm, ml[i].x);
      const float f0 = ex2(M - nm);
      M = nm;
      L *= f0;
      o.x *= f0; o.y *= f0; o.z *= f0; o.w *= f0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = ex2(ml[i].x - nm);
        L = fmaf(ml[i].y, f, L);
        o.x = fmaf(v[i].x, f, o.x); o.y = fmaf(v[i].y, f, o.y); o.z = fmaf(v[i].z, f, o.z); o.w = fmaf(v[i].w, f, o.w);
      }
    }
  }
  so[pg][x] = o;
  if (x == 0) sm[pg] = make_float2(M, L);
  __syncthreads();
  if (part) return;
  for (int i = 1; i < lanes; ++i) {
    const float2 ml = sm[pg + i];
    const float4 v = so[pg + i][x];
    const float nm = fmaxf(M, ml.x), f0 = ex2(M - nm), f1 = ex2(ml.x - nm);
    M = nm;
    L = L * f0 + ml.y * f1;
    o.x = o.x * f0 + v.x * f1; o.y = o.y * f0 + v.y * f1; o.z = o.z * f0 + v.z * f1; o.w = o.w * f0 + v.w * f1;
  }
  finish4<T>(p, q, h, blk * RB + r, 4 * x, M, L, o);
}

int g_attn_sms = 0;

template <int D, int NT, typename T>
int launch_attn(AttnParams p, int ctas, long items, cudaStream_t st) {
  using S = Shape<D, NT>;
  static unsigned long long limit_set = 0;
  if (tf_smem_limit((const void*)paged_attn_kernel<D, NT, T>, S::kBytes, &limit_set) != cudaSuccess) return -2;
  tf_launch(paged_attn_kernel<D, NT, T>, dim3((unsigned)(p.whole ? items : ctas)), dim3(Shape<D, NT>::kWarps * 32), S::kBytes, st, p);
  if (!p.whole) {
    // a group of threads takes about eight parts of a row, and groups that this leaves have rows of their own
    constexpr int groups = 256 / (D / 4), most = groups < S::RB ? groups : S::RB;
    const long parts = ctas / ((long)p.r.seqs * p.c.kv) + 1;
    const bool by_item = items < ctas;
    int lanes = groups / most;
    while (lanes < groups && parts > 8 * lanes) lanes *= 2;
    tf_launch(paged_merge_kernel<D, NT, T>, dim3((unsigned)(by_item ? items : ctas), S::RB * lanes / groups), dim3(256), 0, st, p, ctas, (int)by_item, lanes);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

// Column tiles of a block by the rows that a sequence has on average (0: the many-row form, whose tiles have 128).  Four tiles against it,
// us: 32 rows over 131,072 tokens x 8 heads 105 and 136, 4 x 32,768 of 64 channels 73 and 114; 64 rows (two blocks) over 65,536 106 and
// 85, 32 x 2,048 119 and 86.
int tiles_of(int total, int seqs, int group) {
  const long rows = ((long)total + seqs - 1) / seqs * group;
  return rows <= 8 ? 1 : rows <= 16 ? 2 : rows <= 32 ? 4 : 0;
}
// An item is never cut (a CTA each) where its keys are few, or not many and there is an item for every CTA: 64 sequences of 1,000 tokens x 8
// heads of 128 cut 48 us, whole 35; 256 of 600 x 2: 54 and 31; 64 of 2,000 x 8: 63 and 51.
bool whole_of(int seqs, int kv, long keys, int ctas) { return keys <= 512 || (keys <= 2048 && (long)seqs * kv >= ctas); }
int ctas_of(int nt, int D) { return g_attn_sms * (D * nt <= 256 ? 2 : 1); }
void sms() {
  if (g_attn_sms) return;
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  g_attn_sms = n;
}

}  // namespace

// Floats of workspace that tf_paged_attention needs for `total` rows of `seqs` sequences and tables of `keys` tokens.
TF_API long tf_paged_attention_workspace(int total, int seqs, int heads, int kv, int D, long keys) {
  if (total < 1 || seqs < 1 || heads < 1 || kv < 1 || heads % kv) return 0;
  sms();
  const int nt = tiles_of(total, seqs, heads / kv);
  if (!nt) return paged_tc_workspace(total, seqs, heads, kv, D, keys, g_attn_sms);
  const int ctas = ctas_of(nt, D);
  return whole_of(seqs, kv, keys, ctas) ? 0 : 2l * ctas * 8 * nt * (D + 4);
}

// q [total][heads][D] and out alike (kind 1 f16, 2 bf16; strides in elements, rows of heads 16-byte aligned), lse [total][heads]
// fp32 or null.  Row i of sequence s sees the keys max(first[s], pos - window + 1) .. pos of its pages, pos = lengths[s] -
// (cu[s + 1] - i); window 0: all, first null: 0.  A row without keys gives zeros and lse -inf (with a sink: the sink's).
// work: tf_paged_attention_workspace floats (keys = width * page) that no other launch in flight uses.
TF_API int tf_paged_attention(const void* q, long q_row, long q_head, int heads, int kind, void* out, long o_row, long o_head,
                              float* lse, const void* kc, const void* vc, int pages, int kv, int page, int D, const int* table,
                              int width, const int* lengths, const int* cu, int seqs, int total, float scale, int window,
                              const int* first, const float* sink, float* work, void* status, cudaStream_t st) {
  AttnCall a = {};
  if (!cache_ok(kc, vc, pages, kv, page, D, &a.c) || !rows_ok(cu, lengths, table, seqs, width, fp4::page_shift(page), total, &a.r)) return -1;
  if (!q || !out || heads < 1 || heads % kv || (kind != 1 && kind != 2) || window < 0) return -1;
  if (!(scale > 0.f) || scale > 1e30f) return -1;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(work)) & 15) ||
      ((q_row | q_head | o_row | o_head) & 7))
    return -1;
  const long keys = (long)width * page;
  if (!work && tf_paged_attention_workspace(total, seqs, heads, kv, D, keys)) return -1;
  sms();
  a.q = q; a.out = out; a.lse = lse;
  a.q_row = q_row; a.q_head = q_head; a.o_row = o_row; a.o_head = o_head;
  a.heads = heads; a.group = heads / kv; a.kind = kind; a.window = window;
  a.scale2 = scale * 1.4426950408889634f;
  a.first = first; a.sink = sink; a.work = work; a.st = (TfStatusWord*)status;
  const int nt = tiles_of(total, seqs, a.group);
  if (!nt) return paged_tc_attention(a, g_attn_sms, st);
  AttnParams p = {};
  static_cast<AttnCall&>(p) = a;
  const int rb = 8 * nt, ctas = ctas_of(nt, D);
  // items: row blocks of the sequences (each may end with a part of one) x kv heads
  const long items = ((long)total * p.group / rb + seqs) * kv;
  if (items > 0x7fffffffl) return -1;
  p.whole = whole_of(seqs, kv, keys, ctas);
#define TF_ATTN(DD, N) (kind == 1 ? launch_attn<DD, N, __half>(p, ctas, items, st) : launch_attn<DD, N, __nv_bfloat16>(p, ctas, items, st))
  if (D == 128) return nt == 1 ? TF_ATTN(128, 1) : nt == 2 ? TF_ATTN(128, 2) : TF_ATTN(128, 4);
  return nt == 1 ? TF_ATTN(64, 1) : nt == 2 ? TF_ATTN(64, 2) : TF_ATTN(64, 4);
#undef TF_ATTN
}
