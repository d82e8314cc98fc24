// Paged KV cache held in 4 bits (e2m1 values, one e4m3 scale per 16: the arithmetic of the compressed KV rows), and what
// writes and reads it back; the attention over it is paged_attn.cu (few rows a sequence) and paged_tc.cu (many).
//
//   key   of token t: kv4(R(pos) k)      R: rotation of the last `rope` channels of every head, in pairs
//   value of token t: kv4(v)             kv4: s = e4m3(max(amax / 6, 2^-6)) per 16, e2m1(x / s)
//   query of token t: R(pos) q           rounded to the query's own type
//
// The rotation of a key is computed in 64 bits and rounded ONCE, to the 4-bit grid: the product of a 16-bit number and
// an fp32 table entry is exact there, so a key next to a border of the grid falls on the side that the formula says.  The
// query's rotation, which is rounded to 16 bits, is computed in fp32.
//
// Bound by HBM.  A thread takes 16 channels of one head (one block of the format): 32 bytes of the projection's row in,
// 8 bytes and a scale out (keys), 32 bytes out (queries); of a value, the two tokens that share its bytes.  Where only one
// token of such a pair is new, the other's nibbles are read and kept: no other thread touches that pair.
#include "divide.h"
#include "paged.cuh"

namespace {

using namespace paged;

struct AppendParams {
  Rows r;
  Cache c;
  const void *q, *k, *v;
  void* q_out;
  long q_row, q_head, k_row, k_head, v_row, v_head;     // strides in elements
  int heads;                                             // query heads (0: no queries)
  const float* rope;                                     // [positions][rope]: cosines, then sines
  int positions, rope_dim, interleaved;
  TfStatusWord* st;
};

// 16 channels of a row as they lie in memory
struct Raw {
  uint4 a, b;
};
template <typename T>
__device__ __forceinline__ Raw raw16(const T* p) {
  const uint4* q = reinterpret_cast<const uint4*>(p);
  return {__ldcs(q), __ldcs(q + 1)};
}
template <typename T>
__device__ __forceinline__ void unpack16(const Raw& r, float x[16]) {
  const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = two<T>(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
// 16 channels from channel j0 of the rotated part on (own: their values, other: those of the 16 that they pair with where pairs
// are halves apart), rotated by a row of the table; F: the type that the rotation is computed in
template <typename F, typename T>
__device__ __forceinline__ void rotate16(const Raw& own, const Raw& other, int j0, int rope, int inter, const float* tab, F y[16]) {
  const int half = rope >> 1;
  float x[16];
  unpack16<T>(own, x);
  if (inter) {
    float cs[8], sn[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      *reinterpret_cast<float4*>(cs + 4 * i) = __ldg(reinterpret_cast<const float4*>(tab + (j0 >> 1)) + i);
      *reinterpret_cast<float4*>(sn + 4 * i) = __ldg(reinterpret_cast<const float4*>(tab + half + (j0 >> 1)) + i);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const F a = x[2 * i], b = x[2 * i + 1], c = cs[i], s = sn[i];
      y[2 * i] = fma(a, c, -(b * s));
      y[2 * i + 1] = fma(a, s, b * c);
    }
  } else {
    const bool low = j0 < half;
    const int j = low ? j0 : j0 - half;
    float o[16];
    unpack16<T>(other, o);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 cs = __ldg(reinterpret_cast<const float4*>(tab + j) + i), sn = __ldg(reinterpret_cast<const float4*>(tab + half + j) + i);
      const float c4[4] = {cs.x, cs.y, cs.z, cs.w}, s4[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const F a = x[4 * i + e], b = o[4 * i + e], c = c4[e], s = low ? -s4[e] : s4[e];
        y[4 * i + e] = fma(a, c, b * s);
      }
    }
  }
}

// NaN is stored as zero and infinity as the largest value: the cache never holds a number that a masked key could poison
__device__ __forceinline__ void tame(float x[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float a = fabsf(x[i]);
    if (!(a <= 3.4028235e38f)) x[i] = a != a ? 0.f : copysignf(3.4028235e38f, x[i]);
  }
}
// largest magnitude of 16 packed values; NaN where one is
template <typename T>
__device__ __forceinline__ float amax16(const Raw& r);
template <>
__device__ __forceinline__ float amax16<__half>(const Raw& r) {
  const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
  __half2 m = __habs2(*reinterpret_cast<const __half2*>(&w[0]));
#pragma unroll
  for (int i = 1; i < 8; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __half2*>(&w[i])));
  return __half2float(__hmax_nan(__low2half(m), __high2half(m)));
}
template <>
__device__ __forceinline__ float amax16<__nv_bfloat16>(const Raw& r) {
  const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
  __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[0]));
#pragma unroll
  for (int i = 1; i < 8; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[i])));
  return __bfloat162float(__hmax_nan(__low2bfloat16(m), __high2bfloat16(m)));
}
// 16 values as they came -> their quotients by the block's scale; true where one was not finite
template <typename T>
__device__ __forceinline__ bool block16(const Raw& r, float y[16], uint8_t* sc) {
  float am = amax16<T>(r);
  unpack16<T>(r, y);
  const bool wild = !(am <= 3.4028235e38f);
  if (wild) {
    tame(y);
    am = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) am = fmaxf(am, fabsf(y[i]));
  }
  *sc = fp4::kv4_scale(am);
  const fp4::Recip rc = fp4::recip(e4m3_to_float(*sc));
#pragma unroll
  for (int i = 0; i < 16; ++i) y[i] = fp4::over(y[i], rc);
  return wild;
}

// Where a row goes.  The first warp of a CTA looks its rows up together, one a lane: the chain of loads (offsets and lengths, page) is
// paid once.
constexpr int kRowsMax = 32;
constexpr int kMostHeads = 1024;           // of a row (kMostHeads * 8 blocks of 16 channels: what Divide::small counts)
struct Spot {
  int page, slot, pos;                     // page -1: not stored; pos: row of the angles (0 where it has none)
  int flags;                               // 1: this row stores its pair of values, 2: the even token is new, 4: the odd one is,
                                           // 8: row of a sequence, 16: its position has angles
};
__device__ __forceinline__ Spot spot_at(const Rows& r, const Cache& c, int row, int seq, int first, int end, int length, int positions, bool angles,
                                        TfStatusWord* st) {
  Spot s = {-1, 0, 0, 8};
  const int pos = length - end + row;
  if (pos < 0 || (pos >> c.shift) >= r.width || (angles && pos >= positions)) {
    tf_report(st, TF_BAD_INDEX, 180, row, pos);
    return s;
  }
  s.flags |= 16;
  s.pos = pos;
  s.slot = pos & ((1 << c.shift) - 1);
  const int page = __ldg(r.table + (long)seq * r.width + (pos >> c.shift));
  if (page < 0 || page >= c.pages) {
    tf_report(st, TF_BAD_INDEX, 181, row, page);
    return s;
  }
  s.page = page;
  if (pos & 1) {
    s.flags |= 4 | (row == max(first, 0) ? 1 : 0);       // its pair is stored by the even token's row unless that one is not new
  } else {
    s.flags |= 1 | 2 | (row + 1 < end && row + 1 < r.total && !(angles && pos + 1 >= positions) ? 4 : 0);
  }
  return s;
}
// rows row0 .. row0 + n, n <= 32; all lanes of one warp.  Offsets are taken as they are (a range is clipped to the batch); who looks the first rows up
// reports ranges that leave the batch or run backwards.
__device__ __forceinline__ void look_up(const Rows& r, const Cache& c, int row0, int n, int positions, bool angles, TfStatusWord* st, Spot* spots) {
  const int lane = threadIdx.x & 31, row = row0 + lane;
  int seq = 0, first = 0, end = 0, length = 0;
  if (!r.cu) {
    seq = first = row;
    end = row + 1;
    if (row < r.seqs) length = __ldg(r.lengths + row);
  } else if (r.seqs <= 32) {
    int b = 0, e = 0x7fffffff, l = 0;
    if (lane < r.seqs) {
      b = __ldg(r.cu + lane);
      e = __ldg(r.cu + lane + 1);
      l = __ldg(r.lengths + lane);
    }
    if (st && !row0 && lane < r.seqs && (b < 0 || e < b || e > r.total)) tf_report(st, TF_BAD_INDEX, 182, lane, e);
    for (int i = 0; i < r.seqs; ++i) seq += __shfl_sync(0xffffffffu, e, i) <= row;
    first = __shfl_sync(0xffffffffu, b, seq & 31);
    end = __shfl_sync(0xffffffffu, e, seq & 31);
    length = __shfl_sync(0xffffffffu, l, seq & 31);
  } else {
    if (st && !row0) {
#pragma unroll 4
      for (int s = lane; s < r.seqs; s += 32) {
        const int b = __ldg(r.cu + s), e = __ldg(r.cu + s + 1);
        if (b < 0 || e < b || e > r.total) tf_report(st, TF_BAD_INDEX, 182, s, e);
      }
    }
    int hi = r.seqs;                       // the sequence whose rows end behind this one
    while (seq < hi) {
      const int mid = (seq + hi) >> 1;
      if (__ldg(r.cu + mid + 1) > row) hi = mid;
      else seq = mid + 1;
    }
    if (seq < r.seqs) {
      first = __ldg(r.cu + seq);
      end = __ldg(r.cu + seq + 1);
      length = __ldg(r.lengths + seq);
    }
  }
  if (lane < n) {
    if (seq < r.seqs && row >= first) spots[lane] = spot_at(r, c, row, seq, first, end, length, positions, angles, st);
    else spots[lane] = {-1, 0, 0, 0};
  }
}

// What a CTA does with its rows: one of five lists of (row, head, block of 16 channels).  Blocks that are rotated and blocks that
// are not are lists of their own, so that no warp does both; the entries of the values are pairs of tokens.
enum { kKeysTurned, kKeysPlain, kValues, kQueriesTurned, kQueriesPlain, kLists };
struct Lists {
  int end[kLists];                         // CTAs up to the end of each list
};

template <typename T, int LIST>
__device__ __forceinline__ void run_list(const AppendParams& p, Spot* spots, int* lead, int group, bool report, int rows, int start, int step) {
  constexpr bool kQuery = LIST >= kQueriesTurned, kTurn = LIST == kKeysTurned || LIST == kQueriesTurned, kValue = LIST == kValues;
  const int D = p.c.D, nb = D >> 4, turned = p.rope_dim >> 4, plain = nb - turned, row0 = group * rows, n = min(rows, p.r.total - row0);
  const int mb = kValue ? nb : kTurn ? turned : plain, heads = kQuery ? p.heads : p.c.kv, values = (D >> 1) << p.c.shift;
  const Divide by_row(heads * mb), by_head(mb);
  const long row_step = kQuery ? p.q_row : kValue ? p.v_row : p.k_row, head_step = kQuery ? p.q_head : kValue ? p.v_head : p.k_head;
  const T* base = (const T*)(kQuery ? p.q : kValue ? p.v : p.k) + row_step * row0 + (kTurn ? plain * 16 : 0);
  const int mate = p.rope_dim >> 1;
  int i = start, k, h, b, j;
  Raw x0 = {}, x1 = {};
  auto load = [&](int row) {
    const T* src = base + row * row_step + h * head_step + b * 16;
    x0 = raw16(src);
    if (kTurn && !p.interleaved) x1 = raw16(src + (b < turned >> 1 ? mate : -mate));
  };
  k = by_row.small(i, &j);
  h = by_head.small(j, &b);
  // the first entry's numbers are on their way while the rows' places are looked up
  if (!kValue && k < n) load(k);
  if (threadIdx.x < 32) {
    look_up(p.r, p.c, row0, n, p.positions, p.rope_dim != 0, report ? p.st : nullptr, spots);
    __syncwarp();
    if (kValue) {
      // rows that store a pair
      const bool l = threadIdx.x < n && (spots[threadIdx.x].flags & 1) && spots[threadIdx.x].page >= 0;
      const unsigned all = __ballot_sync(0xffffffffu, l);
      if (l) lead[__popc(all & ((1u << threadIdx.x) - 1u))] = threadIdx.x;
      if (threadIdx.x == 0) lead[kRowsMax] = __popc(all);
    }
  }
  __syncthreads();
  const int count = kValue ? lead[kRowsMax] : n;
  for (; k < count;) {
    const int row = kValue ? lead[k] : k;
    const Spot s = spots[row];
    if (kValue) load(row);
    const Raw c0 = x0, c1 = x1;
    const int hh = h, bb = b;
    const T* at = base + row * row_step + h * head_step + b * 16;
    i += step;
    k = by_row.small(i, &j);
    h = by_head.small(j, &b);
    if (!kValue && k < n) load(k);         // the next entry's, while this one is rounded
    const float* tab = p.rope + (long)s.pos * p.rope_dim;
    if constexpr (kQuery) {
      if (!(s.flags & 8)) continue;
      uint4* dst = reinterpret_cast<uint4*>((T*)p.q_out + ((long)(row0 + row) * p.heads + hh) * D + (bb + (kTurn ? plain : 0)) * 16);
      Raw o = c0;
      if (kTurn && (s.flags & 16)) {
        float y[16];
        rotate16<float, T>(c0, c1, bb * 16, p.rope_dim, p.interleaved, tab, y);
        uint32_t w[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) w[c] = pack<T>(y[2 * c], y[2 * c + 1]);
        o = {make_uint4(w[0], w[1], w[2], w[3]), make_uint4(w[4], w[5], w[6], w[7])};
      }
      dst[0] = o.a;
      dst[1] = o.b;
    } else if constexpr (!kValue) {
      if (s.page < 0) continue;
      float z[16];
      uint8_t sc;
      bool wild = false;
      if constexpr (kTurn) {
        double y[16];
        rotate16<double, T>(c0, c1, bb * 16, p.rope_dim, p.interleaved, tab, y);
        float am = 0.f;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          z[c] = fp4::sticky(y[c]);
          am = fmaxf(am, fabsf(z[c]));
          wild |= !(fabsf(z[c]) <= 3.4028235e38f);
        }
        if (wild) {
          tame(z);
          am = 0.f;
#pragma unroll
          for (int c = 0; c < 16; ++c) am = fmaxf(am, fabsf(z[c]));
        }
        sc = fp4::kv4_scale(am);
        const float f = e4m3_to_float(sc), r = __frcp_rn(f);
#pragma unroll
        for (int c = 0; c < 16; ++c) z[c] = fp4::over_sticky(z[c], f, r);
      } else {
        wild = block16<T>(c0, z, &sc);
      }
      if (wild) tf_report(p.st, TF_NONFINITE, 180, row0 + row, hh);
      uint32_t w[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float lo[4] = {z[8 * c], z[8 * c + 2], z[8 * c + 4], z[8 * c + 6]}, hi[4] = {z[8 * c + 1], z[8 * c + 3], z[8 * c + 5], z[8 * c + 7]};
        w[c] = fp4::e2m1x8(lo, hi);
      }
      const int blk = bb + (kTurn ? plain : 0);
      uint8_t* out = p.c.k + ((long)s.page * p.c.kv + hh) * p.c.block;
      *reinterpret_cast<uint2*>(out + s.slot * (D >> 1) + blk * 8) = make_uint2(w[0], w[1]);
      out[values + s.slot * nb + blk] = sc;
    } else {
      const bool even = s.flags & 2, odd = s.flags & 4;
      Raw e0 = c0, e1 = {};
      if (even && odd) e1 = raw16(at + row_step);
      if (!even) {
        e1 = e0;
        e0 = {};
      }
      float z[16], z2[16];
      uint8_t sc, sc2;
      const bool wild0 = block16<T>(e0, z, &sc), wild1 = block16<T>(e1, z2, &sc2);     // (zeros where a token is not new)
      if (wild0 || wild1) tf_report(p.st, TF_NONFINITE, 180, row0 + row, hh);
      uint32_t w[4], both = sc | (uint32_t)sc2 << 8;
#pragma unroll
      for (int c = 0; c < 4; ++c) w[c] = fp4::e2m1x8(z + 4 * c, z2 + 4 * c);
      uint8_t* out = p.c.v + ((long)s.page * p.c.kv + hh) * p.c.block;
      uint4* dst = reinterpret_cast<uint4*>(out + (s.slot >> 1) * D + bb * 16);
      uint16_t* sd = reinterpret_cast<uint16_t*>(out + values + (s.slot >> 1) * (2 * nb) + 2 * bb);
      if (!even || !odd) {
        // the other token's numbers stay
        const uint32_t keep = even ? 0xf0f0f0f0u : 0x0f0f0f0fu, skeep = even ? 0xff00u : 0xffu;
        const uint4 old = *dst;
        w[0] = (w[0] & ~keep) | (old.x & keep);
        w[1] = (w[1] & ~keep) | (old.y & keep);
        w[2] = (w[2] & ~keep) | (old.z & keep);
        w[3] = (w[3] & ~keep) | (old.w & keep);
        both = (both & ~skeep) | (*sd & skeep);
      }
      *dst = make_uint4(w[0], w[1], w[2], w[3]);
      *sd = (uint16_t)both;
    }
  }
}

// CTA `y` of those that share the rows of `group`; QUERIES false: keys and values only
template <typename T, bool QUERIES>
__device__ __forceinline__ void run_lists(const AppendParams& p, Spot* spots, int* lead, int group, int y, int rows, const Lists& lists) {
  int list = 0;
  while (list < kLists - 1 && y >= lists.end[list]) ++list;
  const int before = list ? lists.end[list - 1] : 0, start = (y - before) * 256 + threadIdx.x, step = 256 * (lists.end[list] - before);
  if (list == kKeysTurned) run_list<T, kKeysTurned>(p, spots, lead, group, !y, rows, start, step);
  else if (list == kKeysPlain) run_list<T, kKeysPlain>(p, spots, lead, group, !y, rows, start, step);
  else if (list == kValues) run_list<T, kValues>(p, spots, lead, group, !y, rows, start, step);
  else if (QUERIES && list == kQueriesTurned) run_list<T, kQueriesTurned>(p, spots, lead, group, !y, rows, start, step);
  else if (QUERIES) run_list<T, kQueriesPlain>(p, spots, lead, group, !y, rows, start, step);
}

// Queries of many rows.  A warp takes a row, eight channels (16 bytes) a lane: 256 channels a step are whole heads, so a lane is at the
// same place of every head and keeps its four cosines and sines for the row.  Pairs that are halves apart meet by a shuffle.
// Bound by HBM: 16,384 rows of 64 x 128 (537 MB in and out) 91 us alone.  Eight steps are in flight: beside the CTAs for keys and values
// (paged_append_many_kernel) four left the memory idle (129 us in all, 123 so).
constexpr int kSteps = 8;
constexpr int kQueryRows = 16;             // of a CTA of eight warps
template <typename T>
__device__ __forceinline__ void turn_queries(const AppendParams& p, Spot* spots, int group) {
  const int D = p.c.D, row0 = group * kQueryRows, n = min(kQueryRows, p.r.total - row0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < 32) look_up(p.r, p.c, row0, n, p.positions, p.rope_dim != 0, nullptr, spots);
  __syncthreads();
  const int c = lane * 8 & (D - 1), per = 256 / D;       // first channel of the lane, heads of a step
  const int j = c - (D - p.rope_dim), half = p.rope_dim >> 1;
  const bool low = j < half;
  const int mate = j < 0 ? lane : low ? lane + (half >> 3) : lane - (half >> 3);
  for (int k = warp; k < n; k += 8) {
    const Spot s = spots[k];
    if (!(s.flags & 8)) continue;
    const bool turn = j >= 0 && (s.flags & 16);
    // of lanes whose pairs are halves apart: eight cosines and sines
    float cs[8], sn[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      cs[i] = 1.f;
      sn[i] = 0.f;
    }
    if (turn) {
      const float* tab = p.rope + (long)s.pos * p.rope_dim;
      if (p.interleaved) {
        *reinterpret_cast<float4*>(cs) = __ldg(reinterpret_cast<const float4*>(tab + (j >> 1)));
        *reinterpret_cast<float4*>(sn) = __ldg(reinterpret_cast<const float4*>(tab + half + (j >> 1)));
      } else {
        const float4* t = reinterpret_cast<const float4*>(tab + (low ? j : j - half));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          *reinterpret_cast<float4*>(cs + 4 * i) = __ldg(t + i);
          float4 v = __ldg(t + (half >> 2) + i);
          if (low) v = make_float4(-v.x, -v.y, -v.z, -v.w);
          *reinterpret_cast<float4*>(sn + 4 * i) = v;
        }
      }
    }
    const T* src = (const T*)p.q + (long)(row0 + k) * p.q_row + c;
    uint4* dst = reinterpret_cast<uint4*>((T*)p.q_out + (long)(row0 + k) * p.heads * D) + lane;
    const int h0 = lane * 8 / D;
    for (int h = 0; h < p.heads; h += kSteps * per) {
      uint4 x[kSteps];
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        const int head = h + u * per + h0;
        x[u] = make_uint4(0u, 0u, 0u, 0u);
        if (head < p.heads) x[u] = __ldcs(reinterpret_cast<const uint4*>(src + (long)head * p.q_head));
      }
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
        if (p.interleaved) {
          if (turn) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 f = two<T>(w[i]);
              w[i] = pack<T>(fmaf(f.x, cs[i], -(f.y * sn[i])), fmaf(f.x, sn[i], f.y * cs[i]));
            }
          }
        } else if (p.rope_dim) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = two<T>(w[i]), g = two<T>(__shfl_sync(0xffffffffu, w[i], mate));
            if (turn) w[i] = pack<T>(fmaf(f.x, cs[2 * i], g.x * sn[2 * i]), fmaf(f.y, cs[2 * i + 1], g.y * sn[2 * i + 1]));
          }
        }
        if (h + u * per + h0 < p.heads) dst[(h + u * per) * (D >> 3)] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

// Few rows: one launch of lists, a row a CTA (latency)
template <typename T>
__global__ void __launch_bounds__(256, 3) paged_append_kernel(const AppendParams p, int rows, Lists lists) {
  __shared__ Spot spots[kRowsMax];
  __shared__ int lead[kRowsMax + 1];
  tf_pdl_sync();
  run_lists<T, true>(p, spots, lead, blockIdx.x, blockIdx.y, rows, lists);
}
// Many rows: `query_ctas` CTAs for the queries are spread evenly among those for keys and values (whose rounding hides under the queries' bytes:
// 16,384 rows of 64 query and 8 kv heads in two launches 137 us, in one 123 - 126; keys and values alone are 51).
template <typename T>
__global__ void __launch_bounds__(256, 3) paged_append_many_kernel(const AppendParams p, int rows, Lists lists, int query_ctas) {
  __shared__ Spot spots[kRowsMax];
  __shared__ int lead[kRowsMax + 1];
  tf_pdl_sync();
  const long all = gridDim.x, b = blockIdx.x, q = b * query_ctas / all;
  if ((b + 1) * query_ctas / all > q) {
    turn_queries<T>(p, spots, (int)q);
  } else {
    const int a = (int)(b - q), ny = lists.end[kLists - 1];
    run_lists<T, false>(p, spots, lead, a / ny, a % ny, rows, lists);
  }
}

// Cached rows back as bf16 (a 4-bit value times its scale has six significant bits: exact).  One thread per 16 channels of a
// row's keys and values.
struct ReadParams {
  Rows r;
  Cache c;
  __nv_bfloat16 *k, *v;                    // [total][kv][D]
  TfStatusWord* st;
};
__global__ void __launch_bounds__(256) paged_read_kernel(const ReadParams p, int rows) {
  __shared__ Spot spots[kRowsMax];
  tf_pdl_sync();
  const int row0 = blockIdx.x * rows, D = p.c.D, nb = D >> 4, kvb = p.c.kv * nb;
  const int n = min(rows, p.r.total - row0);
  if (threadIdx.x < 32) look_up(p.r, p.c, row0, n, 0, false, blockIdx.y ? nullptr : p.st, spots);
  __syncthreads();
  const int values = (D >> 1) << p.c.shift;
  const Divide by_row(2 * kvb), by_head(nb);
  for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < 2 * n * kvb; i += gridDim.y * blockDim.x) {
    int y, b;
    const int x = by_row(i, &y), row = row0 + x;
    const bool val = y >= kvb;
    const int h = by_head(val ? y - kvb : y, &b);
    const int page = spots[x].page, slot = spots[x].slot;
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    float s = 0.f;
    if (page >= 0) {
      const uint8_t* base = (val ? p.c.v : p.c.k) + ((long)page * p.c.kv + h) * p.c.block;
      if (val) {
        const uint4 r = *reinterpret_cast<const uint4*>(base + (slot >> 1) * D + b * 16);
        const int sh = (slot & 1) * 4;
        const uint32_t a[4] = {r.x >> sh & 0x0f0f0f0fu, r.y >> sh & 0x0f0f0f0fu, r.z >> sh & 0x0f0f0f0fu, r.w >> sh & 0x0f0f0f0fu};
        // nibbles of four bytes -> the low half-word's four
#pragma unroll
        for (int c = 0; c < 4; ++c) w[c >> 1] |= ((a[c] | a[c] >> 4) & 0xffu | (a[c] >> 8 | a[c] >> 12) & 0xff00u) << 16 * (c & 1);
        s = e4m3_to_float(base[values + (slot >> 1) * (2 * nb) + 2 * b + (slot & 1)]);
      } else {
        const uint2 r = *reinterpret_cast<const uint2*>(base + slot * (D >> 1) + b * 8);
        w[0] = r.x;
        w[1] = r.y;
        s = e4m3_to_float(base[values + slot * nb + b]);
      }
    }
    uint32_t o[8];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint32_t hh[4];
      fp4::e2m1x8_to_h2x4(w[c], hh);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = two<__half>(hh[e]);
        o[4 * c + e] = pack<__nv_bfloat16>(f.x * s, f.y * s);
      }
    }
    uint4* dst = reinterpret_cast<uint4*>((val ? p.v : p.k) + ((long)row * p.c.kv + h) * D + b * 16);
    dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

constexpr int kManyRows = 512;
// Rows of a CTA: one where they are few (latency), else as many as leave four groups of rows an SM
int rows_of(int total) {
  const int n = total / (4 * 148);
  return n < 1 ? 1 : n > kRowsMax ? kRowsMax : n;
}
// CTAs that share the `blocks` 16-channel blocks of a CTA's rows
int parts_of(long blocks, int groups) {
  const long most = (blocks + 255) / 256, want = (4 * 148 + groups - 1) / groups;
  const long n = want < most ? want : most;
  return n < 1 ? 1 : (int)n;
}

}  // namespace

// Rotates keys and appends them and the values to the cache; with q also rotates the queries into q_out.
//   k, v [total][kv][D], q [total][heads][D]: kind 1 f16, 2 bf16; strides in elements, rows of heads 16-byte aligned
//   rope [positions][rope_dim] fp32, cosines then sines (null with rope_dim 0); rope_dim a multiple of 32, at most D
//   row i of sequence s (rows cu[s] .. cu[s + 1]) is token lengths[s] - (cu[s + 1] - i); rows behind cu[seqs] are left alone
// A row whose position, page or row of angles is out of range is not stored and is reported in `status`, as are offsets that leave 0 .. total
// or run backwards.
TF_API int tf_paged_append(const void* q, long q_row, long q_head, int heads, const void* k, long k_row, long k_head, const void* v,
                           long v_row, long v_head, int kind, void* q_out, void* kc, void* vc, int pages, int kv, int page, int D,
                           const int* table, int width, const int* lengths, const int* cu, int seqs, int total, const float* rope,
                           int positions, int rope_dim, int interleaved, void* status, cudaStream_t st) {
  AppendParams p = {};
  if (!cache_ok(kc, vc, pages, kv, page, D, &p.c) || !rows_ok(cu, lengths, table, seqs, width, fp4::page_shift(page), total, &p.r)) return -1;
  if (!k || !v || (heads && (!q || !q_out)) || heads < 0 || heads > kMostHeads || kv > kMostHeads || (kind != 1 && kind != 2)) return -1;
  if (rope_dim < 0 || rope_dim % 32 || rope_dim > D || (rope_dim && (!rope || positions < 1))) return -1;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                         (heads ? reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) : 0) |
                         (rope_dim ? reinterpret_cast<uintptr_t>(rope) : 0);
  if ((bits & 15) || ((q_row | q_head | k_row | k_head | v_row | v_head) & 7)) return -1;
  p.q = q; p.k = k; p.v = v; p.q_out = q_out;
  p.q_row = q_row; p.q_head = q_head; p.k_row = k_row; p.k_head = k_head; p.v_row = v_row; p.v_head = v_head;
  p.heads = heads; p.rope = rope; p.positions = positions; p.rope_dim = rope_dim; p.interleaved = interleaved;
  p.st = (TfStatusWord*)status;
  // Few rows: a row a CTA (latency).  Many: rows of which every list fills its CTAs, and CTAs for the queries between them.
  const bool few = total < kManyRows;
  const int rows = few ? 1 : rows_of(total), groups = (total + rows - 1) / rows, nb = D / 16, turned = rope_dim / 16;
  const int items[kLists] = {kv * turned, kv * (nb - turned), rows > 1 ? kv * nb / 2 : kv * nb, few ? heads * turned : 0, few ? heads * (nb - turned) : 0};
  Lists l;
  const int each = 256 * (rows >= 32 ? 4 : rows >= 16 ? 2 : 1);           // entries of a CTA
  for (int i = 0, at = 0; i < kLists; ++i) l.end[i] = at += (rows * items[i] + each - 1) / each;
  if (l.end[kLists - 1] > 65535) return -1;
  if (few) {
    const dim3 grid(groups, l.end[kLists - 1]);
    if (kind == 1) tf_launch(paged_append_kernel<__half>, grid, dim3(256), 0, st, p, rows, l);
    else tf_launch(paged_append_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, p, rows, l);
  } else {
    const int query_ctas = heads ? (total + kQueryRows - 1) / kQueryRows : 0;
    const long ctas = (long)groups * l.end[kLists - 1] + query_ctas;
    if (ctas > 0x7fffffffl) return -1;
    if (kind == 1) tf_launch(paged_append_many_kernel<__half>, dim3((unsigned)ctas), dim3(256), 0, st, p, rows, l, query_ctas);
    else tf_launch(paged_append_many_kernel<__nv_bfloat16>, dim3((unsigned)ctas), dim3(256), 0, st, p, rows, l, query_ctas);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

// Keys and values of the same rows out of the cache: k, v [total][kv][D] bf16 (a row that has none reads zero, one of no sequence too).
TF_API int tf_paged_read(void* k, void* v, const void* kc, const void* vc, int pages, int kv, int page, int D, const int* table,
                         int width, const int* lengths, const int* cu, int seqs, int total, void* status, cudaStream_t st) {
  ReadParams p = {};
  if (!cache_ok(kc, vc, pages, kv, page, D, &p.c) || !rows_ok(cu, lengths, table, seqs, width, fp4::page_shift(page), total, &p.r)) return -1;
  if (!k || !v || kv > kMostHeads || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15)) return -1;
  p.k = (__nv_bfloat16*)k;
  p.v = (__nv_bfloat16*)v;
  p.st = (TfStatusWord*)status;
  const int rows = rows_of(total), groups = (total + rows - 1) / rows;
  tf_launch(paged_read_kernel, dim3(groups, parts_of((long)rows * 2 * kv * (D / 16), groups)), dim3(256), 0, st, p, rows);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
