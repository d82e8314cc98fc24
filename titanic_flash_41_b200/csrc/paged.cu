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
#include "paged.cuh"

namespace {

using namespace paged;

template <typename T>
__device__ __forceinline__ void load16(const T* p, float x[16]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p), b = *reinterpret_cast<const uint4*>(p + 8);
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = two<T>(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

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

// the 16 channels at c0 of a head's row, rotated; F: the type that the rotation is computed in
template <typename F, typename T>
__device__ __forceinline__ void rotated16(const T* row, int c0, int D, int rope, int inter, const float* tab, F y[16]) {
  float x[16];
  load16(row + c0, x);
  const int j0 = c0 - (D - rope), half = rope >> 1;
  if (j0 < 0) {
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = x[i];
    return;
  }
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
    float o[16], cs[16], sn[16];
    load16(row + (low ? c0 + half : c0 - half), o);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      *reinterpret_cast<float4*>(cs + 4 * i) = __ldg(reinterpret_cast<const float4*>(tab + j) + i);
      *reinterpret_cast<float4*>(sn + 4 * i) = __ldg(reinterpret_cast<const float4*>(tab + half + j) + i);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const F a = x[i], b = o[i], c = cs[i], s = sn[i];
      y[i] = low ? fma(a, c, -(b * s)) : fma(a, c, b * s);
    }
  }
}

// NaN is stored as zero and infinity as the largest value: the cache never holds a number that a masked key could poison
__device__ __forceinline__ bool tame(float x[16]) {
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float a = fabsf(x[i]);
    if (!(a <= 3.4028235e38f)) {
      odd = true;
      x[i] = a != a ? 0.f : copysignf(3.4028235e38f, x[i]);
    }
  }
  return odd;
}

template <typename T>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendParams p) {
  tf_pdl_sync();
  const int row = blockIdx.x, D = p.c.D, nb = D >> 4, kvb = p.c.kv * nb, qb = p.heads * nb;
  Place at;
  if (!place_of(p.r, row, &at)) return;
  const int seq = at.seq, pos = at.pos;
  bool bad_pos = pos < 0 || (pos >> p.c.shift) >= p.r.width;
  if (p.rope_dim && pos >= p.positions) bad_pos = true;
  if (bad_pos && threadIdx.x == 0 && blockIdx.y == 0) tf_report(p.st, TF_BAD_INDEX, 180, row, pos);
  const float* tab = p.rope + (bad_pos || !p.rope_dim ? 0l : (long)pos * p.rope_dim);
  int page = bad_pos ? -1 : p.r.table[(long)seq * p.r.width + (pos >> p.c.shift)];
  if (!bad_pos && (page < 0 || page >= p.c.pages)) {
    if (threadIdx.x == 0 && blockIdx.y == 0) tf_report(p.st, TF_BAD_INDEX, 181, row, page);
    page = -1;
  }
  const int slot = pos & ((1 << p.c.shift) - 1), values = (D >> 1) << p.c.shift;
  // the row that writes a pair of values: its even token's, or its odd token's where the even one is not new
  const bool lead = !(pos & 1) || row == at.first, lone_odd = pos & 1;
  const bool second = lone_odd || (row + 1 < at.first + at.count && row + 1 < p.r.total);   // the pair's odd token is new
  for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < qb + 2 * kvb; i += gridDim.y * blockDim.x) {
    if (i < kvb) {
      // ---- keys
      if (page < 0) continue;
      const int h = i / nb, b = i - h * nb;
      double y[16];
      rotated16<double>((const T*)p.k + (long)row * p.k_row + h * p.k_head, b * 16, D, p.rope_dim, p.interleaved, tab, y);
      float x[16], z[16];
#pragma unroll
      for (int c = 0; c < 16; ++c) x[c] = fp4::sticky(y[c]);
      if (tame(x)) tf_report(p.st, TF_NONFINITE, 180, row, h);
      const uint8_t sc = fp4::kv4_scale(x, z);
      uint32_t w[2] = {0u, 0u};
#pragma unroll
      for (int c = 0; c < 8; ++c) w[c >> 2] |= fp4::f2_to_e2m1x2(z[2 * c], z[2 * c + 1]) << 8 * (c & 3);
      uint8_t* base = p.c.k + ((long)page * p.c.kv + h) * p.c.block;
      *reinterpret_cast<uint2*>(base + slot * (D >> 1) + b * 8) = make_uint2(w[0], w[1]);
      base[values + slot * nb + b] = sc;
    } else if (i < 2 * kvb) {
      // ---- values: both tokens of a pair
      if (page < 0 || !lead) continue;
      const int j = i - kvb, h = j / nb, b = j - h * nb;
      const T* src = (const T*)p.v + (long)row * p.v_row + h * p.v_head + b * 16;
      float x[16], z[16], z2[16];
      load16(src, x);
      bool odd = tame(x);
      uint32_t sc = fp4::kv4_scale(x, z), sc2 = 0;
      if (lone_odd) {
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          z2[c] = z[c];
          z[c] = 0.f;
        }
        sc2 = sc;
        sc = 0;
      } else if (second) {
        load16(src + p.v_row, x);
        odd |= tame(x);
        sc2 = fp4::kv4_scale(x, z2);
      } else {
#pragma unroll
        for (int c = 0; c < 16; ++c) z2[c] = 0.f;
      }
      if (odd) tf_report(p.st, TF_NONFINITE, 180, row, h);
      uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int c = 0; c < 16; ++c) w[c >> 2] |= fp4::f2_to_e2m1x2(z[c], z2[c]) << 8 * (c & 3);
      uint8_t* base = p.c.v + ((long)page * p.c.kv + h) * p.c.block;
      uint4* dst = reinterpret_cast<uint4*>(base + (slot >> 1) * D + b * 16);
      uint16_t* sd = reinterpret_cast<uint16_t*>(base + values + (slot >> 1) * (2 * nb) + 2 * b);
      uint32_t s = sc | sc2 << 8;
      if (lone_odd || !second) {
        const uint32_t keep = lone_odd ? 0x0f0f0f0fu : 0xf0f0f0f0u, skeep = lone_odd ? 0xffu : 0xff00u;
        const uint4 old = *dst;
        w[0] = (w[0] & ~keep) | (old.x & keep);
        w[1] = (w[1] & ~keep) | (old.y & keep);
        w[2] = (w[2] & ~keep) | (old.z & keep);
        w[3] = (w[3] & ~keep) | (old.w & keep);
        s = (s & ~skeep) | (*sd & skeep);
      }
      *dst = make_uint4(w[0], w[1], w[2], w[3]);
      *sd = (uint16_t)s;
    } else {
      // ---- queries
      const int j = i - 2 * kvb, h = j / nb, b = j - h * nb;
      float y[16];
      rotated16<float>((const T*)p.q + (long)row * p.q_row + h * p.q_head, b * 16, D, bad_pos ? 0 : p.rope_dim, p.interleaved, tab, y);
      uint32_t w[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) w[c] = pack<T>(y[2 * c], y[2 * c + 1]);
      uint4* dst = reinterpret_cast<uint4*>((T*)p.q_out + ((long)row * p.heads + h) * D + b * 16);
      dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
      dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
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
__global__ void __launch_bounds__(256) paged_read_kernel(const ReadParams p) {
  tf_pdl_sync();
  const int row = blockIdx.x, D = p.c.D, nb = D >> 4, kvb = p.c.kv * nb;
  Place at;
  if (!place_of(p.r, row, &at)) return;
  const int pos = at.pos;
  int page = -1;
  if (pos >= 0 && (pos >> p.c.shift) < p.r.width) page = p.r.table[(long)at.seq * p.r.width + (pos >> p.c.shift)];
  if (page < 0 || page >= p.c.pages) {
    if (threadIdx.x == 0 && blockIdx.y == 0) tf_report(p.st, TF_BAD_INDEX, 182, row, pos);
    page = -1;
  }
  const int slot = pos & ((1 << p.c.shift) - 1), values = (D >> 1) << p.c.shift;
  for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < 2 * kvb; i += gridDim.y * blockDim.x) {
    const bool val = i >= kvb;
    const int j = val ? i - kvb : i, h = j / nb, b = j - h * nb;
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

// CTAs that share a row's blocks: one wave of CTAs where the rows are few
int row_parts(int rows, int blocks) {
  const int most = (blocks + 255) / 256;
  const int want = (296 + rows - 1) / rows;
  return want < most ? want : most;
}

}  // namespace

// Rotates keys and appends them and the values to the cache; with q also rotates the queries into q_out.
//   k, v [total][kv][D], q [total][heads][D]: kind 1 f16, 2 bf16; strides in elements, rows of heads 16-byte aligned
//   rope [positions][rope_dim] fp32, cosines then sines (null with rope_dim 0); rope_dim a multiple of 32, at most D
//   row i of sequence s (rows cu[s] .. cu[s + 1]) is token lengths[s] - (cu[s + 1] - i); rows behind cu[seqs] are left alone
// A row whose position, page or table row is out of range is not stored and is reported in `status`.
TF_API int tf_paged_append(const void* q, long q_row, long q_head, int heads, const void* k, long k_row, long k_head, const void* v,
                           long v_row, long v_head, int kind, void* q_out, void* kc, void* vc, int pages, int kv, int page, int D,
                           const int* table, int width, const int* lengths, const int* cu, int seqs, int total, const float* rope,
                           int positions, int rope_dim, int interleaved, void* status, cudaStream_t st) {
  AppendParams p = {};
  if (!cache_ok(kc, vc, pages, kv, page, D, &p.c) || !rows_ok(cu, lengths, table, seqs, width, total, &p.r)) return -1;
  if (!k || !v || (heads && (!q || !q_out)) || heads < 0 || (kind != 1 && kind != 2)) return -1;
  if (rope_dim < 0 || rope_dim % 32 || rope_dim > D || (rope_dim && (!rope || positions < 1))) return -1;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                         (heads ? reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) : 0) |
                         (rope_dim ? reinterpret_cast<uintptr_t>(rope) : 0);
  if ((bits & 15) || ((q_row | q_head | k_row | k_head | v_row | v_head) & 7)) return -1;
  p.q = q; p.k = k; p.v = v; p.q_out = q_out;
  p.q_row = q_row; p.q_head = q_head; p.k_row = k_row; p.k_head = k_head; p.v_row = v_row; p.v_head = v_head;
  p.heads = heads; p.rope = rope; p.positions = positions; p.rope_dim = rope_dim; p.interleaved = interleaved;
  p.st = (TfStatusWord*)status;
  const dim3 grid(total, row_parts(total, (heads + 2 * kv) * (D / 16)));
  if (kind == 1) tf_launch(paged_append_kernel<__half>, grid, dim3(256), 0, st, p);
  else tf_launch(paged_append_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, p);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

// Keys and values of the same rows out of the cache: k, v [total][kv][D] bf16 (a row that has none reads zero).
TF_API int tf_paged_read(void* k, void* v, const void* kc, const void* vc, int pages, int kv, int page, int D, const int* table,
                         int width, const int* lengths, const int* cu, int seqs, int total, void* status, cudaStream_t st) {
  ReadParams p = {};
  if (!cache_ok(kc, vc, pages, kv, page, D, &p.c) || !rows_ok(cu, lengths, table, seqs, width, total, &p.r)) return -1;
  if (!k || !v || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15)) return -1;
  p.k = (__nv_bfloat16*)k;
  p.v = (__nv_bfloat16*)v;
  p.st = (TfStatusWord*)status;
  tf_launch(paged_read_kernel, dim3(total, row_parts(total, 2 * kv * (D / 16))), dim3(256), 0, st, p);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
