// The many-row form of the attention over the paged cache (paged_tc.cu), called by tf_paged_attention (paged_attn.cu).
#pragma once
#include "paged.cuh"

namespace paged {
struct AttnCall {                          // checked arguments of tf_paged_attention
  Rows r;
  Cache c;
  const void* q;
  void* out;
  float* lse;
  long q_row, q_head, o_row, o_head;
  int heads, group, kind, window;
  float scale2;
  const int* first;
  const float* sink;
  float* work;
  TfStatusWord* st;
};
// Rows of sequence s that lie in the batch, their first one, and its position (offsets may be anything: what lies outside is no row).
__device__ __forceinline__ int rows_of(const Rows& r, int s, int* row0, int* pos0) {
  const int end = r.cu ? r.cu[s + 1] : s + 1, first = max(r.cu ? r.cu[s] : s, 0);
  *row0 = first;
  *pos0 = r.lengths[s] - (end - first);
  return max(min(end, r.total) - first, 0);
}
// first key that a row of sequence s at position `pos` sees (before the first token there is none to see)
__device__ __forceinline__ int first_key(const AttnCall& p, int s, int pos) {
  const int lo = max(p.first ? p.first[s] : 0, 0);
  return p.window ? max(lo, max(pos, 0) - p.window + 1) : lo;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// A row's maximum M and sum L (base 2, relative to M; 0: no keys) -> the logarithm of its softmax's sum
__device__ __forceinline__ float row_lse(float M, float L) { return L == 0.f ? -INFINITY : (M + log2f(L)) * 0.69314718055994531f; }
// The same with a sink, whose share L then has; returns the factor of the row's values.  A sink beyond base 2's range takes all, one of a row
// without keys is all there is: its logarithm is the sum's (a NaN on either side stays one).
__device__ __forceinline__ float take_sink(float sink, float M, float* L, float* lse) {
  const float s2 = sink * 1.4426950408889634f;
  if (s2 == INFINITY || (*L == 0.f && s2 == s2)) {
    *L = *L * 0.f + 1.f;
    *lse = *L - 1.f + sink;
    return 0.f;
  }
  const float m = fmaxf(M, s2), f = ex2(M - m);
  *L = *L * f + ex2(s2 - m);
  *lse = row_lse(m, *L);
  return f;
}
}  // namespace paged

long paged_tc_workspace(int total, int seqs, int heads, int kv, int D, long keys, int sms);   // floats
int paged_tc_attention(const paged::AttnCall& a, int sms, cudaStream_t st);
