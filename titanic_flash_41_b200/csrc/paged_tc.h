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
}  // namespace paged

long paged_tc_workspace(int total, int seqs, int heads, int kv, int D, long keys, int sms);   // floats
int paged_tc_attention(const paged::AttnCall& a, int sms, cudaStream_t st);
