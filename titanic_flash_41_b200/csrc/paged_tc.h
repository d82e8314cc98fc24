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
}  // namespace paged

long paged_tc_workspace(int total, int seqs, int heads, int kv, int D, long keys, int sms);   // floats
int paged_tc_attention(const paged::AttnCall& a, int sms, cudaStream_t st);
