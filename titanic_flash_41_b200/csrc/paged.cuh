// The batch of rows that a call on the paged cache works on, shared by paged.cu, paged_attn.cu and paged_tc.cu.
#pragma once
#include "fp4.cuh"

namespace paged {

using fp4::Cache;

struct Rows {                              // where the rows of the batch lie
  const int* cu;                           // [seqs + 1] row offsets, or null: row i is the one row of sequence i
  const int* lengths;                      // [seqs] tokens in the cache once the rows are in it
  const int* table;                        // [seqs][width] page of every 2^shift tokens
  int seqs, width, total;
};

template <typename T>
__device__ __forceinline__ float2 two(uint32_t w);
template <>
__device__ __forceinline__ float2 two<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
template <>
__device__ __forceinline__ float2 two<__nv_bfloat16>(uint32_t w) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w)); }
template <typename T>
__device__ __forceinline__ uint32_t pack(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
inline bool cache_ok(const void* k, const void* v, int pages, int kv, int page, int D, Cache* c) {
  const int shift = fp4::page_shift(page);
  if (!k || !v || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15)) return false;
  if (pages < 1 || kv < 1 || shift < 0 || (D != 64 && D != 128)) return false;
  c->k = (uint8_t*)k;
  c->v = (uint8_t*)v;
  c->pages = pages;
  c->kv = kv;
  c->shift = shift;
  c->D = D;
  c->block = (long)page * (D / 2 + D / 16);
  return true;
}
constexpr long kMostTokens = (1l << 31) - 1024;            // of a table: positions and the ends of the tiles behind them are 32-bit numbers
inline bool rows_ok(const int* cu, const int* lengths, const int* table, int seqs, int width, int shift, int total, Rows* r) {
  if (!lengths || !table || seqs < 1 || width < 1 || total < 1 || (!cu && total > seqs)) return false;
  if ((long)width << shift > kMostTokens) return false;
  *r = {cu, lengths, table, seqs, width, total};
  return true;
}
}  // namespace paged
