// kvattn.cuh -- arguments and row geometry of the attention over the paged
// 4-bit cache, shared by its kernels.
#pragma once
#include "kvcache.cuh"

namespace wh {

struct KvAttnArgs {
  KvCacheDev c;
  const void* q;
  void* out;
  int dtype;  // WH_DTYPE_*
  int tokens, heads, group;  // group = heads / kv_heads
  long long q_token_stride, q_head_stride, out_token_stride, out_head_stride;  // elements
  int requests;
  const int32_t* cu_q;  // nullable: one query a request
  const int32_t* kv_lens;
  const int32_t* block_table;
  int max_blocks;
  float scale;
  int window, first;
  const float* sink;
  uint32_t* status;
};

// The queries of request r, clipped to the call's tokens.
__device__ __forceinline__ int2 kv_queries(const KvAttnArgs& a, int r) {
  if (!a.cu_q) return make_int2(r, 1);
  const int t0 = min(max(a.cu_q[r], 0), a.tokens);
  const int t1 = min(max(a.cu_q[r + 1], t0), a.tokens);
  return make_int2(t0, t1 - t0);
}
// The request that owns token t, -1 for a token past the last request's.
__device__ __forceinline__ int kv_request_of(const KvAttnArgs& a, int t) {
  if (!a.cu_q) return t < a.requests ? t : -1;
  if (t < a.cu_q[0] || t >= a.cu_q[a.requests]) return -1;
  int lo = 0, hi = a.requests - 1;  // the last r with cu_q[r] <= t
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.cu_q[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}
// Rows of the request, clipped to what its block table can hold.
__device__ __forceinline__ int kv_rows_of(const KvAttnArgs& a, int r) {
  return min(max(a.kv_lens[r], 0), a.max_blocks * a.c.page);
}
// What a query at position p sees of n rows: [0, head) and [start, end).
struct KvSpan {
  int head, start, end;
};
__device__ __forceinline__ KvSpan kv_span(const KvAttnArgs& a, int p, int n) {
  KvSpan s;
  s.end = max(0, min(p + 1, n));
  s.start = a.window > 0 ? max(0, min(p + 1 - a.window, s.end)) : 0;
  s.head = min(a.first, s.start);
  return s;
}

constexpr float kLog2e = 1.4426950408889634f;

}  // namespace wh
