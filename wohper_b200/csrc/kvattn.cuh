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
  int window, first;  // window 0: none
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
// What the queries at positions p0 .. p1 see of n rows, taken together:
// [0, head) and [start, end).
struct KvSpan {
  int head, start, end;
};
__device__ __forceinline__ KvSpan kv_span(const KvAttnArgs& a, int p0, int p1, int n) {
  KvSpan s;
  s.end = p1 < 0 ? 0 : min(p1 + 1, n);
  s.start = a.window > 0 && p0 + 1 > a.window ? min(p0 + 1 - a.window, s.end) : 0;
  s.head = min(a.first, s.start);
  return s;
}

constexpr float kLog2e = 1.4426950408889634f;

// ---------------------------------------------------------------------------
// The tensor-core kernel's work list.  An item is the query rows of `tt` tokens
// of a request (or a part of one token's heads) that share a kv head; its rows
// of the cache, in order of position, are cut into tiles of kKvTile.  The tiles
// of all items, in the order request, tokens, kv head, head part, form one
// sequence that the CTAs share evenly; an item that lies in several CTAs is
// joined afterwards from their partial sums.
// ---------------------------------------------------------------------------
constexpr int kKvTile = 64;

struct KvWork {
  int rn;  // query rows an item has room for
  int tt;  // tokens of an item
  int ht;  // items that one token's heads of one kv head take
  int ctas, min_tiles;
  int4* meta;       // [tokens][heads]: first CTA, CTAs, its slot, redo
  float* part_o;    // [2 * ctas][rn][head_dim]
  float2* part_ml;  // [2 * ctas][rn]: maximum (base 2), sum
  int* part_redo;   // [2 * ctas]
};

struct KvItem {
  int t0, nt;  // its tokens
  int p0;      // position of the first
  int head, start, seen;  // rows [0, head) and [start, start + seen - head)
  int tiles;
};
__device__ __forceinline__ KvItem kv_item(const KvAttnArgs& a, const KvWork& w, int r, int2 tq,
                                          int i) {
  KvItem it;
  it.t0 = tq.x + i * w.tt;
  it.nt = min(w.tt, tq.y - i * w.tt);
  it.p0 = max(a.kv_lens[r], 0) - tq.y + i * w.tt;
  const KvSpan s = kv_span(a, it.p0, it.p0 + it.nt - 1, kv_rows_of(a, r));
  it.head = s.head;
  it.start = s.start;
  it.seen = s.head + s.end - s.start;
  it.tiles = max(1, (it.seen + kKvTile - 1) / kKvTile);
  return it;
}
// Tiles of request r over all its items.
__device__ __forceinline__ long long kv_request_tiles(const KvAttnArgs& a, const KvWork& w, int r) {
  const int2 tq = kv_queries(a, r);
  long long n = 0;
  for (int i = 0; i * w.tt < tq.y; ++i) n += kv_item(a, w, r, tq, i).tiles;
  return n * a.c.kv_heads * w.ht;
}
// CTAs that the sequence of `total` tiles is shared by, and the first tile of CTA i.
__device__ __forceinline__ int kv_ctas(const KvWork& w, long long total) {
  const long long n = (total + w.min_tiles - 1) / w.min_tiles;
  return n < w.ctas ? (int)n : w.ctas;
}
__device__ __forceinline__ long long kv_cta_start(long long total, int ctas, int i) {
  return total * i / ctas;
}
// The CTA that holds tile g: the last i with total * i / ctas <= g.
__device__ __forceinline__ int kv_cta_of(long long total, int ctas, long long g) {
  return (int)(((g + 1) * ctas - 1) / total);
}

}  // namespace wh
