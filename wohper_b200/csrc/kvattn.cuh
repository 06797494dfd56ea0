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
// A request's rows, clipped to what its block table can hold.
__device__ __forceinline__ int kv_clip(const KvAttnArgs& a, int len) {
  return min(max(len, 0), a.max_blocks * a.c.page);
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
// of the cache, in order of position, are cut into tiles of kKvTile.  The items,
// in the order request, tokens, kv head, head part, lie on one line, each
// w.lead units (what starting and ending an item costs, in tiles) and then one
// unit a tile; the CTAs share the line evenly.  An item that lies in several
// CTAs is joined afterwards from their partial sums.
// ---------------------------------------------------------------------------
constexpr int kKvTile = 64;

struct KvWork {
  int rn;    // query rows an item has room for
  int tt;    // tokens of an item
  int ht;    // items that one token's heads of one kv head take
  int lead;  // units ahead of an item's tiles
  int ctas, min_units;
  int4* meta;       // [tokens][heads]: first CTA, CTAs, its slot and row, redo
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
__device__ __forceinline__ KvItem kv_item(const KvAttnArgs& a, const KvWork& w, int len, int2 tq,
                                          int i) {
  KvItem it;
  it.t0 = tq.x + i * w.tt;
  it.nt = min(w.tt, tq.y - i * w.tt);
  it.p0 = max(len, 0) - tq.y + i * w.tt;
  const KvSpan s = kv_span(a, it.p0, it.p0 + it.nt - 1, kv_clip(a, len));
  it.head = s.head;
  it.start = s.start;
  it.seen = s.head + s.end - s.start;
  it.tiles = max(1, (it.seen + kKvTile - 1) / kKvTile);
  return it;
}
// The line, cut into ctas parts: CTA i has [start(i), start(i + 1)).  In 32 bits
// where it fits (a 64-bit division is some hundred cycles).
struct KvCut {
  long long total;
  int ctas;
  long long each;  // units of a CTA; the first `more` have one more
  int more;
  __device__ __forceinline__ KvCut(const KvWork& w, long long units) : total(units) {
    if (units <= 0x7fffffffLL) {
      const int u = (int)units;
      ctas = min(w.ctas, u / w.min_units + (u % w.min_units != 0));
      each = u / max(ctas, 1);
      more = u - (int)each * ctas;
    } else {
      ctas = w.ctas;
      each = units / ctas;
      more = (int)(units - each * ctas);
    }
  }
  __device__ __forceinline__ long long start(int i) const { return each * i + min(i, more); }
  __device__ __forceinline__ int cta_of(long long x) const {
    const long long big = (each + 1) * more;
    const bool in = x < big;
    const long long y = in ? x : x - big, d = in ? each + 1 : each;
    const int q = total <= 0x7fffffffLL ? (int)y / (int)d : (int)(y / d);
    return in ? q : more + q;
  }
};

}  // namespace wh
