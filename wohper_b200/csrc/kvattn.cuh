// kvattn.cuh -- arguments and row geometry of the attention over the paged
// 4-bit cache, shared by its kernels.
#pragma once
#include "kvcache.cuh"

namespace wh {

struct KvAttnArgs {
  static constexpr bool kTree = false;
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

// The same for a step that checks a tree of drafted tokens: the request's n queries
// are the tree's nodes and its last n rows theirs, rows base .. base + n - 1.  A
// node sees the rows before base as a query at its own position does, and row
// base + j where bit j of its mask is set.
struct KvTreeAttnArgs : KvAttnArgs {
  static constexpr bool kTree = true;
  const uint32_t* masks;  // [tokens][words]
  int words;
  const int32_t* positions;
};
// Does the query of token tok see row i?  last: the request's last row.
__device__ __forceinline__ bool kv_tree_sees(const KvTreeAttnArgs& a, int tok, int i, int base, int last) {
  if (i >= base) {
    const int j = i - base;
    return j < 32 * a.words && (__ldg(a.masks + (long long)tok * a.words + (j >> 5)) >> (j & 31) & 1);
  }
  if (a.window == 0 || i < a.first) return true;
  return i > min(max(__ldg(a.positions + tok), base), last) - a.window;
}

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
  int align;  // rows that an item's list begins at multiples of (a power of two)
  int ctas;
  int4* meta;       // [tokens][heads]: first CTA, CTAs, its slot and row, redo
  float* part_o;    // [2 * ctas][rn][head_dim]
  float2* part_ml;  // [2 * ctas][rn]: maximum (base 2), sum
  int* part_redo;   // [2 * ctas]
};

struct KvItem {
  int t0, nt;  // its tokens
  int p0;      // position of the first; of a tree: the first node's row
  int lo, from;           // sees rows [0, lo) and [from, ...)
  int head, start, seen;  // its list: [0, head), [start, start + seen - head), from w.align multiples
  int tiles;
};
// The u-th row of an item's list.
__device__ __forceinline__ int kv_key(int head, int start, int u) {
  return u < head ? u : start + (u - head);
}
template <class Args>
__device__ __forceinline__ KvItem kv_item(const Args& a, const KvWork& w, int len, int2 tq, int i) {
  KvItem it;
  it.t0 = tq.x + i * w.tt;
  it.nt = min(w.tt, tq.y - i * w.tt);
  it.p0 = max(len, 0) - tq.y + (Args::kTree ? 0 : i * w.tt);
  // a tree's positions lie between its first row and its last
  const KvSpan s = kv_span(a, it.p0, Args::kTree ? max(len, 0) - 1 : it.p0 + it.nt - 1, kv_clip(a, len));
  it.lo = s.head;
  it.from = s.start;
  it.head = (s.head + w.align - 1) & -w.align;
  it.start = s.start & -w.align;
  it.seen = it.head + s.end - it.start;
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
      ctas = min(w.ctas, u);
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

// A CTA's piece of the line and the item at its start (shared memory).
struct KvPlace {
  long long part[2][32];
  long long total, begin, end;  // units of the line; the piece
  long long first_tile, last_tile;
  KvItem item;
  int2 tq;
  int r, len, i, kvh, ht, j, into;  // j: the first tile; into: units into the item
  __device__ __forceinline__ int ntiles() const { return end > begin ? (int)(last_tile - first_tile) : 0; }
};
// Fills m; every thread of the CTA calls it.  A scan of the requests' units and
// tiles; the thread whose request holds an end of the piece finds the place.
template <int kThreads, class Args>
__device__ __forceinline__ void kv_place(const Args& a, const KvWork& w, KvPlace& m) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int kWarps = kThreads / 32;
  // a request's length and tokens, its units and tiles
  struct Req {
    int len;
    int2 tq;
    long long units, tiles;
  };
  auto request = [&](int r) {
    Req q{0, make_int2(0, 0), 0, 0};
    if (r >= a.requests) return q;
    q.len = a.kv_lens[r];
    q.tq = kv_queries(a, r);
    int items = 0;
    if (Args::kTree) {  // a tree's items see the same rows
      items = (q.tq.y + w.tt - 1) / w.tt;
      if (items > 0) q.tiles = (long long)kv_item(a, w, q.len, q.tq, 0).tiles * items;
    } else {
      for (int i = 0; i * w.tt < q.tq.y; ++i, ++items) q.tiles += kv_item(a, w, q.len, q.tq, i).tiles;
    }
    q.units = (q.tiles + (long long)items * w.lead) * (a.c.kv_heads * w.ht);
    q.tiles *= a.c.kv_heads * w.ht;
    if (q.tq.y > 0 && kv_clip(a, q.len) != q.len) flag(a.status, WH_DEV_BADARG);
    return q;
  };
  // Unit x of the line is unit `off` of request r, whose tiles follow `tiles`
  // earlier ones: the first tile at or after x, and (where) the item it is in.
  auto find = [&](int r, const Req& q, long long off, long long tiles, bool where) {
    const int per = a.c.kv_heads * w.ht;  // items of the same tokens
    int i = 0;
    KvItem it = kv_item(a, w, q.len, q.tq, 0);
    if (Args::kTree) {
      const long long each = (long long)(it.tiles + w.lead) * per;
      i = int(off / each);
      off -= i * each;
      tiles += (long long)i * it.tiles * per;
      if (i > 0) it = kv_item(a, w, q.len, q.tq, i);
    }
    while (!Args::kTree && off >= (long long)(it.tiles + w.lead) * per) {
      off -= (long long)(it.tiles + w.lead) * per;
      tiles += (long long)it.tiles * per;
      it = kv_item(a, w, q.len, q.tq, ++i);
    }
    const int one = it.tiles + w.lead;
    const int u = off <= 0x7fffffffLL ? (int)off / one : (int)(off / one);
    const int in = (int)(off - (long long)u * one);
    const int j = max(0, in - w.lead);
    if (where) {
      m.item = it;
      m.tq = q.tq;
      m.r = r;
      m.len = q.len;
      m.i = i;
      m.kvh = u / w.ht;
      m.ht = u % w.ht;
      m.j = j;
      m.into = in;
    }
    return tiles + (long long)u * it.tiles + j;
  };
  // Inclusive sums over kThreads requests at a time; with more requests than that
  // the line's length first.  Loops are kept rolled: this code runs once.
  long long total[2] = {0, 0}, base[2] = {0, 0};
  if (a.requests > kThreads) {
    for (int r = tid; r < a.requests; r += kThreads) {
      const Req p = request(r);
      total[0] += p.units;
      total[1] += p.tiles;
    }
#pragma unroll 1
    for (int o = 16; o; o >>= 1) {
      total[0] += __shfl_xor_sync(0xffffffffu, total[0], o);
      total[1] += __shfl_xor_sync(0xffffffffu, total[1], o);
    }
    if (lane == 0) {
      m.part[0][warp] = total[0];
      m.part[1][warp] = total[1];
    }
    __syncthreads();
    total[0] = total[1] = 0;
    for (int k = 0; k < kWarps; ++k) {
      total[0] += m.part[0][k];
      total[1] += m.part[1][k];
    }
    __syncthreads();
  }
#pragma unroll 1
  for (int r0 = 0; r0 < a.requests; r0 += kThreads) {
    const Req q = request(r0 + tid);
    long long x[2] = {q.units, q.tiles};
    if (r0 + warp * 32 < a.requests) {
#pragma unroll 1
      for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const long long p = __shfl_up_sync(0xffffffffu, x[k], o);
          if (lane >= o) x[k] += p;
        }
      }
      if (lane == 31) {
        m.part[0][warp] = x[0];
        m.part[1][warp] = x[1];
      }
    }
    __syncthreads();
    long long before[2] = {base[0], base[1]};
#pragma unroll 1
    for (int k = 0; k < kWarps && r0 + k * 32 < a.requests; ++k) {
      if (k < warp) {
        before[0] += m.part[0][k];
        before[1] += m.part[1][k];
      }
      base[0] += m.part[0][k];
      base[1] += m.part[1][k];
    }
    if (a.requests <= kThreads) {
      total[0] = base[0];
      total[1] = base[1];
    }
    const KvCut cut(w, total[0]);
    const bool in = (int)blockIdx.x < cut.ctas;
    const long long b = in ? cut.start(blockIdx.x) : 0, e = in ? cut.start(blockIdx.x + 1) : 0;
    if (tid == 0 && r0 == 0) {
      m.total = total[0];
      m.begin = b;
      m.end = e;
      if (e == total[0]) m.last_tile = total[1];
    }
    const long long u0 = before[0] + x[0] - q.units, t0 = before[1] + x[1] - q.tiles;
#pragma unroll 1
    for (int k = 0; in && k < 2; ++k) {
      const long long at = k ? e : b;
      if (u0 > at || at >= u0 + q.units) continue;
      const long long tile = find(r0 + tid, q, at - u0, t0, k == 0);
      (k ? m.last_tile : m.first_tile) = tile;
    }
    if (base[0] > e) break;  // uniform
    __syncthreads();
  }
  __syncthreads();
}
// Walks the items from a CTA's place on.
struct KvWalk {
  int r, len, i, kvh, ht, j;
  int2 tq;
  KvItem it;
  long long at;  // where the item begins on the line
  __device__ __forceinline__ explicit KvWalk(const KvPlace& p)
      : r(p.r), len(p.len), i(p.i), kvh(p.kvh), ht(p.ht), j(p.j), tq(p.tq), it(p.item), at(p.begin - p.into) {}
  template <class Args>
  __device__ __forceinline__ void next(const Args& a, const KvWork& w) {
    at += it.tiles + w.lead;
    j = 0;
    if (++ht < w.ht) return;
    ht = 0;
    if (++kvh < a.c.kv_heads) return;
    kvh = 0;
    ++i;
    if (i * w.tt >= tq.y) {
      i = 0;
      do {
        ++r;
        tq = kv_queries(a, r);
      } while (tq.y == 0);
      len = a.kv_lens[r];
    }
    it = kv_item(a, w, len, tq, i);
  }
};

}  // namespace wh
