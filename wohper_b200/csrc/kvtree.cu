// kvtree.cu -- a step that checks a tree of drafted tokens over the paged cache:
// the tokens' ancestors and positions (kv_tree_kernel), the path that agrees with
// the model's own tokens and the blocks that go back (kv_walk_kernel,
// kv_accept_kernel), and the kept rows moved to their places (kv_commit_kernel).
// The attention of such a step is the paged cache's own (kvattn.cuh).
//
// Token t = cu_q[r] + j is node j of request r; its row of the cache is row
// base + j, base = kv_lens[r] - n, n the request's nodes.  A parent comes before
// its children.
#include "kvcache.cuh"

namespace wh {

constexpr int kTreeNodes = 256;       // most nodes of a request
constexpr int kTreeTokens = 1 << 30;  // most tokens of a call: sums of two indices fit an int

// ---------------------------------------------------------------------------
// ancestors and positions
// ---------------------------------------------------------------------------
struct KvTreeArgs {
  int requests, tokens, words;
  const int32_t* parents;
  const int32_t* cu_q;
  const int32_t* kv_lens;
  uint64_t* masks;      // [tokens][words]
  int32_t* positions;
  uint32_t* status;
};

// A CTA a request, a thread a node.  With A_k(j) the 2^k nearest of j and its
// ancestors and u_k(j) the next one above them,
//   A_{k+1}(j) = A_k(j) + A_k(u_k(j)),  u_{k+1}(j) = u_k(u_k(j)):
// at most eight rounds in shared memory whatever the tree's depth.  Bound by the
// latency of the launch and of two dependent loads: 32 trees of 16 nodes 2.9 us, 1000 of
// 100 5.9 (1.6 MB out, 0.25 us at the copy's rate).
__global__ void __launch_bounds__(kTreeNodes) kv_tree_kernel(KvTreeArgs a) {
  __shared__ unsigned long long bits[2][kTreeNodes / 64][kTreeNodes];
  __shared__ short up[2][kTreeNodes], deep[2][kTreeNodes];
  pdl_wait_prior();
  const int r = blockIdx.x, j = threadIdx.x, room = blockDim.x;  // room: 64 * words
  const int t0 = min(max(a.cu_q[r], 0), a.tokens), t1 = min(max(a.cu_q[r + 1], t0), a.tokens);
  const int all = t1 - t0, n = min(all, room);
  if (j == 0 && all > room) flag(a.status, WH_DEV_BADARG);
  const int base = a.kv_lens[r] - all;
  int u = -1;
  if (j < n) {
    u = a.parents[t0 + j];
    if (u < -1 || u >= j) {
      flag(a.status, WH_DEV_BADARG);
      u = -1;
    }
  }
  unsigned long long own[kTreeNodes / 64];
#pragma unroll
  for (int w = 0; w < kTreeNodes / 64; ++w) own[w] = (j >> 6) == w ? 1ull << (j & 63) : 0;
  int d = u >= 0;
  for (int b = 0; __syncthreads_or(u >= 0); b ^= 1) {
    up[b][j] = (short)u;
    deep[b][j] = (short)d;
    for (int w = 0; w < a.words; ++w) bits[b][w][j] = own[w];
    __syncthreads();
    if (u >= 0) {
#pragma unroll
      for (int w = 0; w < kTreeNodes / 64; ++w)
        if (w < a.words) own[w] |= bits[b][w][u];
      d += deep[b][u];
      u = up[b][u];
    }
  }
  if (j < n) {
#pragma unroll
    for (int w = 0; w < kTreeNodes / 64; ++w)
      if (w < a.words) a.masks[(long long)(t0 + j) * a.words + w] = own[w];
    a.positions[t0 + j] = base + d;
  }
  // tokens of no request, and those that a request has too many
  const int first = min(max(a.cu_q[0], 0), a.tokens), past = min(max(a.cu_q[a.requests], first), a.tokens);
  auto none = [&](int t) {
    for (int w = 0; w < a.words; ++w) a.masks[(long long)t * a.words + w] = 0;
    a.positions[t] = -1;
  };
  for (int t = t0 + room + j; t < t1; t += room) none(t);
  for (long long i = (long long)blockIdx.x * room + j; i < a.tokens - past + first; i += (long long)gridDim.x * room)
    none(int(i < first ? i : past + i - first));
}

// ---------------------------------------------------------------------------
// accept
// ---------------------------------------------------------------------------
struct KvAcceptArgs {
  int requests, page, max_blocks, tokens, capacity;
  const int32_t* parents;
  const int32_t* drafts;
  const int32_t* targets;
  const int32_t* cu_q;
  const int32_t* kv_lens;
  const int32_t* block_table;
  int32_t* free_blocks;
  const int32_t* free_top;
  int32_t* free_top_out;
  int32_t* kv_lens_out;
  int32_t* counts;
  int32_t* path;  // [tokens]
  int32_t* next_tokens;
  uint32_t* status;
};

constexpr int kAcceptThreads = 1024;
// Requests up to which the accepting CTA walks the trees itself, two a warp; a
// second launch over many CTAs pays from there on.
constexpr int kAcceptInline = 2 * kAcceptThreads / 32;

// One request's path, by a warp.  Node c fits when its draft is the token that the
// model put after its parent; all nodes are compared at once, so that the walk
// itself is a ballot a step.
__device__ __forceinline__ void kv_walk_request(const KvAcceptArgs& a, int r) {
  const int lane = threadIdx.x & 31;
  const int t0 = a.cu_q[r], n = a.cu_q[r + 1] - t0, len = a.kv_lens[r];
  const bool bad = t0 < 0 || n < 0 || n > kTreeNodes || t0 > a.tokens - n || len < n ||
                   len > (long long)a.max_blocks * a.page;
  if (bad || n == 0) {
    if (bad && lane == 0) flag(a.status, WH_DEV_BADARG);
    const int from = min(max(t0, 0), a.tokens), to = min(max(a.cu_q[r + 1], from), a.tokens);
    for (int t = from + lane; t < to; t += 32) a.path[t] = -1;
    if (lane == 0) {
      a.counts[r] = 0;
      a.next_tokens[r] = -1;
      a.kv_lens_out[r] = len;
    }
    return;
  }
  constexpr int kPer = kTreeNodes / 32;
  int fits[kPer];  // the parent that node lane + 32 i fits, -1: none
  bool wrong = false;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int c = lane + 32 * i;
    fits[i] = -1;
    if (32 * i < n && c < n && c > 0) {
      const int p = a.parents[t0 + c];
      if (p < -1 || p >= c)
        wrong = true;
      else if (p >= 0 && a.drafts[t0 + c] == a.targets[t0 + p])
        fits[i] = p;
    }
  }
  if (wrong) flag(a.status, WH_DEV_BADARG);  // the node is on no path
  int at = 0, count = 1;
  if (lane == 0) a.path[t0] = 0;
  for (;;) {
    int next = -1;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (32 * i >= n || next >= 0) continue;
      const unsigned m = __ballot_sync(0xffffffffu, fits[i] == at);
      if (m) next = 32 * i + __ffs(m) - 1;
    }
    if (next < 0) break;
    at = next;
    if (lane == 0) a.path[t0 + count] = at;
    ++count;
  }
  for (int i = count + lane; i < n; i += 32) a.path[t0 + i] = -1;
  if (lane == 0) {
    a.counts[r] = count;
    a.next_tokens[r] = a.targets[t0 + at];
    a.kv_lens_out[r] = len - n + count;
  }
}

__global__ void __launch_bounds__(256) kv_walk_kernel(KvAcceptArgs a) {
  pdl_wait_prior();
  const int r = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (r < a.requests) kv_walk_request(a, r);
}

// One CTA: the blocks past each request's new length go on the stack, in the order
// of requests and pages, found by one scan; a stack that they do not fit undoes the
// step.  Latency of dependent loads, as kv_plan_kernel: 32 trees of 16 nodes 5.4 us, 1000
// of 100 9.7 with the launch before it.
__global__ void __launch_bounds__(kAcceptThreads) kv_accept_kernel(KvAcceptArgs a, int walk) {
  __shared__ long long part[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait_prior();
  if (walk) {
    for (int r = warp; r < a.requests; r += kAcceptThreads / 32) kv_walk_request(a, r);
    __syncthreads();
  }
  const int top = *a.free_top;
  const int per = ceil_div(a.requests, kAcceptThreads), r0 = tid * per;
  // blocks that request r holds, needs
  auto pages = [&](int r, int& held, int& need) {
    const int len = a.kv_lens[r], after = a.kv_lens_out[r];
    const bool none = after >= len || after < 0;  // nothing dropped, or a bad request
    held = none ? 0 : ceil_div(len, a.page);
    need = none ? 0 : ceil_div(after, a.page);
  };
  long long sum = 0;
  for (int i = 0; i < per && r0 + i < a.requests; ++i) {
    int held, need;
    pages(r0 + i, held, need);
    sum += held - need;
  }
  long long x = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long p = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += p;
  }
  if (lane == 31) part[warp] = x;
  __syncthreads();
  if (warp == 0) {
    long long v = part[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long p = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += p;
    }
    part[lane] = v;
  }
  __syncthreads();
  const long long total = part[31];
  const bool ok = top >= 0 && top <= a.capacity && top + total <= a.capacity;
  if (tid == 0) {
    if (!ok) flag(a.status, WH_DEV_BADARG);
    *a.free_top_out = ok ? int(top + total) : top;
  }
  long long to = top + x - sum + (warp ? part[warp - 1] : 0);
  for (int i = 0; i < per && r0 + i < a.requests; ++i) {
    const int r = r0 + i;
    if (ok) {
      int held, need;
      pages(r, held, need);
      for (int p = need; p < held; ++p) a.free_blocks[to++] = a.block_table[(long long)r * a.max_blocks + p];
    } else {
      a.counts[r] = 0;
      a.next_tokens[r] = -1;
      a.kv_lens_out[r] = a.kv_lens[r];
    }
  }
  // tokens of no request; all of them where the step is undone
  const int first = min(max(a.cu_q[0], 0), a.tokens), past = min(max(a.cu_q[a.requests], first), a.tokens);
  for (int t = tid; t < (ok ? first : a.tokens); t += kAcceptThreads) a.path[t] = -1;
  for (int t = past + tid; t < a.tokens; t += kAcceptThreads) a.path[t] = -1;
}

// ---------------------------------------------------------------------------
// commit
// ---------------------------------------------------------------------------
struct KvCommitArgs {
  KvCacheDev c;
  int requests, tokens, max_blocks;
  const int32_t* counts;
  const int32_t* path;
  const int32_t* cu_q;
  const int32_t* kv_lens;
  const int32_t* block_table;
  uint32_t* status;
};

// A CTA moves one kv head's keys (or values) of one request: 16 bytes of codes and
// the scale byte of the same 32 columns a thread.  path[i] >= i grows with i, so a
// chunk of rows that is read before it is written never loses a later chunk's
// rows.  Bound by the latency of its chain of loads (lengths, path, blocks, rows); with
// a read of the rows after it 8 trees of 8 nodes take 5.3 us, 32 of 16 in 43 layers
// inside a block 14.8 (17.7 MB read and written, 2.7 us at the copy's rate).
constexpr int kCommitThreads = 128, kCommitEach = 4;
__global__ void __launch_bounds__(kCommitThreads) kv_commit_kernel(KvCommitArgs a) {
  pdl_wait_prior();
  const int parts = a.c.head_dim / 32, heads = a.c.kv_heads * (a.c.shared ? 1 : 2);
  const int r = blockIdx.x / heads;
  int head = blockIdx.x - r * heads;
  const bool values = head >= a.c.kv_heads;
  if (values) head -= a.c.kv_heads;
  const int t0 = a.cu_q[r], n = a.cu_q[r + 1] - t0, len = a.kv_lens[r], count = a.counts[r];
  if (count == 0) return;
  bool bad = t0 < 0 || n < 0 || t0 > a.tokens - n || count < 0 || count > n || len < n ||
             len > (long long)a.max_blocks * a.c.page;
  for (int i = threadIdx.x; !bad && i < count; i += kCommitThreads) {
    const int p = a.path[t0 + i];
    bad = p < i || p >= n || (i > 0 && p <= a.path[t0 + i - 1]);
  }
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) flag(a.status, WH_DEV_BADARG);
    return;
  }
  uint8_t* codes = values ? a.c.values : a.c.keys;
  uint8_t* scales = values ? a.c.value_scales : a.c.key_scales;
  const int base = len - n;
  const int32_t* table = a.block_table + (long long)r * a.max_blocks;
  // the head's row i: where its codes and scales begin; false where its block is none
  auto locate = [&](int i, long long& co, long long& so) {
    const int pg = kv_page_of(a.c, i), block = table[pg];
    const long long row = (long long)head * a.c.page + (i - pg * a.c.page);
    co = block * a.c.block_stride + row * (a.c.head_dim / 2);
    so = block * a.c.scale_block_stride + row * parts;
    return block >= 0 && block < a.c.blocks;
  };
  const int rows = kCommitThreads * kCommitEach / parts;  // of a chunk
  for (int i0 = 0; i0 < count; i0 += rows) {
    const int pieces = min(rows, count - i0) * parts;
    uint4 w[kCommitEach];
    uint8_t sb[kCommitEach];
    long long co[kCommitEach], so[kCommitEach];
#pragma unroll
    for (int k = 0; k < kCommitEach; ++k) {
      const int at = threadIdx.x + k * kCommitThreads;
      co[k] = -1;
      if (at >= pieces) continue;
      const int i = i0 + at / parts, part = at % parts, p = a.path[t0 + i];
      if (p == i) continue;
      long long from, from_s;
      const bool src = locate(base + p, from, from_s), dst = locate(base + i, co[k], so[k]);
      if (!src || !dst) {
        flag(a.status, WH_DEV_BADARG);
        co[k] = -1;
        continue;
      }
      w[k] = *reinterpret_cast<const uint4*>(codes + from + part * 16);
      sb[k] = scales[from_s + part];
      co[k] += part * 16;
      so[k] += part;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kCommitEach; ++k)
      if (co[k] >= 0) {
        *reinterpret_cast<uint4*>(codes + co[k]) = w[k];
        scales[so[k]] = sb[k];
      }
    __syncthreads();
  }
}

}  // namespace wh

// ---------------------------------------------------------------------------
// C entry points
// ---------------------------------------------------------------------------
extern "C" {

wh_status wh_kv_tree(wh_ctx* c, int requests, int tokens, int max_nodes, const int32_t* parents,
                     const int32_t* cu_q, const int32_t* kv_lens, uint64_t* masks,
                     int32_t* positions, wh_stream_t stream) {
  if (wh_status st = kv_device_check(c)) return st;
  if (requests < 1 || max_nodes < 1) return fail(WH_ERR_EMPTY_SHAPE, "tree: requests, max_nodes");
  if (tokens < 0) return fail(WH_ERR_INVALID_SHAPE, "tree: tokens");
  if (tokens > kTreeTokens) return fail(WH_ERR_UNSUPPORTED, "tree: tokens > 2^30");
  if (max_nodes > kTreeNodes) return fail(WH_ERR_UNSUPPORTED, "tree: max_nodes > 256");
  if (tokens == 0) return WH_OK;
  if (!parents || !cu_q || !kv_lens || !masks || !positions)
    return fail(WH_ERR_INVALID_POINTER, "tree: null pointer");
  const int words = (max_nodes + 63) / 64;
  const KvTreeArgs a{requests, tokens, words, parents, cu_q, kv_lens, masks, positions, c->status};
  WH_CUDA(launch_pdl(kv_tree_kernel, dim3(requests), 64 * words, 0, (cudaStream_t)stream, c->pdl(), a));
  return WH_OK;
}

wh_status wh_kv_accept(wh_ctx* c, int requests, int page, int max_blocks, int tokens,
                       const int32_t* parents, const int32_t* drafts, const int32_t* targets,
                       const int32_t* cu_q, const int32_t* kv_lens, const int32_t* block_table,
                       int32_t* free_blocks, int capacity, const int32_t* free_top,
                       int32_t* free_top_out, int32_t* kv_lens_out, int32_t* counts,
                       int32_t* path, int32_t* next_tokens, wh_stream_t stream) {
  if (wh_status st = kv_device_check(c)) return st;
  if (requests < 1 || page < 1 || max_blocks < 1)
    return fail(WH_ERR_EMPTY_SHAPE, "accept: requests, page, max_blocks");
  if (tokens < 0 || capacity < 0) return fail(WH_ERR_INVALID_SHAPE, "accept: tokens, capacity");
  if (tokens > kTreeTokens) return fail(WH_ERR_UNSUPPORTED, "accept: tokens > 2^30");
  if ((long long)max_blocks * page > 0x7fffffffLL || page > (1 << 20))
    return fail(WH_ERR_UNSUPPORTED, "accept: max_blocks * page > 2^31 - 1");
  if (!cu_q || !kv_lens || !block_table || !free_blocks || !free_top || !free_top_out ||
      !kv_lens_out || !counts || !next_tokens ||
      (tokens > 0 && (!parents || !drafts || !targets || !path)))
    return fail(WH_ERR_INVALID_POINTER, "accept: null pointer");
  if (free_top == free_top_out || kv_lens == kv_lens_out)
    return fail(WH_ERR_INVALID_POINTER, "accept: an output may not be an input");
  const KvAcceptArgs a{requests, page,        max_blocks,  tokens,   capacity,     parents,     drafts,
                       targets,  cu_q,        kv_lens,     block_table, free_blocks, free_top,  free_top_out,
                       kv_lens_out, counts,   path,        next_tokens, c->status};
  const cudaStream_t s = (cudaStream_t)stream;
  const bool inl = requests <= kAcceptInline;
  if (!inl)
    WH_CUDA(launch_pdl(kv_walk_kernel, dim3((requests + 7) / 8), 256, 0, s, c->pdl(), a));
  WH_CUDA(launch_pdl(kv_accept_kernel, dim3(1), kAcceptThreads, 0, s, c->pdl(), a, inl ? 1 : 0));
  return WH_OK;
}

wh_status wh_kv_commit(wh_ctx* c, const wh_kv_cache* cache, int requests, int tokens,
                       const int32_t* counts, const int32_t* path, const int32_t* cu_q,
                       const int32_t* kv_lens, const int32_t* block_table, int max_blocks,
                       wh_stream_t stream) {
  if (wh_status st = kv_device_check(c)) return st;
  KvCommitArgs a{};
  if (wh_status st = kv_cache_check(cache, &a.c)) return st;
  if (requests < 1 || max_blocks < 1) return fail(WH_ERR_EMPTY_SHAPE, "commit: requests, max_blocks");
  if (tokens < 0) return fail(WH_ERR_INVALID_SHAPE, "commit: tokens");
  if ((long long)max_blocks * cache->page > 0x7fffffffLL)
    return fail(WH_ERR_UNSUPPORTED, "commit: max_blocks * page > 2^31 - 1");
  const long long ctas = (long long)requests * cache->kv_heads * (cache->values ? 2 : 1);
  if (ctas > 0x7fffffffLL) return fail(WH_ERR_UNSUPPORTED, "commit: requests * kv_heads too large");
  if (tokens == 0) return WH_OK;
  if (!counts || !path || !cu_q || !kv_lens || !block_table)
    return fail(WH_ERR_INVALID_POINTER, "commit: null pointer");
  a.requests = requests;
  a.tokens = tokens;
  a.max_blocks = max_blocks;
  a.counts = counts;
  a.path = path;
  a.cu_q = cu_q;
  a.kv_lens = kv_lens;
  a.block_table = block_table;
  a.status = c->status;
  WH_CUDA(launch_pdl(kv_commit_kernel, dim3((unsigned)ctas), kCommitThreads, 0, (cudaStream_t)stream, c->pdl(), a));
  return WH_OK;
}

}  // extern "C"
