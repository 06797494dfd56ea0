// kvattn.cu -- attention over the paged 4-bit key/value cache.
//
// Query row (token t of request r at position p, head h), over the rows i it
// sees (kv_span):
//   s_i = scale * q . k_i        m = max_i s_i       l = sum_i e^(s_i - m)
//   o = sum_i e^(s_i - m) v_i / (l + e^(sink - m))
// in one pass over the rows with a running maximum: when m grows, l and o
// shrink by e^(m_old - m).
#include "kvattn.cuh"

namespace wh {

// ---------------------------------------------------------------------------
// One query row per CTA on the CUDA cores, f32 throughout: any head_dim that is
// a multiple of 32, any scale byte, any value of q.
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 128;
struct KvRowSmem {
  float q[512];
  float p[kRowThreads];
  long long row[kRowThreads];    // row index in its block (code and scale offsets follow)
  int block[kRowThreads];
  float red[8];
  float acc[kRowThreads * 8];
};

__device__ __forceinline__ float row_reduce_max(float v, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}
__device__ __forceinline__ float row_reduce_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

template <class T>
__device__ void kv_attend_row(const KvAttnArgs& a, int r, int t, int h, KvRowSmem& sm) {
  const int tid = threadIdx.x;
  const int D = a.c.head_dim, parts = D / 8;
  const int kvh = h / a.group;
  const int2 tq = kv_queries(a, r);
  const int p = max(a.kv_lens[r], 0) - tq.y + (t - tq.x);
  const int n = kv_clip(a, a.kv_lens[r]);
  if (tid == 0 && n != a.kv_lens[r]) flag(a.status, WH_DEV_BADARG);
  const KvSpan sp = kv_span(a, p, p, n);
  const int seen = sp.head + sp.end - sp.start;
  const T* q = reinterpret_cast<const T*>(a.q) + t * a.q_token_stride + h * a.q_head_stride;
  __syncthreads();
  if (tid < parts) {
    float v[8];
    kv_load8(q + tid * 8, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) sm.q[tid * 8 + j] = v[j];
  }
  // value columns: lane group `part` of 8 columns, keys sub, sub + subs, ...
  const int subs = kRowThreads / parts, part = tid % parts, sub = tid / parts;
  const float inf = __int_as_float(0x7f800000);
  float m = -inf, l = 0.0f;
  float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  for (int u0 = 0; u0 < seen; u0 += kRowThreads) {
    __syncthreads();
    const int u = u0 + tid;
    float s = -inf;
    int block = -1;
    long long row = 0;
    if (u < seen) {
      const int i = u < sp.head ? u : sp.start + (u - sp.head);
      block = a.block_table[(long long)r * a.max_blocks + i / a.c.page];
      if (block < 0 || block >= a.c.blocks) {
        flag(a.status, WH_DEV_BADARG);
        block = -1;
      }
      row = (long long)kvh * a.c.page + i % a.c.page;
    }
    if (block >= 0) {
      const uint8_t* codes = a.c.keys + block * a.c.block_stride + row * (D / 2);
      const uint8_t* scales = a.c.key_scales + block * a.c.scale_block_stride + row * (D / 32);
      float dot = 0.0f;
      for (int b = 0; b < D / 32; ++b) {
        const uint4 w = reinterpret_cast<const uint4*>(codes)[b];
        const uint32_t sb = scales[b];
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
        float part_sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float v[8];
          kv_decode8(ws[j], sb, v);
#pragma unroll
          for (int e = 0; e < 8; ++e) part_sum = fmaf(v[e], sm.q[b * 32 + j * 8 + e], part_sum);
        }
        dot += part_sum;
      }
      s = dot * a.scale;
    }
    sm.block[tid] = block;
    sm.row[tid] = row;
    const float mx = fmaxf(m, row_reduce_max(s, sm.red));  // fmaxf passes over NaN
    const float base = mx == -inf ? 0.0f : mx;
    const float shrink = m == -inf ? 0.0f : exp2f((m - base) * kLog2e);
    const float w = block >= 0 ? exp2f((s - base) * kLog2e) : 0.0f;
    sm.p[tid] = w;
    l = l * shrink + row_reduce_sum(w, sm.red);
    m = mx;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= shrink;
    const int cnt = min(kRowThreads, seen - u0);
    if (sub < subs)
      for (int k = sub; k < cnt; k += subs) {
        if (sm.block[k] < 0) continue;
        const uint8_t* codes = a.c.values + sm.block[k] * a.c.block_stride + sm.row[k] * (D / 2);
        const uint8_t* scales =
            a.c.value_scales + sm.block[k] * a.c.scale_block_stride + sm.row[k] * (D / 32);
        float v[8];
        kv_decode8(reinterpret_cast<const uint32_t*>(codes)[part], scales[part >> 2], v);
        const float w = sm.p[k];
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = fmaf(w, v[e], acc[e]);
      }
  }
  // the sink's share, then the sum over the key subsets
  float o_scale = 1.0f;
  if (a.sink && seen > 0) {
    const float sk = a.sink[h];
    const float mx = fmaxf(m, sk), base = mx == -inf ? 0.0f : mx;
    o_scale = m == -inf ? 0.0f : exp2f((m - base) * kLog2e);
    l = l * o_scale + exp2f((sk - base) * kLog2e);
  }
  o_scale = l == 0.0f ? 0.0f : o_scale / l;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 8; ++e) sm.acc[tid * 8 + e] = acc[e];
  __syncthreads();
  if (tid < parts) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float x = 0.0f;
      for (int k = 0; k < subs; ++k) x += sm.acc[(k * parts + tid) * 8 + e];
      v[e] = x * o_scale;
    }
    kv_store8(reinterpret_cast<T*>(a.out) + t * a.out_token_stride + h * a.out_head_stride +
                  tid * 8,
              v);
  }
}

template <class T>
__global__ void __launch_bounds__(kRowThreads) kv_attend_row_kernel(KvAttnArgs a) {
  __shared__ KvRowSmem sm;
  pdl_wait_prior();
  const int t = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
  const int r = kv_request_of(a, t);
  if (r < 0) return;
  kv_attend_row<T>(a, r, t, h, sm);
}

// ---------------------------------------------------------------------------
// Joins the tensor-core kernel's partial sums of items that lie in several CTAs
// and computes rows again that its f16 tiles cannot hold.  kWpr warps share a
// row's parts (added in the order of the rows they cover within a warp, then
// over the warps), a lane has kV groups of 4 columns.  Many rows: a warp each,
// all columns; few rows (long contexts, many parts): a CTA each and 128 columns.
// Bound by the latency of its dependent loads (row, parts' maxima, sums): about 6 us
// for 2048 rows in five parts, 8 for 64 rows in 148.
// ---------------------------------------------------------------------------
constexpr int kJoinParts = 640;  // most CTAs that a line is cut into
template <class T, int kV, int kWpr>
__global__ void __launch_bounds__(kRowThreads) kv_join_kernel(KvAttnArgs a, KvWork w) {
  __shared__ KvRowSmem sm;
  __shared__ int redo_row[4];
  __shared__ float red[4];
  extern __shared__ float2 part[];  // [rows][kJoinParts]: maximum (then weight), sum
  constexpr int kRows = kRowThreads / 32 / kWpr;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = warp % kWpr;
  const long long id = (long long)blockIdx.x * kRows + warp / kWpr;
  const int t = int(id / a.heads), h = int(id % a.heads);
  pdl_wait_prior();
  const int first = a.cu_q ? max(a.cu_q[0], 0) : 0;
  const int past = min(a.cu_q ? a.cu_q[a.requests] : a.requests, a.tokens);
  const bool mine = t >= first && t < past;
  const int4 mt = mine ? w.meta[id] : make_int4(0, 1, 0, 0);
  const int parts = mt.y, row = mt.z >> 1;
  // a meta that the tensor-core kernel did not write: it gave up on a wait
  const bool bad = mt.x < 0 || parts < 1 || parts > w.ctas || mt.x > w.ctas - parts || row < 0 || row >= w.rn;
  if (bad) flag(a.status, WH_DEV_BADARG);
  auto slot_of = [&](int p) { return 2 * (mt.x + p) + (p == 0 ? mt.z & 1 : 0); };
  const float inf = __int_as_float(0x7f800000);
  int redo = bad ? 0 : mt.w;
  bool join = !bad && parts > 1;
  // the parts' maxima and sums, kept beside; the row's maximum
  float2* ml = &part[warp / kWpr * kJoinParts];
  float top = -inf;
  if (join)
    for (int p = sub * 32 + lane; p < parts; p += 32 * kWpr) {
      const float2 x = w.part_ml[(long long)slot_of(p) * w.rn + row];
      redo |= w.part_redo[slot_of(p)];
      ml[p] = x;
      top = fmaxf(top, x.x);
    }
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  redo = __any_sync(0xffffffffu, redo);
  if (kWpr > 1) {  // one row a CTA
    if (lane == 0) red[warp] = top;
    redo = __syncthreads_or(redo);
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  } else {
    __syncwarp();
  }
  join = join && !redo;
  const float sk = a.sink && join ? a.sink[h] * kLog2e : -inf;
  const float to = fmaxf(top, sk), base = to == -inf ? 0.0f : to;
  // their weights; the row's sum
  float z = 0.0f;
  if (join)
    for (int p = sub * 32 + lane; p < parts; p += 32 * kWpr) {
      const float2 x = ml[p];
      const float f = x.x == -inf ? 0.0f : exp2f(x.x - base);
      z += x.y * f;
      ml[p].x = f;
    }
#pragma unroll
  for (int o = 16; o; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
  if (kWpr > 1) {
    __syncthreads();
    if (lane == 0) red[warp] = z;
    __syncthreads();
    z = (red[0] + red[1]) + (red[2] + red[3]);
  } else {
    __syncwarp();
  }
  if (a.sink && join) z += exp2f(sk - base + kLift);
  float4 acc[kV];
#pragma unroll
  for (int v = 0; v < kV; ++v) acc[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  const int D = a.c.head_dim, dim = blockIdx.y * 128 + lane * 4;
  if (join && dim < D) {
#pragma unroll(kV == 1 ? 8 : 8 / kV)
    for (int p = sub; p < parts; p += kWpr) {
      const float f = ml[p].x;
      const float* at = w.part_o + ((long long)slot_of(p) * w.rn + row) * D + dim;
#pragma unroll
      for (int v = 0; v < kV; ++v) {
        const float4 o = *reinterpret_cast<const float4*>(at + v * 128);
        acc[v].x = fmaf(f, o.x, acc[v].x);
        acc[v].y = fmaf(f, o.y, acc[v].y);
        acc[v].z = fmaf(f, o.z, acc[v].z);
        acc[v].w = fmaf(f, o.w, acc[v].w);
      }
    }
  }
  if (kWpr > 1) {
    static_assert(kWpr == 1 || kV == 1, "one group of columns where warps share a row");
    *reinterpret_cast<float4*>(&sm.acc[threadIdx.x * 4]) = acc[0];
    __syncthreads();
    acc[0] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k = 0; k < kWpr; ++k) {
      const float4 o = *reinterpret_cast<const float4*>(&sm.acc[(k * 32 + lane) * 4]);
      acc[0].x += o.x;
      acc[0].y += o.y;
      acc[0].z += o.z;
      acc[0].w += o.w;
    }
  }
  if (join && sub == 0 && dim < D) {
    const float inv = z == 0.0f ? 0.0f : 1.0f / z;
    T* out = reinterpret_cast<T*>(a.out) + t * a.out_token_stride + h * a.out_head_stride + dim;
#pragma unroll
    for (int v = 0; v < kV; ++v) kv_store4(out + v * 128, acc[v], inv);
  }
  // rows to be computed again, one after the other by the whole CTA
  if (lane == 0 && sub == 0) redo_row[warp / kWpr] = redo && mine && blockIdx.y == 0;
  __syncthreads();
  for (int k = 0; k < kRows; ++k) {
    if (!redo_row[k]) continue;
    const long long i = (long long)blockIdx.x * kRows + k;
    const int r = kv_request_of(a, int(i / a.heads));
    if (r >= 0) kv_attend_row<T>(a, r, int(i / a.heads), int(i % a.heads), sm);
  }
}

}  // namespace wh

// ---------------------------------------------------------------------------
// C entry points
// ---------------------------------------------------------------------------
namespace {

// Which kernel takes the call and how it cuts the queries.
//  - few: a pass over the cache for every 16 query rows (8 of f32) of a kv head,
//    bound by latency (56 % of the issue slots, 40 % of the memory rate);
//  - tc: one pass for 64 rows (32 of f32), bound by the tile pipeline;
//  - row: a CTA a query row, for rows of other widths (16 x 4096, 32 heads on 8 x 96,
//    bf16: 202 us; 128 wide on the few-rows kernel 38).
// Measured on 8 requests of 4096 rows, 8 kv heads, us (few / tc), rows to a kv head:
//   64 wide,  bf16: 16 20/47, 32 31/47, 48 39/47;         f32: 16 29/45, 24 40/46, 32 49/46
//   128 wide, bf16: 16 26/47, 32 42/48, 40 55/48, 48 56/49; f32: 16 39/47, 24 53/47, 32 66/48
//   256 wide, bf16: 16 50/65, 24 72/65, 32 74/66;         f32: 8 42/64, 16 66/66, 24 90/66
// The limits lie in the pass above the crossing of such equal requests (128 wide 33-40
// and f32 17-20 rows, 256 wide 17-24), which costs them up to 7 us here.
// A call's tokens are taken as evenly spread over its requests, the one thing
// the host knows.  An item with fewer rows than it has room for is still right, but
// where one request has most of the tokens the other requests, or it, get the kernel
// that suits them less: 31 decodes x 4096 rows 66 us, a prompt of 512 tokens 49, both
// in one call 184 (32 heads on 8 x 128, bf16).
enum class KvWay { few, tc, row };
struct KvHow {
  KvWay way;
  bool split;  // f32 queries: two f16 to a value
  KvWork w;
};
KvHow kv_how(const wh_ctx* c, int head_dim, int kv_heads, int tokens, int heads, int requests,
             int dtype) {
  KvHow p{};
  p.way = KvWay::row;
  const int d = head_dim, group = heads / kv_heads;
  if (d != 64 && d != 128 && d != 256 && d != 512) return p;
  p.split = dtype == WH_DTYPE_F32;
  const long long each = (long long)group * ((tokens + requests - 1) / requests);
  KvWork& w = p.w;
  const int most = p.split ? (d == 256 ? 16 : d == 128 ? 20 : 24) : (d == 256 ? 24 : d == 128 ? 40 : 48);
  if (d <= 256 && each <= most) {
    p.way = KvWay::few;
    w.rn = p.split || each <= 8 ? 8 : 16;
    w.ctas = c->num_sms * (d * w.rn <= 8 * 128 ? 4 : d * w.rn == 8 * 256 ? 3 : 2);
    w.lead = 8;
    w.align = kFewKeys;
  } else {
    p.way = KvWay::tc;
    w.rn = p.split ? kTcCols / 2 : kTcCols;
    w.ctas = c->num_sms;
    w.lead = 4;
    w.align = 1;
  }
  w.ctas = std::min(w.ctas, kJoinParts);
  w.tt = std::max(1, w.rn / group);
  w.ht = (group + w.rn - 1) / w.rn;
  return p;
}
// Places the scratch arrays; returns their bytes.
size_t kv_scratch(KvWork& w, int head_dim, int tokens, int heads, uint8_t* base) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    uint8_t* q = base + at;
    at += align256(bytes);
    return q;
  };
  const size_t slots = 2 * (size_t)w.ctas;
  w.meta = reinterpret_cast<int4*>(take(sizeof(int4) * tokens * heads));
  w.part_o = reinterpret_cast<float*>(take(sizeof(float) * slots * w.rn * head_dim));
  w.part_ml = reinterpret_cast<float2*>(take(sizeof(float2) * slots * w.rn));
  w.part_redo = reinterpret_cast<int*>(take(sizeof(int) * slots));
  return at;
}
template <int kD>
cudaError_t kv_launch_tc(const KvAttnArgs& a, const KvHow& p, cudaStream_t s, bool pdl) {
  if (a.c.shared)
    return p.split ? launch_attend_tc<kD, true, false>(a, p.w, s, pdl)
                   : launch_attend_tc<kD, false, false>(a, p.w, s, pdl);
  return p.split ? launch_attend_tc<kD, true, true>(a, p.w, s, pdl)
                 : launch_attend_tc<kD, false, true>(a, p.w, s, pdl);
}
template <int kD>
cudaError_t kv_launch_few(const KvAttnArgs& a, const KvHow& p, cudaStream_t s, bool pdl) {
  if (p.split) return launch_attend_few<kD, 1, true>(a, p.w, s, pdl);
  return p.w.rn == 8 ? launch_attend_few<kD, 1, false>(a, p.w, s, pdl)
                     : launch_attend_few<kD, 2, false>(a, p.w, s, pdl);
}
template <class T>
cudaError_t kv_launch(const KvAttnArgs& a, const KvHow& p, cudaStream_t s, bool pdl) {
  const unsigned rows = (unsigned)((long long)a.tokens * a.heads);
  if (p.way == KvWay::row)
    return launch_pdl(kv_attend_row_kernel<T>, dim3(rows), kRowThreads, 0, s, pdl, a);
  const int d = a.c.head_dim;
  const cudaError_t e = p.way == KvWay::few ? (d == 256   ? kv_launch_few<256>(a, p, s, pdl)
                                               : d == 128 ? kv_launch_few<128>(a, p, s, pdl)
                                                          : kv_launch_few<64>(a, p, s, pdl))
                        : d == 512 ? kv_launch_tc<512>(a, p, s, pdl)
                        : d == 256 ? kv_launch_tc<256>(a, p, s, pdl)
                        : d == 128 ? kv_launch_tc<128>(a, p, s, pdl)
                                   : kv_launch_tc<64>(a, p, s, pdl);
  if (e != cudaSuccess) return e;
  if (rows <= 4u * p.w.ctas)
    return launch_pdl(kv_join_kernel<T, 1, 4>, dim3(rows, std::max(1, d / 128)), kRowThreads,
                      kJoinParts * sizeof(float2), s, pdl, a, p.w);
  const dim3 grid((rows + 3) / 4);
  const size_t smem = 4 * kJoinParts * sizeof(float2);
  return d == 512   ? launch_pdl(kv_join_kernel<T, 4, 1>, grid, kRowThreads, smem, s, pdl, a, p.w)
         : d == 256 ? launch_pdl(kv_join_kernel<T, 2, 1>, grid, kRowThreads, smem, s, pdl, a, p.w)
                    : launch_pdl(kv_join_kernel<T, 1, 1>, grid, kRowThreads, smem, s, pdl, a, p.w);
}

}  // namespace

extern "C" {

size_t wh_kv_attention_scratch_bytes(const wh_ctx* c, const wh_kv_cache* cache, int tokens,
                                     int heads, int requests, int dtype) {
  if (!c || !cache || tokens < 1 || heads < 1 || requests < 1 || cache->kv_heads < 1 ||
      heads % cache->kv_heads != 0)
    return 0;
  KvHow p = kv_how(c, cache->head_dim, cache->kv_heads, tokens, heads, requests, dtype);
  return p.way == KvWay::row ? 256 : kv_scratch(p.w, cache->head_dim, tokens, heads, nullptr);
}

wh_status wh_kv_attention(wh_ctx* c, const wh_kv_cache* cache, const void* q, int dtype,
                          int tokens, int heads, long long q_token_stride,
                          long long q_head_stride, int requests, const int32_t* cu_q,
                          const int32_t* kv_lens, const int32_t* block_table, int max_blocks,
                          float scale, int window, int first, const float* sink, void* out,
                          long long out_token_stride, long long out_head_stride, void* scratch,
                          size_t scratch_bytes, wh_stream_t stream) {
  if (wh_status st = kv_device_check(c)) return st;
  KvAttnArgs a{};
  if (wh_status st = kv_cache_check(cache, &a.c)) return st;
  int size;
  if (!kv_dtype_size(dtype, &size)) return fail(WH_ERR_UNSUPPORTED, "attention: dtype");
  if (requests < 1 || heads < 1 || max_blocks < 1)
    return fail(WH_ERR_EMPTY_SHAPE, "attention: requests, heads, max_blocks");
  if (tokens < 0 || heads % cache->kv_heads != 0 || window < 0 || first < 0 ||
      (!cu_q && tokens != requests))
    return fail(WH_ERR_INVALID_SHAPE, "attention: tokens, heads % kv_heads, window, first");
  if (tokens == 0) return WH_OK;
  if ((long long)max_blocks * cache->page > 0x7fffffffLL)
    return fail(WH_ERR_UNSUPPORTED, "attention: max_blocks * page > 2^31 - 1");
  if ((long long)tokens * heads > 0x7fffffffLL)
    return fail(WH_ERR_UNSUPPORTED, "attention: tokens * heads > 2^31 - 1");
  if (!(scale == scale) || scale - scale != 0.0f)
    return fail(WH_ERR_INVALID_SHAPE, "attention: scale is not finite");
  if (!q || !kv_lens || !block_table || !out || !scratch)
    return fail(WH_ERR_INVALID_POINTER, "attention: null pointer");
  if (!aligned(scratch, 16))
    return fail(WH_ERR_INVALID_POINTER, "attention: scratch must be 16-byte aligned");
  if (!kv_rows_aligned(q, q_token_stride, q_head_stride, size) ||
      !kv_rows_aligned(out, out_token_stride, out_head_stride, size))
    return fail(WH_ERR_INVALID_POINTER, "attention: rows of q and out must start on 16 bytes");
  if (scratch_bytes < wh_kv_attention_scratch_bytes(c, cache, tokens, heads, requests, dtype))
    return fail(WH_ERR_SCRATCH_TOO_SMALL, "attention: scratch too small");
  a.q = q;
  a.out = out;
  a.dtype = dtype;
  a.tokens = tokens;
  a.heads = heads;
  a.group = heads / cache->kv_heads;
  a.q_token_stride = q_token_stride;
  a.q_head_stride = q_head_stride;
  a.out_token_stride = out_token_stride;
  a.out_head_stride = out_head_stride;
  a.requests = requests;
  a.cu_q = cu_q;
  a.kv_lens = kv_lens;
  a.block_table = block_table;
  a.max_blocks = max_blocks;
  a.scale = scale;
  a.window = window;
  a.first = first;
  a.sink = sink;
  a.status = c->status;
  // a window that holds every row the table can is none
  if (window >= (long long)max_blocks * cache->page) a.window = 0;
  const cudaStream_t s = (cudaStream_t)stream;
  KvHow p = kv_how(c, cache->head_dim, cache->kv_heads, tokens, heads, requests, dtype);
  if (p.way != KvWay::row)
    kv_scratch(p.w, cache->head_dim, tokens, heads, static_cast<uint8_t*>(scratch));
  if (dtype == WH_DTYPE_F32)
    WH_CUDA(kv_launch<float>(a, p, s, c->pdl()));
  else if (dtype == WH_DTYPE_BF16)
    WH_CUDA(kv_launch<__nv_bfloat16>(a, p, s, c->pdl()));
  else
    WH_CUDA(kv_launch<__half>(a, p, s, c->pdl()));
  return WH_OK;
}

}  // extern "C"
