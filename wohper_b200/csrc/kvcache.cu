// kvcache.cu -- the paged 4-bit key/value cache: one step's block tables and
// slots (kv_plan_kernel, kv_slots_kernel), quantised writes (kv_append_kernel)
// and reads (kv_gather_kernel), with their C entry points.  The attention over
// the cache is kvattn.cu.
//
// A row is E2M1 codes and one UE8M0 scale per 32 of them; inside a block the
// rows of one kv head are contiguous ([kv head][row][bytes]), so that a kernel
// that walks one head reads whole pages in order.
#include <cuda_bf16.h>

#include "kvcache.cuh"

namespace wh {

// ---------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------
struct KvPlanArgs {
  int requests, page, max_blocks, tokens, capacity;
  const int32_t* kv_lens;
  const int32_t* q_lens;
  const uint8_t* finished;
  int32_t* block_table;
  int32_t* free_blocks;
  const int32_t* free_top;
  int32_t* free_top_out;
  int32_t* kv_lens_out;
  int32_t* cu_q;
  int64_t* slots;
  int32_t* positions;
  int32_t* token_requests;
  int32_t* page_base;  // scratch [requests]: stack index of the request's first new page
  uint32_t* status;
};

constexpr int kPlanThreads = 1024;
constexpr int kPlanShared = 4096;  // requests whose cu_q the planning CTA keeps in shared memory
// Tokens up to which the planning CTA finds the slots itself.  A second launch
// over many CTAs pays only when one CTA would loop for longer than a launch
// takes.
constexpr int kPlanInlineTokens = 4096;

__device__ __forceinline__ int ceil_div(int a, int b) { return a / b + (a % b != 0); }

// Where token t of the step goes.  cu: cu_q (global or shared memory).
__device__ __forceinline__ void kv_slot_of(const KvPlanArgs& a, const int32_t* cu, int t) {
  if (t >= cu[a.requests]) {
    a.slots[t] = -1;
    a.positions[t] = -1;
    a.token_requests[t] = -1;
    return;
  }
  int lo = 0, hi = a.requests - 1;  // the last r with cu[r] <= t
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid - 1;
  }
  const int r = lo;
  const int old = a.kv_lens_out[r] - (cu[r + 1] - cu[r]);
  const int pos = old + (t - cu[r]);
  const int held = ceil_div(old, a.page);
  const int pg = pos / a.page, row = pos - pg * a.page;
  int32_t* entry = a.block_table + (long long)r * a.max_blocks + pg;
  int block;
  if (pg < held) {
    block = *entry;
  } else {
    block = a.free_blocks[a.page_base[r] - (pg - held)];
    if (row == 0) *entry = block;  // the page's first row is one of the new tokens
  }
  if (block < 0) flag(a.status, WH_DEV_BADARG);
  a.slots[t] = block < 0 ? -1 : (int64_t)block * a.page + row;
  a.positions[t] = pos;
  a.token_requests[t] = r;
}

// One CTA.  Thread i owns a contiguous run of requests; three block-wide sums
// (blocks freed, blocks needed, new tokens) decide whether the step fits, and
// the same scan gives each request its place on the free stack and in the
// tokens.  A few thousand lengths are one load per thread: the kernel is the
// latency of a handful of dependent loads and two barriers (32 requests: 3.9 us;
// 1000 with prompts, the second kernel included: 9.8 us).
__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(KvPlanArgs a, int inline_tokens) {
  __shared__ long long part[3][32];
  __shared__ int32_t scu[kPlanShared + 1];
  __shared__ int bad_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool small = a.requests <= kPlanShared;
  if (tid == 0) bad_s = 0;
  pdl_wait_prior();
  const int per = ceil_div(a.requests, kPlanThreads);
  const int r0 = tid * per;
  const int top = *a.free_top;
  __syncthreads();

  auto read = [&](int r, int& old, int& q, bool& fin) {
    old = a.kv_lens[r];
    q = a.q_lens[r];
    fin = a.finished && a.finished[r];
  };
  long long sum[3] = {0, 0, 0};  // freed, fresh, q
  bool bad = false;
  for (int i = 0; i < per; ++i) {
    const int r = r0 + i;
    if (r >= a.requests) break;
    int old, q;
    bool fin;
    read(r, old, q, fin);
    const long long room = (long long)a.max_blocks * a.page;
    if (old < 0 || q < 0 || (fin && q != 0) || (long long)old + q > room) {
      bad = true;
      continue;
    }
    const int held = ceil_div(old, a.page);
    if (fin)
      sum[0] += held;
    else
      sum[1] += ceil_div(old + q, a.page) - held;
    sum[2] += q;
  }
  if (bad) bad_s = 1;
  // exclusive scan of the three sums over the threads
  long long ex[3], tot[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    long long v = sum[k];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long p = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += p;
    }
    if (lane == 31) part[k][warp] = v;
    ex[k] = v - sum[k];
  }
  __syncthreads();
  if (warp < 3) {
    long long v = part[warp][lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long p = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += p;
    }
    part[warp][lane] = v;  // inclusive over warps
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    if (warp > 0) ex[k] += part[k][warp - 1];
    tot[k] = part[k][31];
  }
  const bool ok = !bad_s && top >= 0 && top <= a.capacity && top + tot[0] <= a.capacity &&
                  tot[1] <= top + tot[0] && tot[2] <= a.tokens;
  if (tid == 0) {
    if (!ok) flag(a.status, WH_DEV_BADARG);
    *a.free_top_out = ok ? (int)(top + tot[0] - tot[1]) : top;
    const int n = ok ? (int)tot[2] : 0;
    a.cu_q[a.requests] = n;
    if (small) scu[a.requests] = n;
  }
  for (int i = 0; i < per; ++i) {  // per is uniform: every lane takes part in the ballots
    const int r = r0 + i;
    int old = 0, q = 0, held = 0;
    bool fin = false;
    if (r < a.requests) {
      read(r, old, q, fin);
      if (ok) held = ceil_div(old, a.page);
      const int start = ok ? (int)ex[2] : 0;
      a.cu_q[r] = start;
      if (small) scu[r] = start;
      a.kv_lens_out[r] = !ok ? old : fin ? 0 : old + q;
      if (ok) a.page_base[r] = (int)(top + tot[0] - 1 - ex[1]);
    }
    // a warp pushes the blocks of its lanes' finished requests, one request at a time
    const bool push = ok && fin && held > 0;
    for (unsigned m = __ballot_sync(0xffffffffu, push); m; m &= m - 1) {
      const int src = __ffs(m) - 1;
      const int n = __shfl_sync(0xffffffffu, held, src);
      const int rr = __shfl_sync(0xffffffffu, r, src);
      const long long at = top + __shfl_sync(0xffffffffu, ex[0], src);
      for (int p = lane; p < n; p += 32)
        a.free_blocks[at + p] = a.block_table[(long long)rr * a.max_blocks + p];
    }
    if (ok && r < a.requests) {
      if (fin)
        ex[0] += held;
      else
        ex[1] += ceil_div(old + q, a.page) - held;
      ex[2] += q;
    }
  }
  pdl_launch_dependents();
  if (!inline_tokens) return;
  __syncthreads();
  for (int t = tid; t < a.tokens; t += kPlanThreads) kv_slot_of(a, small ? scu : a.cu_q, t);
}

__global__ void __launch_bounds__(256) kv_slots_kernel(KvPlanArgs a) {
  pdl_wait_prior();
  const int t = blockIdx.x * blockDim.x + threadIdx.x;
  if (t < a.tokens) kv_slot_of(a, a.cu_q, t);
}

template <class K, class... A>
static cudaError_t launch_pdl(K* kernel, dim3 grid, int threads, size_t smem, cudaStream_t s,
                              bool pdl, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
struct KvAppendArgs {
  KvCacheDev c;
  const int64_t* slots;
  int rows;
  const void* x[2];           // new keys, new values
  long long row_stride[2], head_stride[2];  // elements
  uint32_t* status;
};

// The least k with amax <= 6 * 2^k = 1.5 * 2^(k+2): the exponent less two, one
// more where the mantissa is past 1.5; clamped to [-126, 125] so that 2^k and
// 2^-k are normal floats (values past 6 * 2^125 saturate).
__device__ __forceinline__ int e2m1_block_exp(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int k = int(u >> 23) - 127 - 2 + int((u & 0x7FFFFFu) > 0x400000u);
  return max(-126, min(125, k));
}
// Two values -> one byte of codes (lo in the low nibble), to nearest, ties to
// even, saturated at +-6.
__device__ __forceinline__ uint32_t e2m1x2_rn(float lo, float hi) {
  uint32_t r;
  asm("{ .reg .b8 t; cvt.rn.satfinite.e2m1x2.f32 t, %1, %2; cvt.u32.u8 %0, t; }"
      : "=r"(r)
      : "f"(hi), "f"(lo));
  return r;
}

// How a CTA walks rows: a row is `units` lanes of 8 values (all heads), `side`
// rows lie side by side in the CTA, and a thread takes `kEach` of them, whose
// loads are all issued before the first is used.
constexpr int kRowCta = 256;
struct KvRows {
  int units, wide, side;  // wide: units that one pass of the CTA covers
  int ctas;
};
static KvRows kv_rows(const KvCacheDev& c, int rows, int each) {
  KvRows r;
  r.units = c.kv_heads * (c.head_dim / 8);
  r.wide = std::min(r.units, kRowCta);
  r.side = kRowCta / r.wide;
  r.ctas = (rows + r.side * each - 1) / (r.side * each);
  return r;
}
struct KvSlot {
  int block, row;  // block -1: not there
};
__device__ __forceinline__ KvSlot kv_slot(const KvCacheDev& c, int64_t slot, uint32_t* status) {
  if (slot < 0) return {-1, 0};
  if (slot >= (int64_t)c.blocks * c.page) {
    flag(status, WH_DEV_BADARG);
    return {-1, 0};
  }
  KvSlot s;
  s.block = c.page_shift >= 0 ? int(slot >> c.page_shift) : int(slot / c.page);
  s.row = int(slot - (int64_t)s.block * c.page);
  return s;
}

// Four lanes take a block of 32 values, 8 each: wide contiguous loads, the
// block's maximum by two shuffles, 4 bytes of codes a lane, the scale byte from
// the first.  Reads 32 values and writes 17 bytes a block; bound by the latency of
// scattered rows: 8191 rows of 8 x 128 keys and values about 20 us (2.1 TB/s), 32
// rows 3 us.
constexpr int kAppendEach = 2;
template <class T>
__global__ void __launch_bounds__(kRowCta, 5) kv_append_kernel(KvAppendArgs a, KvRows r) {
  constexpr int kEach = kAppendEach;
  pdl_wait_prior();
  const bool values = blockIdx.y;
  const int side = threadIdx.x / r.wide;
  if (side >= r.side) return;  // r.wide is a multiple of 4: whole groups leave
  const unsigned group = 0xFu << (threadIdx.x & 28);
  const long long row_stride = values ? a.row_stride[1] : a.row_stride[0];
  const long long head_stride = values ? a.head_stride[1] : a.head_stride[0];
  const T* x = static_cast<const T*>(values ? a.x[1] : a.x[0]);
  uint8_t* codes = values ? a.c.values : a.c.keys;
  uint8_t* scales = values ? a.c.value_scales : a.c.key_scales;
  const int row0 = blockIdx.x * r.side * kEach + side;
  const int parts = a.c.head_dim / 8;
  for (int u = threadIdx.x - side * r.wide; u < r.units; u += r.wide) {
    const int head = u / parts, part = u - head * parts;
    // the rows' values and slots are asked for together
    KvRaw8<T> raw[kEach];
    int64_t slot[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int row = min(row0 + k * r.side, a.rows - 1);
      slot[k] = row0 + k * r.side < a.rows ? a.slots[row] : -1;
      raw[k].load(x + row * row_stride + head * head_stride + part * 8);
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const KvSlot at = kv_slot(a.c, slot[k], a.status);
      if (at.block < 0) continue;  // the four lanes alike
      float v[8];
      raw[k].widen(v);
      float m = 0.0f;
      bool fin = true;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        m = fmaxf(m, fabsf(v[j]));
        fin &= isfinite(v[j]);
      }
      m = fmaxf(m, __shfl_xor_sync(group, m, 1));
      m = fmaxf(m, __shfl_xor_sync(group, m, 2));
      fin = __all_sync(group, fin);
      const int e = e2m1_block_exp(m);
      const uint32_t byte = !fin ? 255u : m == 0.0f ? 0u : uint32_t(e + 127);
      const float inv = exp2i(-e);
      uint32_t w = 0;
      if (fin) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w |= e2m1x2_rn(__fmul_rn(v[2 * j], inv), __fmul_rn(v[2 * j + 1], inv)) << (8 * j);
      }
      const long long row = (long long)head * a.c.page + at.row;
      reinterpret_cast<uint32_t*>(codes + at.block * a.c.block_stride + row * (a.c.head_dim / 2))[part] = w;
      if ((part & 3) == 0)
        scales[at.block * a.c.scale_block_stride + row * (a.c.head_dim / 32) + (part >> 2)] = (uint8_t)byte;
    }
  }
}

// ---------------------------------------------------------------------------
// gather
// ---------------------------------------------------------------------------
struct KvGatherArgs {
  KvCacheDev c;
  const int64_t* slots;
  int rows;
  void* out[2];
  uint32_t* status;
};

// A lane takes 8 values: 4 bytes of codes and the block's scale byte in, one
// 16-byte store (two for f32) out, all contiguous over a row.  9600 rows of 8 x 128
// keys and values to bf16: about 14 us (3.6 TB/s).
constexpr int kGatherEach = 4;
template <class T>
__global__ void __launch_bounds__(kRowCta) kv_gather_kernel(KvGatherArgs a, KvRows r) {
  constexpr int kEach = kGatherEach;
  pdl_wait_prior();
  const bool values = blockIdx.y;
  const int side = threadIdx.x / r.wide;
  if (side >= r.side) return;
  const uint8_t* codes = values ? a.c.values : a.c.keys;
  const uint8_t* scales = values ? a.c.value_scales : a.c.key_scales;
  T* out = static_cast<T*>(values ? a.out[1] : a.out[0]);
  const int row0 = blockIdx.x * r.side * kEach + side;
  KvSlot at[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int row = row0 + k * r.side;
    at[k] = row < a.rows ? kv_slot(a.c, a.slots[row], a.status) : KvSlot{-1, 0};
  }
  const int parts = a.c.head_dim / 8;
  for (int u = threadIdx.x - side * r.wide; u < r.units; u += r.wide) {
    const int head = u / parts, part = u - head * parts;
    uint32_t w[kEach], sb[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      w[k] = sb[k] = 0;
      if (at[k].block >= 0) {
        const long long row = (long long)head * a.c.page + at[k].row;
        w[k] = __ldg(reinterpret_cast<const uint32_t*>(codes + at[k].block * a.c.block_stride + row * (a.c.head_dim / 2)) + part);
        sb[k] = __ldg(scales + at[k].block * a.c.scale_block_stride + row * (a.c.head_dim / 32) + (part >> 2));
      }
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int row = row0 + k * r.side;
      if (row >= a.rows) continue;
      float v[8];
      kv_decode8(w[k], sb[k], v);
      kv_store8(out + ((long long)row * r.units + u) * 8, v);
    }
  }
}

}  // namespace wh

// ---------------------------------------------------------------------------
// C entry points
// ---------------------------------------------------------------------------
namespace {
using namespace wh;

wh_status kv_cache_check(const wh_kv_cache* c, KvCacheDev* out) {
  if (!c) return fail(WH_ERR_INVALID_POINTER, "cache is null");
  if (c->blocks < 1 || c->page < 1 || c->kv_heads < 1 || c->head_dim < 1)
    return fail(WH_ERR_EMPTY_SHAPE, "cache: blocks, page, kv_heads, head_dim");
  if (c->head_dim % 32 != 0) return fail(WH_ERR_INVALID_SHAPE, "cache: head_dim % 32 != 0");
  if (c->head_dim > 512) return fail(WH_ERR_UNSUPPORTED, "cache: head_dim > 512");
  const long long rows = (long long)c->kv_heads * c->page;
  if (rows > 0x7fffffffLL || c->page > (1 << 20))
    return fail(WH_ERR_UNSUPPORTED, "cache: block too large");
  const long long dense = rows * (c->head_dim / 2), dense_s = rows * (c->head_dim / 32);
  if (!c->keys || !c->key_scales || !c->values != !c->value_scales)
    return fail(WH_ERR_INVALID_POINTER, "cache: null pointer");
  if (!aligned(c->keys, 16) || !aligned(c->values, 16) || !aligned(c->key_scales, 16) ||
      !aligned(c->value_scales, 16))
    return fail(WH_ERR_INVALID_POINTER, "cache: arrays must be 16-byte aligned");
  if ((c->block_stride && (c->block_stride < dense || c->block_stride % 16)) ||
      (c->scale_block_stride &&
       (c->scale_block_stride < dense_s || c->scale_block_stride % (c->head_dim / 32))))
    return fail(WH_ERR_INVALID_SHAPE, "cache: block stride");
  out->blocks = c->blocks;
  out->page = c->page;
  out->kv_heads = c->kv_heads;
  out->head_dim = c->head_dim;
  out->keys = c->keys;
  out->key_scales = c->key_scales;
  out->values = c->values ? c->values : c->keys;
  out->value_scales = c->value_scales ? c->value_scales : c->key_scales;
  out->shared = c->values == nullptr;
  out->page_shift = -1;
  for (int k = 0; k <= 20; ++k)
    if (c->page == 1 << k) out->page_shift = k;
  out->block_stride = c->block_stride ? c->block_stride : dense;
  out->scale_block_stride = c->scale_block_stride ? c->scale_block_stride : dense_s;
  return WH_OK;
}

// The kernels launch on the current device, which has to be the context's.
wh_status kv_device_check(const wh_ctx* c) {
  if (!c) return fail(WH_ERR_INVALID_POINTER, "ctx is null");
  int cur = -1;
  WH_CUDA(cudaGetDevice(&cur));
  if (cur != c->device) return fail(WH_ERR_CUDA, "the context's device is not the current device");
  return WH_OK;
}

bool kv_dtype_size(int dtype, int* size) {
  *size = dtype == WH_DTYPE_F32 ? 4 : 2;
  return dtype == WH_DTYPE_F32 || dtype == WH_DTYPE_BF16 || dtype == WH_DTYPE_F16;
}
// rows of head_dim elements at these strides (elements) all start on 16 bytes
bool kv_rows_aligned(const void* p, long long s0, long long s1, int size) {
  return aligned(p, 16) && (s0 * size) % 16 == 0 && (s1 * size) % 16 == 0;
}
}  // namespace

extern "C" {

size_t wh_kv_plan_scratch_bytes(int requests) {
  return requests > 0 ? align256(sizeof(int32_t) * (size_t)requests) : 0;
}

wh_status wh_kv_plan(wh_ctx* c, int requests, int page, int max_blocks, int tokens,
                     const int32_t* kv_lens, const int32_t* q_lens, const uint8_t* finished,
                     int32_t* block_table, int32_t* free_blocks, int capacity,
                     const int32_t* free_top, int32_t* free_top_out, int32_t* kv_lens_out,
                     int32_t* cu_q, int64_t* slots, int32_t* positions, int32_t* token_requests,
                     void* scratch, size_t scratch_bytes, wh_stream_t stream) {
  if (wh_status st = kv_device_check(c)) return st;
  if (requests < 1 || page < 1 || max_blocks < 1)
    return fail(WH_ERR_EMPTY_SHAPE, "plan: requests, page, max_blocks");
  if (tokens < 0 || capacity < 0) return fail(WH_ERR_INVALID_SHAPE, "plan: tokens, capacity");
  if ((long long)max_blocks * page > 0x7fffffffLL || page > (1 << 20))
    return fail(WH_ERR_UNSUPPORTED, "plan: max_blocks * page > 2^31 - 1");
  if (scratch_bytes < sizeof(int32_t) * (size_t)requests)
    return fail(WH_ERR_SCRATCH_TOO_SMALL, "plan: scratch too small");
  if (!kv_lens || !q_lens || !block_table || !free_blocks || !free_top || !free_top_out ||
      !kv_lens_out || !cu_q || !scratch ||
      (tokens > 0 && (!slots || !positions || !token_requests)))
    return fail(WH_ERR_INVALID_POINTER, "plan: null pointer");
  if (free_top == free_top_out)
    return fail(WH_ERR_INVALID_POINTER, "plan: free_top_out may not be free_top");
  const KvPlanArgs a{requests,   page,         max_blocks,  tokens,      capacity,
                     kv_lens,    q_lens,       finished,    block_table, free_blocks,
                     free_top,   free_top_out, kv_lens_out, cu_q,        slots,
                     positions,  token_requests, static_cast<int32_t*>(scratch), c->status};
  const bool inl = tokens <= kPlanInlineTokens;
  const cudaStream_t s = (cudaStream_t)stream;
  WH_CUDA(launch_pdl(kv_plan_kernel, dim3(1), kPlanThreads, 0, s, c->pdl(), a, inl ? 1 : 0));
  if (!inl)
    WH_CUDA(launch_pdl(kv_slots_kernel, dim3((tokens + 255) / 256), 256, 0, s, c->pdl(), a));
  return WH_OK;
}

wh_status wh_kv_append(wh_ctx* c, const wh_kv_cache* cache, const int64_t* slots, int rows,
                       const void* k, const void* v, int dtype, long long k_row_stride,
                       long long k_head_stride, long long v_row_stride, long long v_head_stride,
                       wh_stream_t stream) {
  if (wh_status st = kv_device_check(c)) return st;
  KvAppendArgs a{};
  if (wh_status st = kv_cache_check(cache, &a.c)) return st;
  int size;
  if (!kv_dtype_size(dtype, &size)) return fail(WH_ERR_UNSUPPORTED, "append: dtype");
  if (rows < 0) return fail(WH_ERR_INVALID_SHAPE, "append: rows");
  if (rows == 0) return WH_OK;
  if (!slots || !k || (v != nullptr) != (cache->values != nullptr))
    return fail(WH_ERR_INVALID_POINTER, "append: slots, k, v (v exactly when the cache has values)");
  if (!kv_rows_aligned(k, k_row_stride, k_head_stride, size) ||
      (v && !kv_rows_aligned(v, v_row_stride, v_head_stride, size)))
    return fail(WH_ERR_INVALID_POINTER, "append: rows must start on 16 bytes");
  const KvRows r = kv_rows(a.c, rows, kAppendEach);
  a.slots = slots;
  a.rows = rows;
  a.x[0] = k;
  a.x[1] = v;
  a.row_stride[0] = k_row_stride;
  a.row_stride[1] = v_row_stride;
  a.head_stride[0] = k_head_stride;
  a.head_stride[1] = v_head_stride;
  a.status = c->status;
  const dim3 grid(r.ctas, v ? 2 : 1);
  const cudaStream_t s = (cudaStream_t)stream;
  if (dtype == WH_DTYPE_F32)
    WH_CUDA(launch_pdl(kv_append_kernel<float>, grid, kRowCta, 0, s, c->pdl(), a, r));
  else if (dtype == WH_DTYPE_BF16)
    WH_CUDA(launch_pdl(kv_append_kernel<__nv_bfloat16>, grid, kRowCta, 0, s, c->pdl(), a, r));
  else
    WH_CUDA(launch_pdl(kv_append_kernel<__half>, grid, kRowCta, 0, s, c->pdl(), a, r));
  return WH_OK;
}

wh_status wh_kv_gather(wh_ctx* c, const wh_kv_cache* cache, const int64_t* slots, int rows,
                       void* k, void* v, int dtype, wh_stream_t stream) {
  if (wh_status st = kv_device_check(c)) return st;
  KvGatherArgs a{};
  if (wh_status st = kv_cache_check(cache, &a.c)) return st;
  int size;
  if (!kv_dtype_size(dtype, &size)) return fail(WH_ERR_UNSUPPORTED, "gather: dtype");
  if (rows < 0) return fail(WH_ERR_INVALID_SHAPE, "gather: rows");
  if (rows == 0) return WH_OK;
  if (!slots || !k || (v && !cache->values))
    return fail(WH_ERR_INVALID_POINTER, "gather: slots, k (v only where the cache has values)");
  if (!aligned(k, 16) || !aligned(v, 16))
    return fail(WH_ERR_INVALID_POINTER, "gather: outputs must be 16-byte aligned");
  const KvRows r = kv_rows(a.c, rows, kGatherEach);
  a.slots = slots;
  a.rows = rows;
  a.out[0] = k;
  a.out[1] = v;
  a.status = c->status;
  const dim3 grid(r.ctas, v ? 2 : 1);
  const cudaStream_t s = (cudaStream_t)stream;
  if (dtype == WH_DTYPE_F32)
    WH_CUDA(launch_pdl(kv_gather_kernel<float>, grid, kRowCta, 0, s, c->pdl(), a, r));
  else if (dtype == WH_DTYPE_BF16)
    WH_CUDA(launch_pdl(kv_gather_kernel<__nv_bfloat16>, grid, kRowCta, 0, s, c->pdl(), a, r));
  else
    WH_CUDA(launch_pdl(kv_gather_kernel<__half>, grid, kRowCta, 0, s, c->pdl(), a, r));
  return WH_OK;
}

}  // extern "C"
