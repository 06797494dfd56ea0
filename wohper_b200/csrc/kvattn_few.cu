// kvattn_few.cu -- attention over the paged 4-bit cache for kv heads with few
// query rows (decoding with grouped heads).
//
// A pass takes 16 query rows (8 of f32) of a kv head; more rows, up to where the
// tensor-core kernel is faster, take further passes.  With so few a cache row gives
// little work; what must not happen is that decoding its codes costs more than
// reading them.  So nothing passes through shared memory: a warp takes 16 rows
// of the cache at a time and decodes its codes in registers straight into the
// operands of mma.m16n8k16:
//   S [16 x 16 keys]  = Q K^T     Q is A (held), K^T is B: lane (g, t) of a key
//                                 tile holds key g's columns [t D/4, (t+1) D/4)
//   O^T [D x 8] += V^T P^T        V^T is A: lane (g, t) holds columns
//                                 [g D/8, (g+1) D/8) of keys 2t, 2t+1, 2t+8, 2t+9;
//                                 P^T is B, which is how S leaves its product
// (the order of the columns within a product is free, so every lane's columns are
// contiguous in memory).  Every warp keeps its own maxima, sums and O^T;
// the CTA joins them when an item ends.
//
// Measured: 16 requests x 16384 rows, 8 kv heads x 128, 4 bf16 query rows each: 71
// us with the join (f32: 77), 2.6 TB/s of codes, 56 % of the issue slots, about 410
// warp instructions for 16 rows of keys and values.  Neither is full: with four warps a
// scheduler it waits on its own loads and dependent instructions.
//
// f16 tiles, scales, query halves (kSplit: rows 8-15 of A are the low halves) and
// rows to be computed again are as in kvattn_tc.cu.  kNt: groups of 8 query rows.
#include "kvattn.cuh"

namespace wh {

constexpr int kFewWarps = 4, kFewThreads = kFewWarps * 32;
constexpr int kFewAhead = 3;  // groups beyond the next that L2 is asked for
constexpr int kFewKeys = 16;  // rows of the cache a warp takes at a time

template <int kD, int kNt, bool kSplit>
struct KvFew {
  static_assert(!kSplit || kNt == 1, "f32 rows take both halves of A");
  static constexpr int kRn = 8 * kNt;
  static constexpr int kSteps = kD / 16;   // products of S along D; 16-column tiles of O^T
  static constexpr int kA = kSplit || kNt == 2 ? 4 : 2;  // registers of A that are not zero
  static constexpr int kKBytes = kD / 8, kVBytes = kD / 16;  // of a row's codes a lane has
  static constexpr int kCtas = kD * kNt <= 128 ? 4 : kD * kNt == 256 ? 3 : 2;      // resident CTAs aimed at
  struct Misc {
    alignas(16) uint32_t q[kSteps][32][kA];  // A's registers of each product, a lane's together
    float fac[kRn];              // accumulator -> log2 score
    KvPlace at;
    float top[kFewWarps][kRn], sum[kFewWarps][kRn];
    float out_scale[kRn];
    long long out_row[kRn];
    int redo;
  };
  static constexpr int kBytes = kFewWarps * kRn * kD * 4 + (int)sizeof(Misc);
};

__device__ __forceinline__ void prefetch_l2(const uint8_t* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p) : "memory");
}
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// kBytes bytes of codes, as words
template <int kBytes>
struct KvWords {
  static constexpr int n = kBytes / 4;
  uint32_t w[n];
  __device__ __forceinline__ void load(const uint8_t* p) {
    if (kBytes == 4) {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    } else if (kBytes == 8) {
      const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = x.x;
      w[1 % n] = x.y;
    } else {
#pragma unroll
      for (int i = 0; i < n / 4; ++i) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(p) + i);
        w[(4 * i) % n] = x.x;
        w[(4 * i + 1) % n] = x.y;
        w[(4 * i + 2) % n] = x.z;
        w[(4 * i + 3) % n] = x.w;
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < n; ++i) w[i] = 0;
  }
};
// The scale of a byte in the ordinary range [109, 136] as f16 in both halves:
// 2^(b - kKvBias); other bytes go through few_scale.
__device__ __forceinline__ uint32_t few_scale_fast(uint32_t b) { return b * 0x04000400u - 108u * 0x04000400u; }
__device__ __forceinline__ bool few_ordinary(uint32_t b) { return b - 109u <= 27u; }
// Any byte: 0 and what f16 does not hold give 0; lost says which.
__device__ __forceinline__ uint32_t few_scale(uint32_t b, bool& lost) {
  const int k = int(b) - kKvBias;
  if (b == 0) return 0;
  if (k < -23 || k > 13) {
    lost = true;
    return 0;
  }
  return (k >= -14 ? uint32_t(k + 15) << 10 : 1u << (k + 24)) * 0x10001u;
}
template <int kD, int kNt, bool kSplit>
__global__ void __launch_bounds__(kFewThreads, KvFew<kD, kNt, kSplit>::kCtas)
    kv_attend_few_kernel(KvAttnArgs a, KvWork w) {
  using L = KvFew<kD, kNt, kSplit>;
  constexpr int kRn = L::kRn, kSteps = L::kSteps;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  float* merge = reinterpret_cast<float*>(smem_raw);  // [warp][row][column]
  typename L::Misc& m = *reinterpret_cast<typename L::Misc*>(smem_raw + kFewWarps * kRn * kD * 4);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const float inf = __int_as_float(0x7f800000);

  pdl_wait_prior();
  kv_place<kFewThreads>(a, w, m.at);
  int left = m.at.ntiles();
  if (left == 0) return;
  KvWalk c(m.at);
  const long long begin = m.at.begin, end = m.at.end;
  const KvCut cut(w, m.at.total);
  const bool even = a.c.page % kFewKeys == 0;  // 16 rows from a multiple of 16 share a block
  int slot1 = 0;

  while (left > 0) {
    // ---------------- a fragment: tiles [c.j, c.j + n) of the item c.it ----------------
    const int n = min(left, c.it.tiles - c.j);
    const KvItem it = c.it;
    const int rows = w.ht > 1 ? min(kRn, a.group - c.ht * kRn) : it.nt * a.group;
    const int h0 = c.kvh * a.group + c.ht * kRn;
    auto row_tok = [&](int row) { return w.ht > 1 ? 0 : row / a.group; };
    auto row_head = [&](int row) { return w.ht > 1 ? row : row % a.group; };
    if (tid == 0) m.redo = 0;
    __syncthreads();

    // The queries as A: lane (g, t) holds columns [t D/4, (t+1) D/4) of row g (and g + 8).
    // One warp makes them, all read them from shared memory: they would take a
    // fifth of the registers.
    if (warp == 0) {
#pragma unroll 1
      for (int u = 0; u < kNt; ++u) {
        const int row = g + 8 * u;
        const bool real = row < rows;
        float v[kD / 4];
        const long long off = real ? (it.t0 + row_tok(row)) * a.q_token_stride + (h0 + row_head(row)) * a.q_head_stride + t * (kD / 4)
                                   : 0;
#pragma unroll
        for (int e = 0; e < kD / 32; ++e) {
          float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
          if (real) {
            if (kSplit)
              kv_load8(static_cast<const float*>(a.q) + off + 8 * e, x);
            else if (a.dtype == WH_DTYPE_BF16)
              kv_load8(static_cast<const __nv_bfloat16*>(a.q) + off + 8 * e, x);
            else
              kv_load8(static_cast<const __half*>(a.q) + off + 8 * e, x);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) v[8 * e + i] = x[i];
        }
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < kD / 4; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const bool fin = top < 0x7f800000u;
        if (!fin) m.redo = 1;
        const int ex = max(int(top >> 23) - 127, -100);
        const float mul = fin ? exp2i(14 - ex) : 0.0f;
        if (t == 0) m.fac[row] = a.scale * kLog2e * exp2i(max(ex - 18, -126));
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int k = 0; k < 2; ++k) {  // A's registers 2k (row g) and 2k + 1 (row g + 8)
            const float x = fin ? v[4 * s + 2 * k] * mul : 0.0f, y = fin ? v[4 * s + 2 * k + 1] * mul : 0.0f;
            const __half2 hi = __floats2half2_rn(x, y);
            if (L::kA == 2) {
              m.q[s][lane][k] = half2_bits(hi);
            } else if (kSplit) {
              m.q[s][lane][(2 * k) % L::kA] = half2_bits(hi);
              m.q[s][lane][(2 * k + 1) % L::kA] = half2_bits(__floats2half2_rn(x - __low2float(hi), y - __high2float(hi)));
            } else {
              m.q[s][lane][(2 * k + u) % L::kA] = half2_bits(hi);
            }
          }
      }
    }
    __syncthreads();
    float fac[kNt];
#pragma unroll
    for (int u = 0; u < kNt; ++u) fac[u] = m.fac[g + 8 * u];

    float o[kSteps][kNt][4];  // tile i: columns g D/8 + 2i (0, 1) and + 2i + 1 (2, 3), rows 2t, 2t + 1
    float off[kNt], sum[kNt];
    bool live[kNt];
#pragma unroll
    for (int u = 0; u < kNt; ++u) {
      off[u] = sum[u] = 0.0f;
      live[u] = false;
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[s][u][e] = 0.0f;
    }

    const int p1 = it.p0 + it.nt - 1;
    const int len = kv_clip(a, c.len);
    // groups of 16 rows of the item's list: this warp takes grp0, grp0 + kFewWarps, ...
    const int past = min((c.j + n) * (kKvTile / kFewKeys), (it.seen + kFewKeys - 1) / kFewKeys);
    const int grp0 = c.j * (kKvTile / kFewKeys) + warp;
    const int groups = grp0 < past ? (past - grp0 + kFewWarps - 1) / kFewWarps : 0;
    auto key0_of = [&](int k) { return kv_key(it.head, it.start, (grp0 + k * kFewWarps) * kFewKeys); };
    const int32_t* table = a.block_table + (long long)c.r * a.max_blocks;
    // Even pages: lane i looks up the warp's group first + i, 32 at a time.  A group
    // that is not there reads block 0 and counts as not seen.
    long long lane_co = 0, lane_so = 0;  // its rows' codes and scales
    uint32_t there = 0, whole_seen = 0;  // bit i: it is there; every query sees all of it
    auto look_up = [&](int first) {
      const int k = first + lane;
      bool th = false, all = false;
      lane_co = lane_so = 0;
      if (even && k < groups) {
        const int u0 = (grp0 + k * kFewWarps) * kFewKeys, key0 = key0_of(k);
        const int pg = kv_page_of(a.c, key0), in = key0 - pg * a.c.page;
        int b = key0 < len ? table[pg] : -1;
        if (key0 < len && (b < 0 || b >= a.c.blocks)) {
          flag(a.status, WH_DEV_BADARG);
          b = -1;
        }
        th = b >= 0;
        lane_co = max(b, 0) * a.c.block_stride + (long long)in * (kD / 2);
        lane_so = max(b, 0) * a.c.scale_block_stride + (long long)in * (kD / 32);
        all = th && key0 + kFewKeys - 1 <= min(it.p0, len - 1) &&
              (u0 < it.head ? key0 + kFewKeys <= it.lo : key0 >= it.from) &&
              (a.window == 0 || key0 > p1 - a.window || key0 + kFewKeys <= a.first);
      }
      there = __ballot_sync(0xffffffffu, th);
      whole_seen = __ballot_sync(0xffffffffu, all);
    };
    // does any query see the key, which the list has in the group of its row u0
    auto seen_by_any = [&](int u0, int key) {
      return key < len && key <= p1 && (u0 < it.head ? key < it.lo : key >= it.from);
    };
    // Uneven pages: block and row of key j of the warp's group k.  The group's other keys
    // may lie in pages that no query sees and the table need not have.
    auto locate = [&](int k, int j, long long& co, long long& so) {
      const int key = key0_of(k) + j;
      const bool seen = seen_by_any((grp0 + k * kFewWarps) * kFewKeys, key);
      const int pg = kv_page_of(a.c, key);
      int b = seen ? table[pg] : -1;
      if (seen && (b < 0 || b >= a.c.blocks)) {
        flag(a.status, WH_DEV_BADARG);
        b = -1;
      }
      const int row = key - pg * a.c.page;
      co = max(b, 0) * a.c.block_stride + (long long)row * (kD / 2);
      so = max(b, 0) * a.c.scale_block_stride + (long long)row * (kD / 32);
      return b >= 0;
    };
    constexpr int kB = kD > 128 ? 2 : 1;  // scale bytes of a key that a lane needs
    // this lane's columns in the head's first row (keys: row g, values: row 2t)
    const long long head_codes = (long long)c.kvh * a.c.page * (kD / 2), head_scales = (long long)c.kvh * a.c.page * (kD / 32);
    const uint8_t* kbase = a.c.keys + head_codes + t * L::kKBytes;
    const uint8_t* ksbase = a.c.key_scales + head_scales + (kD == 64 ? t >> 1 : kD == 128 ? t : 2 * t);
    const uint8_t* vbase = a.c.values + head_codes + g * L::kVBytes;
    const uint8_t* vsbase = a.c.value_scales + head_scales + (kD == 64 ? g >> 2 : kD == 128 ? g >> 1 : g);
    KvWords<L::kKBytes> kc[2];
    uint32_t ksb[2][kB];
    KvWords<L::kVBytes> vc[4];
    uint32_t vsb[4];
    uint32_t have = 0;  // uneven pages: bit j: key 2t + (j & 1) + 8 (j >> 1) is there
    // the loads of the warp's group k, which lane i has looked up
    auto load_k = [&](int k, int i) {
      if (even) {
        const uint8_t* kp = kbase + __shfl_sync(0xffffffffu, lane_co, i) + g * (kD / 2);
        const uint8_t* sp = ksbase + __shfl_sync(0xffffffffu, lane_so, i) + g * (kD / 32);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          kc[j].load(kp + 8 * j * (kD / 2));
#pragma unroll
          for (int b = 0; b < kB; ++b) ksb[j][b] = __ldg(sp + 8 * j * (kD / 32) + b);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          long long co, so;
          locate(k, g + 8 * j, co, so);
          kc[j].load(kbase + co);
#pragma unroll
          for (int b = 0; b < kB; ++b) ksb[j][b] = __ldg(ksbase + so + b);
        }
      }
    };
    auto load_v = [&](int k, int i) {
      if (even) {
        const uint8_t* vp = vbase + __shfl_sync(0xffffffffu, lane_co, i) + 2 * t * (kD / 2);
        const uint8_t* sp = vsbase + __shfl_sync(0xffffffffu, lane_so, i) + 2 * t * (kD / 32);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          vc[j].load(vp + ((j & 1) + 8 * (j >> 1)) * (kD / 2));
          vsb[j] = __ldg(sp + ((j & 1) + 8 * (j >> 1)) * (kD / 32));
        }
      } else {
        have = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          long long co, so;
          if (locate(k, 2 * t + (j & 1) + 8 * (j >> 1), co, so)) have |= 1u << j;
          vc[j].load(vbase + co);
          vsb[j] = __ldg(vsbase + so);
        }
      }
    };
    // The loads of a group are issued half a step ahead, less than DRAM takes: L2 is
    // asked for the group kFewAhead after the next (an even page holds it in one piece).
    const uint8_t* kfetch = a.c.keys + head_codes + lane * 32;
    const uint8_t* vfetch = a.c.values + head_codes + lane * 32;
    const uint8_t* sfetch = (lane < 16 ? a.c.key_scales : a.c.value_scales) + head_scales + (lane & 15) * 32;
    auto fetch = [&](int i) {
      const long long co = __shfl_sync(0xffffffffu, lane_co, i), so = __shfl_sync(0xffffffffu, lane_so, i);
#pragma unroll
      for (int b = 0; b < kFewKeys * kD / 2; b += 1024)
        if (lane * 32 + b < kFewKeys * kD / 2) {
          prefetch_l2(kfetch + co + b);
          if (!a.c.shared) prefetch_l2(vfetch + co + b);
        }
      if ((lane & 15) * 32 < kFewKeys * kD / 32) prefetch_l2(sfetch + so);
    };

    for (int first = 0; first < groups; first += 32 - 1 - kFewAhead) {
     look_up(first);
     if (first == 0) {
       load_k(0, 0);
       load_v(0, 0);
#pragma unroll
       for (int i = 1; i <= kFewAhead; ++i)
         if (even && i < groups) fetch(i);
     }
     const int turn = min(groups - first, 32 - 1 - kFewAhead);
     for (int at = 0; at < turn; ++at) {
      const int k = first + at;
      const bool more = k + 1 < groups;
      if (even && k + 1 + kFewAhead < groups) fetch(at + 1 + kFewAhead);
      const int u0 = (grp0 + k * kFewWarps) * kFewKeys;
      const int key0 = kv_key(it.head, it.start, u0);
      // every row of the group is there and seen by every query
      const bool full = whole_seen >> at & 1;
      auto seen_any = [&](int j) { return seen_by_any(u0, key0 + j); };
      // ---- scores ----
      float s[2][4];
      uint32_t ksc[2][kB];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        bool plain = true;
#pragma unroll
        for (int e = 0; e < kB; ++e) {
          ksc[j][e] = few_scale_fast(ksb[j][e]);
          plain = plain && few_ordinary(ksb[j][e]);
        }
        if (!__all_sync(0xffffffffu, plain)) {
          bool lost = false;
#pragma unroll
          for (int e = 0; e < kB; ++e) ksc[j][e] = few_scale(ksb[j][e], lost);
          if (lost && seen_any(g + 8 * j)) m.redo = 1;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = 0.0f;
      }
      // the two key tiles in turn, so that a product need not wait for the one before
#pragma unroll
      for (int q = 0; q < kSteps; q += 2) {  // 8 codes: two products' columns
        uint32_t b[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint4 h = e2m1x8_to_f16(kc[j].w[q / 2]);
          const uint32_t scale = ksc[j][q * kB / kSteps];
          b[j][0] = hmul2_u(h.x, scale);
          b[j][1] = hmul2_u(h.y, scale);
          b[j][2] = hmul2_u(h.z, scale);
          b[j][3] = hmul2_u(h.w, scale);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t qa[4] = {0, 0, 0, 0};
          if (L::kA == 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(m.q[q + e][lane]);
            qa[0] = x.x;
            qa[2] = x.y;
          } else {
            const uint4 x = *reinterpret_cast<const uint4*>(m.q[q + e][lane]);
            qa[0] = x.x;
            qa[1] = x.y;
            qa[2] = x.z;
            qa[3] = x.w;
          }
#pragma unroll
          for (int j = 0; j < 2; ++j)
            mma_16816(s[j], qa[0], qa[1], qa[2], qa[3], b[j][2 * e], b[j][2 * e + 1]);
        }
      }
      if (more) load_k(k + 1, at + 1);
      // ---- log2 weights: x[u][j][e] of row g + 8u, key 2t + e + 8j ----
      float x[kNt][2][2];
#pragma unroll
      for (int u = 0; u < kNt; ++u)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            x[u][j][e] = fmaf(kSplit ? s[j][e] + s[j][e + 2] : s[j][e + 2 * u], fac[u], off[u]);
      if (!full) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int jj = 2 * t + e + 8 * j, key = key0 + jj;
            const bool any = seen_any(jj) && (even ? there >> at & 1 : have >> (2 * j + e) & 1);
#pragma unroll
            for (int u = 0; u < kNt; ++u) {
              const int p = it.p0 + row_tok(g + 8 * u);
              if (!(any && key <= p && (a.window == 0 || key > p - a.window || key < a.first)))
                x[u][j][e] = -inf;
            }
          }
      }
      // the maxima may lag, as long as no weight is past 2^(kLift + kLag)
      float most = -inf;
#pragma unroll
      for (int u = 0; u < kNt; ++u)
        most = fmaxf(most, fmaxf(fmaxf(x[u][0][0], x[u][0][1]), fmaxf(x[u][1][0], x[u][1][1])));
      bool stay = most <= kLift + kLag;
#pragma unroll
      for (int u = 0; u < kNt; ++u) stay = stay && live[u];
      if (!__all_sync(0xffffffffu, stay)) {
#pragma unroll
        for (int u = 0; u < kNt; ++u) {
          float top = fmaxf(fmaxf(x[u][0][0], x[u][0][1]), fmaxf(x[u][1][0], x[u][1][1]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const bool none = top == -inf;
          const float by = none ? 0.0f : fminf(kLift - top, live[u] ? 0.0f : inf);
          const float sh = ex2(live[u] ? by : 0.0f);
          live[u] = live[u] || !none;
          off[u] += by;
          sum[u] *= sh;
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) x[u][j][e] += by;
          const float sh0 = __shfl_sync(0xffffffffu, sh, 8 * t), sh1 = __shfl_sync(0xffffffffu, sh, 8 * t + 4);
#pragma unroll
          for (int i = 0; i < kSteps; ++i) {
            o[i][u][0] *= sh0;
            o[i][u][1] *= sh1;
            o[i][u][2] *= sh0;
            o[i][u][3] *= sh1;
          }
        }
      }
      uint32_t pb[kNt][2], pl[2] = {0, 0};
#pragma unroll
      for (int u = 0; u < kNt; ++u)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float p0 = ex2(x[u][j][0]), p1_ = ex2(x[u][j][1]);
          sum[u] += p0 + p1_;
          const __half2 h = __floats2half2_rn(p0, p1_);
          pb[u][j] = half2_bits(h);
          if (kSplit) pl[j] = half2_bits(__floats2half2_rn((p0 - __low2float(h)) * kLoUp, (p1_ - __high2float(h)) * kLoUp));
        }
      // ---- O^T ----
      uint32_t sc[4];
      bool plain = true;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sc[j] = few_scale_fast(vsb[j]);
        plain = plain && few_ordinary(vsb[j]);
      }
      if (!__all_sync(0xffffffffu, plain)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          bool lost = false;
          sc[j] = few_scale(vsb[j], lost);
          if (lost && seen_any(2 * t + (j & 1) + 8 * (j >> 1))) m.redo = 1;
        }
      }
      const uint32_t sc01 = __byte_perm(sc[0], sc[1], 0x5410), sc23 = __byte_perm(sc[2], sc[3], 0x5410);
#pragma unroll
      for (int i = 0; i < L::kVBytes / 4; ++i) {  // 8 columns: four tiles
        // a byte of ev / od: the codes of two keys for one even / odd column
        uint32_t ev[2], od[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t x = vc[2 * k].w[i], y = vc[2 * k + 1].w[i];
          ev[k] = (x & 0x0F0F0F0Fu) | (y << 4 & 0xF0F0F0F0u);
          od[k] = (x >> 4 & 0x0F0F0F0Fu) | (y & 0xF0F0F0F0u);
        }
        const uint4 e0 = e2m1x8_to_f16(ev[0]), e1 = e2m1x8_to_f16(ev[1]);
        const uint4 o0 = e2m1x8_to_f16(od[0]), o1 = e2m1x8_to_f16(od[1]);
        const uint32_t b0[4] = {e0.x, e0.y, e0.z, e0.w}, b1[4] = {o0.x, o0.y, o0.z, o0.w};
        const uint32_t b2[4] = {e1.x, e1.y, e1.z, e1.w}, b3[4] = {o1.x, o1.y, o1.z, o1.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t a0 = hmul2_u(b0[k], sc01), a1 = hmul2_u(b1[k], sc01);
          const uint32_t a2 = hmul2_u(b2[k], sc23), a3 = hmul2_u(b3[k], sc23);
          if (kSplit) {
            // A product of its own, added with rounding to nearest: a sum that runs through
            // the tensor core loses half of its last place with each product, always downwards.
            float z[4] = {0, 0, 0, 0};
            mma_16816(z, a0, a1, a2, a3, pl[0], pl[1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] *= 1.0f / kLoUp;
            mma_16816(z, a0, a1, a2, a3, pb[0][0], pb[0][1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[4 * i + k][0][e] += z[e];
          } else {
#pragma unroll
            for (int u = 0; u < kNt; ++u) mma_16816(o[4 * i + k][u], a0, a1, a2, a3, pb[u][0], pb[u][1]);
          }
        }
      }
      if (more) load_v(k + 1, at + 1);
     }
    }

    // ---------------- the CTA's warps joined, the rows out or to a partial slot ----------------
#pragma unroll
    for (int u = 0; u < kNt; ++u) {
      sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], 1);
      sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], 2);
      if (t == 0) {
        m.top[warp][g + 8 * u] = live[u] ? kLift - off[u] : -inf;
        m.sum[warp][g + 8 * u] = sum[u];
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kNt; ++u)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = 2 * t + e + 8 * u;
        float top = -inf;
#pragma unroll
        for (int k = 0; k < kFewWarps; ++k) top = fmaxf(top, m.top[k][row]);
        const float mine = m.top[warp][row];
        const float f = mine == -inf ? 0.0f : ex2(mine - top);
        float* to = merge + (warp * kRn + row) * kD + g * (kD / 8);
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
          *reinterpret_cast<float2*>(to + 2 * i) = make_float2(o[i][u][e] * f, o[i][u][e + 2] * f);
      }
    const bool item_first = c.at + w.lead >= begin, item_last = c.at + w.lead + it.tiles <= end;
    const bool whole = item_first && item_last;
    const int redo = m.redo;
    if (tid < rows) {
      const int row = tid;
      const int part = 2 * blockIdx.x + slot1;
      const int h = h0 + row_head(row), tok = it.t0 + row_tok(row);
      float top = -inf, l = 0.0f;
#pragma unroll
      for (int k = 0; k < kFewWarps; ++k) top = fmaxf(top, m.top[k][row]);
#pragma unroll
      for (int k = 0; k < kFewWarps; ++k) l += m.top[k][row] == -inf ? 0.0f : m.sum[k][row] * ex2(m.top[k][row] - top);
      float os = 1.0f / 16.0f;  // the f16 values are 16 times the cache's
      if (whole) {
        float z = l;
        if (a.sink) {
          const float sk = a.sink[h] * kLog2e;
          const float to = fmaxf(top, sk), base = to == -inf ? 0.0f : to;
          const float sh = top == -inf ? 0.0f : ex2(top - base);
          os *= sh;
          z = l * sh + ex2(sk - base + kLift);
        }
        os = z == 0.0f ? 0.0f : os / z;
        m.out_row[row] = tok * a.out_token_stride + h * a.out_head_stride;
      } else {
        w.part_ml[(long long)part * kRn + row] = make_float2(top, l);
        m.out_row[row] = ((long long)part * kRn + row) * kD;
        if (row == 0) w.part_redo[part] = redo;
      }
      m.out_scale[row] = os;
      if (item_first) {
        const int parts = whole ? 1 : cut.cta_of(c.at + w.lead + it.tiles - 1) - (int)blockIdx.x + 1;
        w.meta[(long long)tok * a.heads + h] = make_int4(blockIdx.x, parts, slot1 | row << 1, redo);
      }
    }
    __syncthreads();
    // rows to be computed again are left alone: out may be q, which that still reads
    const int stored = whole && redo ? 0 : rows;
    for (int i = tid; i < stored * (kD / 4); i += kFewThreads) {
      const int row = i / (kD / 4), col = i % (kD / 4) * 4;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < kFewWarps; ++k) {
        const float4 x = *reinterpret_cast<const float4*>(merge + (k * kRn + row) * kD + col);
        v.x += x.x;
        v.y += x.y;
        v.z += x.z;
        v.w += x.w;
      }
      const long long to = m.out_row[row] + col;
      const float by = m.out_scale[row];
      if (!whole)
        kv_store4(w.part_o + to, v, by);
      else if (kSplit)
        kv_store4(static_cast<float*>(a.out) + to, v, by);
      else if (a.dtype == WH_DTYPE_BF16)
        kv_store4(static_cast<__nv_bfloat16*>(a.out) + to, v, by);
      else
        kv_store4(static_cast<__half*>(a.out) + to, v, by);
    }
    slot1 = 1;
    left -= n;
    if (left > 0) c.next(a, w);
    __syncthreads();
  }
  pdl_launch_dependents();
}

template <int kD, int kNt, bool kSplit>
static cudaError_t launch_attend_few(const KvAttnArgs& a, const KvWork& w, cudaStream_t s, bool pdl) {
  using L = KvFew<kD, kNt, kSplit>;
  if (w.rn != L::kRn) return cudaErrorInvalidValue;
  const cudaError_t e = ensure_smem(kv_attend_few_kernel<kD, kNt, kSplit>, L::kBytes);
  if (e != cudaSuccess) return e;
  return launch_pdl(kv_attend_few_kernel<kD, kNt, kSplit>, dim3(w.ctas), kFewThreads, L::kBytes, s, pdl, a, w);
}

}  // namespace wh
