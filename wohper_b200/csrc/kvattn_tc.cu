// kvattn_tc.cu -- attention over the paged 4-bit cache on the 5th-generation
// tensor cores.
//
// Both products run with the cache as the tall operand, so that a handful of
// query rows costs the tensor core a handful of columns:
//   S^T [64 keys x kN]  = K [64 x D] Q^T          (M = 64)
//   O^T [D x kN]       += V^T [D x 64] P^T        (M = 128, D / 128 blocks)
// K and V are decoded once per tile into f16 in shared memory (rows of 64
// columns, 128-byte swizzle).  The same bytes serve as the K-major operand of
// the first product and, where the values are the keys, as the MN-major
// operand of the second.
//
// f16 holds a code times its scale exactly over 36 octaves of scales (2^-27 to
// 2^9; kept as 16 times the value, scale bytes 100..136).  Items that meet
// another byte, a not-finite query or a not-finite block are marked and computed again row by row in f32.
// A query row is brought to a largest value in [2^14, 2^15) by a power of two;
// 16-bit queries are then one f16 exactly, f32 queries are the sum of two
// (kSplit: columns 2i and 2i + 1), which keeps 22 bits.  Weights are
// 2^(s - m + kLift) with a maximum m that may lag by kLag, so at most 2^15;
// one f16 for 16-bit queries (11 bits), two for f32.  Sums are f32.
//
// Warps: 0-3 softmax and epilogue (TMEM lane quadrants), 4-11 decode, 12 MMA,
// 13 addresses (walks the work list, looks up blocks).
#include "kvattn.cuh"
#include "tc.cuh"

namespace wh {

constexpr int kTcSoft = 4, kTcDec = 8;
constexpr int kTcMma = kTcSoft + kTcDec, kTcAddr = kTcMma + 1;
constexpr int kTcThreads = (kTcAddr + 1) * 32;
constexpr int kTcInfo = 8;   // tiles the address warp may run ahead
constexpr int kTcFrag = 4;   // fragments whose query factors and redo marks are kept
constexpr int kTcRing = 4;   // most ring stages
constexpr float kLag = 6.0f;   // log2 units that the running maximum may lag behind
constexpr float kLift = 9.0f;  // weights are held as 2^(s - m + kLift) <= 2^15
constexpr int kKvBias = 123;   // scale byte b stands for 2^(b - kKvBias) in the f16 tiles

enum : int {
  kFragFirst = 1,   // the CTA's first tile of this item
  kFragLast = 2,    // the CTA's last tile of this item
  kTileMasked = 4,  // some row of the tile is not seen by every query
  kItemFirst = 8,   // the item's first tile is in this CTA
  kItemLast = 16,   // the item's last tile is in this CTA
  kSlot1 = 32,      // partial slot 1 (the fragment does not begin the CTA's range)
};

struct KvTileInfo {
  int2 row[kKvTile];  // block (-1: not seen) and row in the block
  long long end;      // the tile after the item's last one
  int r, t0, nt, p0, kvh, ht, head, start, u0, flags;
};

template <int kD, int kN, bool kSplit>
struct KvTc {
  static constexpr int kRn = kSplit ? kN / 2 : kN;  // query rows
  static constexpr int kChunks = kD / 64;
  static constexpr int kBlocks = kD >= 128 ? kD / 128 : 1;  // 128-row blocks of O^T
  static constexpr int kQBytes = kChunks * kN * 128;
  static constexpr int kTileBytes = kD * 128;
  static constexpr int kPBytes = kKvTile * 128;
  static constexpr int kIt = kD >= 128 ? kD / 128 : 1;  // 32-code units a decode lane takes
  static constexpr int kMax = kN / 4 / (kSplit ? 2 : 1);  // query rows a softmax thread holds
  static constexpr uint32_t kTmemO = 0, kTmemS = kBlocks * kN;
  static constexpr uint32_t kTmemNeed = kBlocks * kN + 2 * kN;
  static constexpr uint32_t kTmemCols = kTmemNeed <= 64 ? 64 : kTmemNeed <= 128 ? 128
                                        : kTmemNeed <= 256 ? 256 : 512;
  static_assert(kTmemNeed <= 512, "TMEM");
  struct Misc {
    KvTileInfo info[kTcInfo];
    float fac[kTcFrag][kRn];   // accumulator -> log2 score, per query row
    float red[2][kTcSoft][kRn];
    float out_scale[kRn];
    float shrink[kRn];
    int redo[kTcFrag];
    int row_tok[kRn];          // token (within the item) and head (within the kv head's) of a row
    int row_head[kRn];
    uint64_t info_full[kTcInfo], info_empty[kTcInfo];
    uint64_t k_full[kTcRing], k_empty[kTcRing], v_full[kTcRing], v_empty[kTcRing];
    uint64_t s_full[2], s_empty[2], p_full[2], p_empty[2];
    uint64_t q_full[kTcFrag], q_empty, o_empty, all_done;
    long long part[16];
    long long total, first_off;
    int first_r;
    uint32_t tmem;
  };
  static constexpr size_t fixed_bytes() { return kQBytes + 2 * kPBytes + sizeof(Misc) + 1024; }
  static size_t bytes(int ks, int vs) { return fixed_bytes() + size_t(ks + vs) * kTileBytes; }
};

// 8 codes (code i in bits 4i..4i+3) -> 8 f16 with the high bytes of their
// magnitudes looked up in t0 (codes 0-3) and t1 (4-7); every value has a zero low byte.
__device__ __forceinline__ uint4 e2m1x8_to_f16(uint32_t w, uint32_t t0, uint32_t t1) {
  const uint32_t mag = w & 0x77777777u, w4 = w << 4;
  uint32_t lo = __byte_perm(t0, t1, mag), hi = __byte_perm(t0, t1, mag >> 16);
  lo |= __byte_perm(w4, w, 0x5140) & 0x80808080u;  // sign of code i at bit 7 of byte i
  hi |= __byte_perm(w4, w, 0x7362) & 0x80808080u;
  return make_uint4(__byte_perm(lo, 0, 0x1404), __byte_perm(lo, 0, 0x3424),
                    __byte_perm(hi, 0, 0x1404), __byte_perm(hi, 0, 0x3424));
}
__device__ __forceinline__ uint32_t hmul2_u(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// One block of 32 codes into half a 128-byte row of a tile (16-byte pieces
// col0 .. col0 + 3, swizzled by the row).  seen = false writes zeros.
// Returns false where the scale byte has no exact f16 form.
__device__ __forceinline__ bool decode_block(const uint4& c, uint32_t sb, bool seen, uint8_t* row,
                                             int col0, int r7) {
  const int k = int(sb) - kKvBias;
  const bool zero = !seen || sb == 0;
  const bool in = zero || (k >= -23 && k <= 13);
  const bool sub = !zero && in && k < -13;  // 2^k times a code may be subnormal: multiply
  // high bytes of 0 0.5 1 1.5 and 2 3 4 6; 2^k adds k to the exponents of all but 0
  const uint32_t step = sub ? 0u : uint32_t(k);
  const uint32_t t0 = zero || !in ? 0u : 0x3E3C3800u + step * 0x04040400u;
  const uint32_t t1 = zero || !in ? 0u : 0x46444240u + step * 0x04040404u;
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  uint4 v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = e2m1x8_to_f16(w[j], t0, t1);
  if (__any_sync(__activemask(), sub)) {
    // 2^k as f16: subnormal below 2^-14
    const uint32_t m = !sub ? 0x3C00u : k >= -14 ? uint32_t(k + 15) << 10 : 1u << (k + 24);
    const uint32_t mm = m | m << 16;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j].x = hmul2_u(v[j].x, mm);
      v[j].y = hmul2_u(v[j].y, mm);
      v[j].z = hmul2_u(v[j].z, mm);
      v[j].w = hmul2_u(v[j].w, mm);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *reinterpret_cast<uint4*>(row + (((col0 + j) ^ r7) << 4)) = v[j];
  return in;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_bits(__half2 h) {
  return *reinterpret_cast<uint32_t*>(&h);
}
// A bounded wait that a whole warp takes together: a lane that times out takes
// the others with it.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t phase, uint32_t* status) {
  return __all_sync(0xffffffffu, mbar_wait(bar, phase, status));
}
__device__ __forceinline__ void kv_load8_any(const KvAttnArgs& a, long long at, float (&v)[8]) {
  if (a.dtype == WH_DTYPE_F32)
    kv_load8(reinterpret_cast<const float*>(a.q) + at, v);
  else if (a.dtype == WH_DTYPE_BF16)
    kv_load8(reinterpret_cast<const __nv_bfloat16*>(a.q) + at, v);
  else
    kv_load8(reinterpret_cast<const __half*>(a.q) + at, v);
}
__device__ __forceinline__ void kv_store_any(const KvAttnArgs& a, long long at, float v) {
  if (a.dtype == WH_DTYPE_F32)
    reinterpret_cast<float*>(a.out)[at] = v;
  else if (a.dtype == WH_DTYPE_BF16)
    reinterpret_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
  else
    reinterpret_cast<__half*>(a.out)[at] = __float2half_rn(v);
}

// A row's scale bytes, 32 / 4 .. of them as one load
template <int kD>
struct KvScaleWord;
template <>
struct KvScaleWord<512> { using T = uint4; };
template <>
struct KvScaleWord<256> { using T = uint2; };
template <>
struct KvScaleWord<128> { using T = uint32_t; };
template <>
struct KvScaleWord<64> { using T = uint16_t; };
__device__ __forceinline__ uint32_t scale_byte(const uint4& w, int it, int pq) {
  const uint32_t x = it == 0 ? w.x : it == 1 ? w.y : it == 2 ? w.z : w.w;
  return x >> (8 * pq) & 0xFFu;
}
__device__ __forceinline__ uint32_t scale_byte(const uint2& w, int it, int pq) {
  return (it == 0 ? w.x : w.y) >> (8 * pq) & 0xFFu;
}
__device__ __forceinline__ uint32_t scale_byte(uint32_t w, int, int pq) { return w >> (8 * pq) & 0xFFu; }
__device__ __forceinline__ uint32_t scale_byte(uint16_t w, int, int pq) { return w >> (8 * (pq & 1)) & 0xFFu; }

template <int kD, int kN, bool kSplit>
__global__ void __launch_bounds__(kTcThreads, 1) kv_attend_tc_kernel(KvAttnArgs a, KvWork w) {
  using L = KvTc<kD, kN, kSplit>;
  using Misc = typename L::Misc;
  constexpr int kRn = L::kRn;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* smem = align_smem_1024(smem_raw);
  uint8_t* qs = smem;
  uint8_t* kring = qs + L::kQBytes;
  uint8_t* vring = kring + (size_t)w.kstages * L::kTileBytes;
  uint8_t* ps = vring + (size_t)w.vstages * L::kTileBytes;
  Misc& m = *reinterpret_cast<Misc*>(ps + 2 * L::kPBytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const bool sep = !a.c.shared;

  if (tid == 0) {
    for (int i = 0; i < kTcInfo; ++i) {
      mbar_init(&m.info_full[i], 1);
      mbar_init(&m.info_empty[i], kTcSoft + kTcDec + 1);
    }
    for (int i = 0; i < kTcRing; ++i) {
      mbar_init(&m.k_full[i], kTcDec);
      mbar_init(&m.v_full[i], kTcDec);
      mbar_init(&m.k_empty[i], 1);
      mbar_init(&m.v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&m.s_full[i], 1);
      mbar_init(&m.s_empty[i], kTcSoft);
      mbar_init(&m.p_full[i], kTcSoft);
      mbar_init(&m.p_empty[i], 1);
    }
    mbar_init(&m.q_empty, 1);
    mbar_init(&m.o_empty, kTcSoft);
    mbar_init(&m.all_done, 1);
    for (int i = 0; i < kTcFrag; ++i) {
      mbar_init(&m.q_full[i], kTcDec);
      m.redo[i] = 0;
    }
    fence_barrier_init();
  }
  for (int i = tid; i < kRn; i += kTcThreads) {
    m.row_tok[i] = w.ht > 1 ? 0 : i / a.group;
    m.row_head[i] = w.ht > 1 ? i : i % a.group;
  }
  if (warp == kTcMma) {
    tc::tmem_alloc(&m.tmem, L::kTmemCols);
    tc::tmem_relinquish();
  }
  pdl_wait_prior();

  // ---- where this CTA's tiles begin: a scan of the requests' tile counts ----
  long long total = 0, begin = 0, end = 0;
  {
    long long mine = 0;
    for (int r = tid; r < a.requests; r += kTcThreads) mine += kv_request_tiles(a, w, r);
    long long v = mine;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) m.part[warp] = v;
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    for (int i = 0; i <= kTcAddr; ++i) total += m.part[i];
    const int ctas = total > 0 ? kv_ctas(w, total) : 0;
    if ((int)blockIdx.x < ctas) {
      begin = kv_cta_start(total, ctas, blockIdx.x);
      end = kv_cta_start(total, ctas, blockIdx.x + 1);
    }
    __syncthreads();
    if (begin < end) {
      long long base = 0;
      for (int r0 = 0; r0 < a.requests; r0 += kTcThreads) {
        const int r = r0 + tid;
        const long long n = a.requests <= kTcThreads ? mine : r < a.requests ? kv_request_tiles(a, w, r) : 0;
        long long x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long p = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += p;
        }
        if (lane == 31) m.part[warp] = x;
        __syncthreads();
        long long before = base, all = base;
        for (int i = 0; i <= kTcAddr; ++i) {
          if (i < warp) before += m.part[i];
          all += m.part[i];
        }
        x += before;
        if (r < a.requests && x - n <= begin && begin < x) {
          m.first_r = r;
          m.first_off = begin - (x - n);
        }
        base = all;
        __syncthreads();
        if (base > begin) break;
      }
    }
  }
  __syncthreads();
  const uint32_t tmem = m.tmem;
  const int ntiles = (int)(end - begin);

  if (warp == kTcAddr) {
    // ---------------- addresses ----------------
    if (ntiles > 0) {
      int r = m.first_r, i = 0, kvh = 0, ht = 0;
      long long off = m.first_off;
      int2 tq = kv_queries(a, r);
      KvItem it = kv_item(a, w, r, tq, 0);
      const int per = a.c.kv_heads * w.ht;  // items of the same tokens
      while (off >= (long long)it.tiles * per) {
        off -= (long long)it.tiles * per;
        it = kv_item(a, w, r, tq, ++i);
      }
      int u = (int)(off / it.tiles);
      kvh = u / w.ht;
      ht = u % w.ht;
      int j = (int)(off % it.tiles);
      if (lane == 0 && kv_rows_of(a, r) != a.kv_lens[r]) flag(a.status, WH_DEV_BADARG);
      bool frag_first = true;
      int slot1 = 0;

      // key index of this lane's row k of tile jj, -1 past the last one seen
      auto key_of = [&](const KvItem& x, int jj, int k) {
        const int v = jj * kKvTile + lane + 32 * k;
        return v >= x.seen ? -1 : v < x.head ? v : x.start + (v - x.head);
      };
      int key[2], blk[2];
      auto look_up = [&](int rr, const KvItem& x, int jj) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          key[k] = key_of(x, jj, k);
          blk[k] = key[k] < 0 ? -1 : a.block_table[(long long)rr * a.max_blocks + key[k] / a.c.page];
        }
      };
      look_up(r, it, j);
      for (int n = 0; n < ntiles; ++n) {
        const int slot = n % kTcInfo;
        if (n >= kTcInfo && !warp_wait(&m.info_empty[slot], ((n / kTcInfo) - 1) & 1, a.status)) break;
        // this tile's entries, then the next tile's look-up, which may need the next item
        const int r_ = r, j_ = j, kvh_ = kvh, ht_ = ht;
        const KvItem x = it;
        int ck[2] = {key[0], key[1]}, cb[2] = {blk[0], blk[1]};
        const bool frag_last = j + 1 == it.tiles || n + 1 == ntiles;
        if (n + 1 < ntiles) {
          if (++j == it.tiles) {
            j = 0;
            if (++ht == w.ht) {
              ht = 0;
              if (++kvh == a.c.kv_heads) {
                kvh = 0;
                ++i;
                if (i * w.tt >= tq.y) {
                  i = 0;
                  do {
                    ++r;
                    tq = kv_queries(a, r);
                  } while (tq.y == 0);
                  if (lane == 0 && kv_rows_of(a, r) != a.kv_lens[r]) flag(a.status, WH_DEV_BADARG);
                }
                it = kv_item(a, w, r, tq, i);
              }
            }
          }
          look_up(r, it, j);
        }
        KvTileInfo& f = m.info[slot];
        bool all = true;
        const int p1 = x.p0 + x.nt - 1;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          int b = cb[k];
          if (ck[k] >= 0 && (b < 0 || b >= a.c.blocks)) {
            flag(a.status, WH_DEV_BADARG);
            b = -1;
          }
          if (ck[k] < 0) b = -1;
          const int row = b < 0 ? 0 : kvh_ * a.c.page + ck[k] % a.c.page;
          all = all && b >= 0 && ck[k] <= x.p0 &&
                (a.window == 0 || ck[k] > p1 - a.window || ck[k] < a.first);
          f.row[lane + 32 * k] = make_int2(b, row);
        }
        all = __all_sync(0xffffffffu, all);
        if (lane == 0) {
          const long long g = begin + n;
          f.end = g + (x.tiles - j_);
          f.r = r_;
          f.t0 = x.t0;
          f.nt = x.nt;
          f.p0 = x.p0;
          f.kvh = kvh_;
          f.ht = ht_;
          f.head = x.head;
          f.start = x.start;
          f.u0 = j_ * kKvTile;
          f.flags = (frag_first ? kFragFirst : 0) | (frag_last ? kFragLast : 0) |
                    (all ? 0 : kTileMasked) | (g - j_ >= begin ? kItemFirst : 0) |
                    (f.end <= end ? kItemLast : 0) | slot1;
        }
        frag_first = frag_last;
        if (frag_last) slot1 = kSlot1;
        __syncwarp();
        if (lane == 0) mbar_arrive(&m.info_full[slot]);
      }
    }
  } else if (warp == kTcMma) {
    // ---------------- MMA issuer ----------------
    if (lane == 0 && ntiles > 0) {
      constexpr uint32_t id_s = tc::idesc_f16(64, kN, false, false);
      constexpr uint32_t id_o = tc::idesc_f16(128, kN, true, true);
      const int vst = sep ? w.vstages : w.kstages;
      uint8_t* vbase = sep ? vring : kring;
      bool ok = true;
      bool first[2], last[2];
      int frags = 0;  // fragments whose first product has been issued for O
      auto products_s = [&](int n) {
        const int slot = n % kTcInfo, ks = n % w.kstages, b = n & 1;
        if (!mbar_wait(&m.info_full[slot], (n / kTcInfo) & 1, a.status)) return false;
        first[b] = m.info[slot].flags & kFragFirst;
        last[b] = m.info[slot].flags & kFragLast;
        mbar_arrive(&m.info_empty[slot]);
        if (!mbar_wait(&m.k_full[ks], (n / w.kstages) & 1, a.status)) return false;
        if (n >= 2 && !mbar_wait(&m.s_empty[b], ((n >> 1) - 1) & 1, a.status)) return false;
        tc::fence_after_sync();
        const uint32_t kt = smem_u32(kring + (size_t)ks * L::kTileBytes), qt = smem_u32(qs);
#pragma unroll 4
        for (int k = 0; k < kD / 16; ++k)
          tc::mma_f16(tmem + L::kTmemS + b * kN,
                      tc::desc_sw128(kt + (k >> 2) * (kKvTile * 128) + (k & 3) * 32),
                      tc::desc_sw128(qt + (k >> 2) * (kN * 128) + (k & 3) * 32), id_s, k != 0);
        tc::commit(&m.s_full[b]);
        if (sep) tc::commit(&m.k_empty[ks]);
        if (last[b]) tc::commit(&m.q_empty);
        return true;
      };
      auto products_o = [&](int n) {
        const int vs = n % vst, b = n & 1;
        if (sep && !mbar_wait(&m.v_full[vs], (n / vst) & 1, a.status)) return false;
        if (!mbar_wait(&m.p_full[b], (n >> 1) & 1, a.status)) return false;
        if (first[b]) {
          if (frags > 0 && !mbar_wait(&m.o_empty, (frags - 1) & 1, a.status)) return false;
          ++frags;
        }
        tc::fence_after_sync();
        const uint32_t vt = smem_u32(vbase + (size_t)vs * L::kTileBytes);
        const uint32_t pt = smem_u32(ps + b * L::kPBytes);
#pragma unroll
        for (int blk = 0; blk < L::kBlocks; ++blk)
#pragma unroll
          for (int k = 0; k < kKvTile / 16; ++k)
            tc::mma_f16(tmem + L::kTmemO + blk * kN,
                        // 64-wide heads: rows 64-127 repeat rows 0-63 and are not read
                        tc::desc_sw128_mn(vt + blk * 2 * (kKvTile * 128) + k * 2048,
                                          kD >= 128 ? kKvTile * 128 : 0),
                        tc::desc_sw128_mn(pt + k * 2048, 1024), id_o, !(first[b] && k == 0));
        tc::commit(&m.p_empty[b]);
        tc::commit(sep ? &m.v_empty[vs] : &m.k_empty[vs]);
        return true;
      };
      ok = products_s(0);
      for (int n = 0; ok && n < ntiles; ++n) {
        if (n + 1 < ntiles) ok = products_s(n + 1);
        if (ok) ok = products_o(n);
      }
      // every product has finished before TMEM is released
      tc::commit(&m.all_done);
      mbar_wait(&m.all_done, 0, a.status);
    }
  } else if (warp >= kTcSoft) {
    // ---------------- decode ----------------
    using SW = typename KvScaleWord<kD>::T;
    const int dw = warp - kTcSoft, r7 = lane & 7, pq = lane >> 3;
    const int key = dw * 8 + r7;  // this lane's row of every tile
    constexpr int kIt = L::kIt;
    const bool part_on = kD >= 128 || pq < 2;
    struct Raw {
      uint4 k[kIt], v[kIt];
      SW ks, vs;
      bool seen;
    };
    auto load = [&](int n, Raw& x) {
      const int slot = n % kTcInfo;
      if (!warp_wait(&m.info_full[slot], (n / kTcInfo) & 1, a.status)) return false;
      const int2 br = m.info[slot].row[key];
      x.seen = br.x >= 0;
#pragma unroll
      for (int i = 0; i < kIt; ++i) x.k[i] = x.v[i] = make_uint4(0, 0, 0, 0);
      x.ks = x.vs = SW{};
      if (x.seen && part_on) {
        const long long co = br.x * a.c.block_stride + (long long)br.y * (kD / 2) + pq * 16;
        const long long so = br.x * a.c.scale_block_stride + (long long)br.y * (kD / 32);
#pragma unroll
        for (int i = 0; i < kIt; ++i)
          x.k[i] = __ldg(reinterpret_cast<const uint4*>(a.c.keys + co + i * 64));
        x.ks = __ldg(reinterpret_cast<const SW*>(a.c.key_scales + so));
        if (sep) {
#pragma unroll
          for (int i = 0; i < kIt; ++i)
            x.v[i] = __ldg(reinterpret_cast<const uint4*>(a.c.values + co + i * 64));
          x.vs = __ldg(reinterpret_cast<const SW*>(a.c.value_scales + so));
        }
      }
      return true;
    };
    auto put = [&](const uint4 (&c)[kIt], const SW& sw, bool seen, uint8_t* tile) {
      bool in = true;
      if (part_on) {
#pragma unroll
        for (int i = 0; i < kIt; ++i) {
          const int part = pq + 4 * i;  // block of 32 columns
          uint8_t* row = tile + (part >> 1) * (kKvTile * 128) + key * 128;
          in = decode_block(c[i], scale_byte(sw, i, pq), seen, row, (part & 1) * 4, r7) && in;
        }
      }
      return in;
    };
    // The item's queries as f16 rows; warp dw takes rows dw, dw + 8, ...
    auto load_q = [&](const KvTileInfo& f, int frag) {
      constexpr int kG = kD / 8;                    // 8-column groups of a row
      constexpr int kPer = kG > 32 ? kG / 32 : 1;   // of them a lane takes
      constexpr int kRows = kRn / kTcDec > 0 ? kRn / kTcDec : 1;
      constexpr int kBatch = kRows < 4 ? kRows : 4;
      const int rows = w.ht > 1 ? min(kRn, a.group - f.ht * kRn) : f.nt * a.group;
#pragma unroll 1
      for (int b0 = 0; b0 < kRows; b0 += kBatch) {
        float v[kBatch][kPer][8];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          const int row = dw + kTcDec * (b0 + b);
#pragma unroll
          for (int g = 0; g < kPer; ++g) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[b][g][e] = 0.0f;
            if (row < rows && lane + 32 * g < kG)
              kv_load8_any(a, (f.t0 + m.row_tok[row]) * a.q_token_stride +
                                  (f.kvh * a.group + f.ht * kRn + m.row_head[row]) * a.q_head_stride +
                                  (lane + 32 * g) * 8,
                           v[b][g]);
          }
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          const int row = dw + kTcDec * (b0 + b);
          if (row >= kRn) continue;
          float top = 0.0f;
          bool fin = true;
#pragma unroll
          for (int g = 0; g < kPer; ++g)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              top = fmaxf(top, fabsf(v[b][g][e]));
              fin &= isfinite(v[b][g][e]);
            }
#pragma unroll
          for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          fin = __all_sync(0xffffffffu, fin);
          // 2^14 <= top * mul < 2^15; below 2^-100 the row's scores vanish anyway
          const int ex = max(int(__float_as_uint(top) >> 23) - 127, -100);
          const float mul = fin ? exp2i(14 - ex) : 0.0f;
          if (lane == 0) {
            if (!fin) m.redo[frag % kTcFrag] = 1;
            m.fac[frag % kTcFrag][row] = a.scale * kLog2e * exp2i(max(ex - 18, -126));
          }
#pragma unroll
          for (int g = 0; g < kPer; ++g) {
            const int gi = lane + 32 * g;
            if (gi >= kG) continue;
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = fin ? v[b][g][2 * e] * mul : 0.0f;
              const float y = fin ? v[b][g][2 * e + 1] * mul : 0.0f;
              const __half2 h = __floats2half2_rn(x, y);
              hi[e] = half2_bits(h);
              if (kSplit)
                lo[e] = half2_bits(__floats2half2_rn(x - __low2float(h), y - __high2float(h)));
            }
            uint8_t* chunk = qs + (gi >> 3) * (kN * 128);
            const int c16 = gi & 7;
            const int r0 = kSplit ? 2 * row : row;
            *reinterpret_cast<uint4*>(chunk + r0 * 128 + ((c16 ^ (r0 & 7)) << 4)) =
                make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if (kSplit)
              *reinterpret_cast<uint4*>(chunk + (r0 + 1) * 128 + ((c16 ^ ((r0 + 1) & 7)) << 4)) =
                  make_uint4(lo[0], lo[1], lo[2], lo[3]);
          }
        }
      }
    };
    Raw cur, nxt;
    bool ok = ntiles == 0 || load(0, cur);
    int frag = -1;
    for (int n = 0; ok && n < ntiles; ++n) {
      if (n + 1 < ntiles && !load(n + 1, nxt)) break;
      const int slot = n % kTcInfo;
      const KvTileInfo& f = m.info[slot];
      if (f.flags & kFragFirst) {
        ++frag;
        if (frag > 0 && !warp_wait(&m.q_empty, (frag - 1) & 1, a.status)) break;
        load_q(f, frag);
        __syncwarp();
        if (lane == 0) mbar_arrive(&m.q_full[frag % kTcFrag]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&m.info_empty[slot]);
      const int ks = n % w.kstages;
      if (n >= w.kstages && !warp_wait(&m.k_empty[ks], ((n / w.kstages) - 1) & 1, a.status)) break;
      bool in = put(cur.k, cur.ks, cur.seen, kring + (size_t)ks * L::kTileBytes);
      tc::fence_proxy_async_smem();
      if (!in) m.redo[frag % kTcFrag] = 1;
      __syncwarp();
      if (lane == 0) mbar_arrive(&m.k_full[ks]);
      if (sep) {
        const int vs = n % w.vstages;
        if (n >= w.vstages && !warp_wait(&m.v_empty[vs], ((n / w.vstages) - 1) & 1, a.status)) break;
        in = put(cur.v, cur.vs, cur.seen, vring + (size_t)vs * L::kTileBytes);
        tc::fence_proxy_async_smem();
        if (!in) m.redo[frag % kTcFrag] = 1;
        __syncwarp();
        if (lane == 0) mbar_arrive(&m.v_full[vs]);
      }
      if (n + 1 < ntiles) cur = nxt;
    }
  } else {
    // ---------------- softmax, epilogue ----------------
    constexpr int kMax = L::kMax;
    const float inf = __int_as_float(0x7f800000);
    const int g8 = lane >> 2, c4 = lane & 3;
    const int key0 = warp * 16 + g8;  // this thread's keys: key0 and key0 + 8
    // query row of the thread's entry e
    auto row_of = [&](int e) { return kSplit ? 4 * e + c4 : 8 * (e >> 1) + 2 * c4 + (e & 1); };
    // Tile n's product is in O^T and its weights may be overwritten.  Asked for
    // n - 2 before tile n's weights are written, so that the phase of p_empty
    // is never more than one ahead of the one asked for.
    auto product_done = [&](int n) {
      return warp_wait(&m.p_empty[n & 1], (n >> 1) & 1, a.status);
    };
    float fac[kMax], mx[kMax], sum[kMax];
    int frag = -1;
    uint32_t parity = 0;
    bool ok = true;
    for (int n = 0; n < ntiles; ++n) {
      const int slot = n % kTcInfo, b = n & 1;
      // A wait that runs out clears ok; the next barrier carries that to all
      // four warps, which leave together.
      ok = ok && warp_wait(&m.info_full[slot], (n / kTcInfo) & 1, a.status);
      const KvTileInfo& f = m.info[slot];
      const int flags = ok ? f.flags : 0;
      if (flags & kFragFirst) {
        ++frag;
        ok = ok && warp_wait(&m.q_full[frag % kTcFrag], (frag / kTcFrag) & 1, a.status);
#pragma unroll
        for (int e = 0; e < kMax; ++e) {
          fac[e] = m.fac[frag % kTcFrag][row_of(e)];
          mx[e] = -inf;
          sum[e] = 0.0f;
        }
      }
      ok = ok && warp_wait(&m.s_full[b], (n >> 1) & 1, a.status);
      tc::fence_after_sync();
      uint32_t raw[kN / 2];
      tc::ld_16x256b(tmem + ((uint32_t)(warp * 32) << 16) + L::kTmemS + b * kN, raw);
      tc::wait_ld_of(raw);
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&m.s_empty[b]);
      // log2 scores: s[e][0] of key0, s[e][1] of key0 + 8
      float s[kMax][2];
#pragma unroll
      for (int e = 0; e < kMax; ++e)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (kSplit)
            s[e][k] = (__uint_as_float(raw[4 * e + 2 * k]) + __uint_as_float(raw[4 * e + 2 * k + 1])) * fac[e];
          else
            s[e][k] = __uint_as_float(raw[4 * (e >> 1) + 2 * k + (e & 1)]) * fac[e];
        }
      if (flags & kTileMasked) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int u = f.u0 + key0 + 8 * k;
          const int i = u < f.head ? u : f.start + (u - f.head);
          const bool real = f.row[key0 + 8 * k].x >= 0;
#pragma unroll
          for (int e = 0; e < kMax; ++e) {
            const int p = f.p0 + m.row_tok[row_of(e)];
            const bool seen = real && i <= p && (a.window == 0 || i > p - a.window || i < a.first);
            if (!seen) s[e][k] = -inf;
          }
        }
      }
      // the tile's maximum per query row: over the warp's 16 keys, then over the warps
      float* red = &m.red[parity][warp][0];
#pragma unroll
      for (int e = 0; e < kMax; ++e) {
        float t = fmaxf(s[e][0], s[e][1]);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
        if (g8 == 0) red[row_of(e)] = t;
      }
      if (!bar_and(1, kTcSoft * 32, ok)) break;
      float tm[kMax];
      bool grow = false;
#pragma unroll
      for (int e = 0; e < kMax; ++e) {
        const int r = row_of(e);
        tm[e] = fmaxf(fmaxf(m.red[parity][0][r], m.red[parity][1][r]),
                      fmaxf(m.red[parity][2][r], m.red[parity][3][r]));
        grow |= tm[e] > mx[e] + kLag;
      }
      parity ^= 1;
      // every warp sees every row's maximum, so all four decide alike
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int e = 0; e < kMax; ++e) {
          const float to = fmaxf(mx[e], tm[e]);
          const float sh = mx[e] == -inf ? 0.0f : ex2(mx[e] - to);
          mx[e] = to;
          sum[e] *= sh;
          if (warp == 0 && g8 == 0) m.shrink[row_of(e)] = sh;
        }
        if (!(flags & kFragFirst)) {
          // O^T shrinks too, once the previous tile's product is in it
          ok = product_done(n - 1);
          tc::fence_after_sync();
          if (!bar_and(1, kTcSoft * 32, ok)) break;
#pragma unroll 1
          for (int c0 = 0; c0 < kN; c0 += 16)
#pragma unroll 1
            for (int blk = 0; blk < L::kBlocks; ++blk) {
              const uint32_t at = tmem + ((uint32_t)(warp * 32) << 16) + L::kTmemO + blk * kN + c0;
              uint32_t o[16];
              tc::ld_32x32b_x16(at, o);
              tc::wait_ld_of(o);
#pragma unroll
              for (int e = 0; e < 16; ++e)
                o[e] = __float_as_uint(__uint_as_float(o[e]) * m.shrink[kSplit ? (c0 + e) >> 1 : c0 + e]);
              tc::st_32x32b_x16(at, o);
            }
          tc::wait_st();
          tc::fence_before_sync();
          if (!bar_and(1, kTcSoft * 32, ok)) break;  // shrink may be written again
        }
      }
      // weights
      if (n >= 2) ok = product_done(n - 2);
      uint8_t* pt = ps + b * L::kPBytes;
#pragma unroll
      for (int e = 0; e < kMax; ++e) {
        const float off = mx[e] == -inf ? 0.0f : kLift - mx[e];
        s[e][0] = ex2(s[e][0] + off);
        s[e][1] = ex2(s[e][1] + off);
        sum[e] += s[e][0] + s[e][1];
      }
#pragma unroll
      for (int j = 0; j < kN / 8; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t bits;
          if (kSplit) {
            const float p = s[j][k];
            const __half hi = __float2half_rn(p);
            bits = half2_bits(__halves2half2(hi, __float2half_rn(p - __half2float(hi))));
          } else {
            bits = half2_bits(__floats2half2_rn(s[kSplit ? 0 : 2 * j][k], s[kSplit ? 0 : 2 * j + 1][k]));
          }
          const int key = key0 + 8 * k;
          *reinterpret_cast<uint32_t*>(pt + key * 128 + ((j ^ (key & 7)) << 4) + 4 * c4) = bits;
        }
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&m.p_full[b]);

      if (flags & kFragLast) {
        // ---- the fragment's sums, then its rows: out, or a partial slot ----
        if (!bar_and(1, kTcSoft * 32, ok)) break;  // every warp has read the maxima in red
#pragma unroll
        for (int e = 0; e < kMax; ++e) {
          float t = sum[e];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
          if (g8 == 0) {
            m.red[0][warp][row_of(e)] = t;
            if (warp == 0) m.red[1][0][row_of(e)] = mx[e];
          }
        }
        ok = product_done(n);
        tc::fence_after_sync();
        if (!bar_and(1, kTcSoft * 32, ok)) break;
        const bool whole = (flags & kItemFirst) && (flags & kItemLast);
        const int rows = w.ht > 1 ? min(kRn, a.group - f.ht * kRn) : f.nt * a.group;
        const int part = 2 * blockIdx.x + (flags & kSlot1 ? 1 : 0);
        const int h0 = f.kvh * a.group + f.ht * kRn;
        const int redo = m.redo[frag % kTcFrag];
        const int tid4 = warp * 32 + lane;
        if (tid4 < kRn) {
          const float l = (m.red[0][0][tid4] + m.red[0][1][tid4]) + (m.red[0][2][tid4] + m.red[0][3][tid4]);
          const float top = m.red[1][0][tid4];
          float os = 1.0f / 16.0f;  // the tiles hold 16 times the values
          if (whole) {
            float z = l;
            if (a.sink && tid4 < rows) {
              const float sk = a.sink[h0 + m.row_head[tid4]] * kLog2e;
              const float to = fmaxf(top, sk), base = to == -inf ? 0.0f : to;
              const float sh = top == -inf ? 0.0f : ex2(top - base);
              os *= sh;
              z = l * sh + ex2(sk - base + kLift);
            }
            os = z == 0.0f ? 0.0f : os / z;
          } else if (tid4 < rows) {
            w.part_ml[(long long)part * kRn + tid4] = make_float2(top, l);
          }
          m.out_scale[tid4] = os;
          if (tid4 < rows && (flags & kItemFirst)) {
            // where the item's other parts lie
            const int ctas = kv_ctas(w, total);
            const int parts = whole ? 1 : kv_cta_of(total, ctas, f.end - 1) - (int)blockIdx.x + 1;
            w.meta[(long long)(f.t0 + m.row_tok[tid4]) * a.heads + h0 + m.row_head[tid4]] =
                make_int4(blockIdx.x, parts, (flags & kSlot1 ? 1 : 0) | tid4 << 1, redo);
          }
          if (tid4 == 0 && !whole) w.part_redo[part] = redo;
          if (tid4 == 0) m.redo[frag % kTcFrag] = 0;
        }
        if (!bar_and(1, kTcSoft * 32, ok)) break;
        const int dim0 = warp * 32 + lane;
#pragma unroll 1
        for (int c0 = 0; c0 < kN; c0 += 16) {
          constexpr int kR = kSplit ? 8 : 16;  // query rows of 16 columns
          const int row0 = kSplit ? c0 / 2 : c0;
          if (row0 >= rows) break;
#pragma unroll 1
          for (int blk = 0; blk < L::kBlocks; ++blk) {
            uint32_t o[16];
            tc::ld_32x32b_x16(tmem + ((uint32_t)(warp * 32) << 16) + L::kTmemO + blk * kN + c0, o);
            tc::wait_ld_of(o);
            const int dim = blk * 128 + dim0;
            if (kD < 128 && dim >= kD) continue;
#pragma unroll
            for (int e = 0; e < kR; ++e) {
              const int row = row0 + e;
              if (row >= rows) continue;
              float v = kSplit ? __uint_as_float(o[2 * e & 15]) + __uint_as_float(o[(2 * e + 1) & 15])
                               : __uint_as_float(o[e]);
              v *= m.out_scale[row];
              if (whole)
                kv_store_any(a, (f.t0 + m.row_tok[row]) * a.out_token_stride +
                                    (h0 + m.row_head[row]) * a.out_head_stride + dim,
                             v);
              else
                w.part_o[((long long)part * kRn + row) * kD + dim] = v;
            }
          }
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&m.o_empty);
        if (!bar_and(1, kTcSoft * 32, ok)) break;  // red and out_scale may be written again
        parity = 0;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&m.info_empty[slot]);
    }
  }
  pdl_launch_dependents();
  tc::fence_before_sync();
  __syncthreads();
  if (warp == kTcMma) tc::tmem_dealloc(tmem, L::kTmemCols);
}

template <int kD, int kN, bool kSplit>
static cudaError_t launch_attend_tc(const KvAttnArgs& a, KvWork w, cudaStream_t s, bool pdl) {
  using L = KvTc<kD, kN, kSplit>;
  const int sets = a.c.shared ? 1 : 2;
  const int depth = std::min<int>(kTcRing, (232448 - L::fixed_bytes()) / (size_t(L::kTileBytes) * sets));
  w.kstages = depth;
  w.vstages = a.c.shared ? 0 : depth;
  const size_t smem = L::bytes(w.kstages, w.vstages);
  static_assert(L::fixed_bytes() + 2 * L::kTileBytes <= 232448, "shared memory over 227 KB");
  const cudaError_t e = ensure_smem(kv_attend_tc_kernel<kD, kN, kSplit>, 232448);
  if (e != cudaSuccess) return e;
  return launch_pdl(kv_attend_tc_kernel<kD, kN, kSplit>, dim3(w.ctas), kTcThreads, smem, s, pdl, a, w);
}

}  // namespace wh
