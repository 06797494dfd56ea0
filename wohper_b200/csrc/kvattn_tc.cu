// kvattn_tc.cu -- attention over the paged 4-bit cache on the 5th-generation
// tensor cores.
//
// Both products run with the cache as the tall operand, so that a kv head's
// query rows cost the tensor core only their columns:
//   S^T [64 keys x 64]  = K [64 x D] Q^T          (M = 64)
//   O^T [D x 64]       += V^T [D x 64] P^T        (M = 128, D / 128 blocks)
// K and V are decoded once per tile into f16 in shared memory (rows of 64
// columns, 128-byte swizzle).  The same bytes serve as the K-major operand of
// the first product and, where the values are the keys, as the MN-major
// operand of the second.
//
// f16 holds a code times its scale exactly over 36 octaves of scales (2^-27 to
// 2^9; kept as 16 times the value, scale bytes 100..136).  Items that meet
// another byte, a not-finite query or a not-finite block are marked and their
// rows computed again in f32.  A query row is brought to a largest value in
// [2^14, 2^15) by a power of two; 16-bit queries are then one f16 (exact, but for
// elements below 2^-28 of the largest), f32 queries are the sum of two (kSplit:
// columns 2i and 2i + 1), which keeps 22 bits down to 2^-16 of the largest.  Weights are 2^(s - m + kLift) with a maximum m that may lag by kLag,
// so at most 2^15: one f16 for 16-bit queries (11 bits), two for f32, the lower
// one times kLoUp: 22 bits down to 2^-23 of the largest weight, then one fewer
// for each halving, nothing below 2^-45.  Sums are f32.
//
// Warps: 0-7 softmax and epilogue (TMEM lane quadrant warp % 4; warps 4-7 the
// upper half of the columns), 8-23 decode, 24 MMA, 25 addresses (walks the work
// list, looks up blocks).  Decoding, scores, weights and sums of a tile follow
// one another; what overlaps them is the neighbouring tile (two fit beside 64
// queries of 512).  The MMA warp takes whichever product is ready, the second
// one first, since it frees a tile.
//
// Measured, 512 wide: decode 1.0-1.4 k cycles a tile, scores 1.15 k and sums 0.9 k
// (both bound by the operands' shared-memory reads), softmax 1.7-2.5 k, two tiles
// in flight: about 4 k cycles a tile; 32 requests x 8192 rows, 64 bf16 heads: 62 us
// with the join, 32 x 4096 of f32 57 us.  M = 128 keys a product would
// read 14 % fewer operand bytes but leave room for one tile only.
// The forms whose values are the keys spill nothing; those with values of their own
// 4-16 bytes, but for 16-bit queries of 64 to 256 columns, which spill nothing (of a
// tree 64 and 128 columns: 4 bytes).
#include "kvattn.cuh"
#include "tc.cuh"

namespace wh {

constexpr int kTcSoft = 8, kTcDec = 16;
constexpr int kTcMma = kTcSoft + kTcDec, kTcAddr = kTcMma + 1;
constexpr int kTcThreads = (kTcAddr + 1) * 32;
// Registers: 72 a thread at launch (26 warps); the decode warps give 16 up, the
// softmax warps take 32: 8 x 104 + 16 x 56 + 2 x 72 = 26 x 72.  More tiles in
// flight a decode warp (kAhead 2) spilled: 61 against 67 us at 32 x 8192 x 512 bf16.
constexpr int kTcSoftRegs = 104, kTcDecRegs = 56, kTcRegs = 72;
static_assert(kTcSoft * kTcSoftRegs + kTcDec * kTcDecRegs <= (kTcSoft + kTcDec) * kTcRegs, "registers");
static_assert(kTcSoft % 4 == 0 && kTcDec % 4 == 0, "whole warpgroups");
constexpr int kTcInfo = 8;   // tiles the address warp may run ahead
constexpr int kTcFrag = 4;   // fragments whose query factors are kept
constexpr int kTcRedo = 8;   // fragments whose redo marks are kept
constexpr int kTcRing = 4;   // most tiles of keys (and of values) in shared memory
constexpr int kTcCols = 64;  // columns of the products
constexpr float kLag = 6.0f;   // log2 units that the running maximum may lag behind
constexpr float kLoUp = 2048.0f;  // the lower f16 of an f32 weight is held times this: its last bit is 2^-35
constexpr float kLift = 9.0f;  // weights are held as 2^(s - m + kLift) <= 2^15
constexpr int kKvBias = 123;   // scale byte b stands for 2^(b - kKvBias) in the f16 tiles

enum : int {
  kFragFirst = 1,   // the first tile of a fragment: a CTA's tiles of an item, at most kFold
  kFragLast = 2,    // its last tile
  kTileMasked = 4,  // some row of the tile is not seen by every query
  kItemFirst = 8,   // the item's first tile is in this CTA
  kItemLast = 16,   // the item's last tile is in this CTA
  kSlot1 = 32,      // partial slot 1 (the item does not begin the CTA's range)
  kFragCut = 64,    // with kFragLast: the CTA goes on with the item in the next fragment
  kFragCont = 128,  // the item's partial slot holds the sums of earlier fragments
};

struct KvTileInfo {
  int2 row[kKvTile];  // block (-1: not seen) and row in the block
  long long first;    // where the item's tiles begin on the line
  int tiles, t0, nt, p0, kvh, ht, head, start, u0, flags;
  int last;  // of a tree: the request's last row
};

template <int kD, bool kSplit>
struct KvTc {
  static constexpr int kN = kTcCols;
  static constexpr int kRn = kSplit ? kN / 2 : kN;  // query rows
  static constexpr int kChunks = kD / 64;
  static constexpr int kBlocks = kD >= 128 ? kD / 128 : 1;  // 128-row blocks of O^T
  static constexpr int kQBytes = kChunks * kN * 128;
  static constexpr int kTileBytes = kD * 128;
  static constexpr int kPBytes = kKvTile * 128;
  // A decode warp takes 8 rows x 128 columns at a time; decode warps w and
  // w + 8 share row group w.  One unit a row: keys to the one, values to the other.
  static constexpr int kUnits = kD >= 128 ? kD / 128 : 1;
  static constexpr int kPer = kUnits > 1 ? kUnits / 2 : 1;
  static constexpr int kFillers = kUnits > 1 ? kTcDec : kTcDec / 2;  // warps that fill a tile
  // Most tiles of a fragment (0: any number).  A sum that runs through the tensor core
  // loses up to 2e-7 of itself with each tile, always downwards (values of one sign: 2.4e-4
  // after 1300 tiles).  After 32 tiles f32 sums are added, in f32, to what the partial slot
  // holds: 1.3e-6 to 2e-6 whatever the length, for 11 % of the time at 32 x 32768 x 512.
  // 16-bit calls, where the code for it alone costs 2 %, keep on: the loss passes f16's
  // own rounding after about 10^3 tiles a CTA (64 requests x 10^5 rows), bf16's after 10^4.
  static constexpr int kFold = kSplit ? 32 : 0;
  static constexpr int kAhead = 1;  // tiles whose codes a decode warp has in flight: more spilled and lost
  static constexpr int kNh = kN / 2;                        // columns of a softmax half
  static constexpr int kRh = kRn / 2;                       // query rows of a softmax half
  static constexpr int kMax = kNh / 4 / (kSplit ? 2 : 1);   // query rows a softmax thread holds
  static constexpr uint32_t kTmemO = 0, kTmemS = kBlocks * kN;
  static constexpr uint32_t kTmemNeed = kBlocks * kN + 2 * kN;
  static constexpr uint32_t kTmemCols = kTmemNeed <= 256 ? 256 : 512;
  static_assert(kTmemNeed <= 512, "TMEM");
  struct Misc {
    KvTileInfo info[kTcInfo];
    float fac[kTcFrag][kRn];   // accumulator -> log2 score, per query row
    float red[2][4][kRn];      // a tile's maxima, a fragment's sums
    float top[kRn];
    float out_scale[kRn];
    float shrink[kRn];
    long long out_row[kRn];    // where a row goes, in elements
    int redo[kTcRedo];
    int row_tok[kRn];          // token (within the item) and head (within its heads) of a row
    int row_head[kRn];
    uint64_t info_full[kTcInfo], info_empty[kTcInfo];
    uint64_t k_full[kTcRing], k_empty[kTcRing], v_full[kTcRing], v_empty[kTcRing];
    uint64_t s_full[2], p_full[2], p_empty[2];
    uint64_t q_full[kTcFrag], q_empty, o_empty, all_done;
    KvPlace at;
    uint32_t tmem;
  };
};
template <int kD, bool kSplit, bool kSep>
struct KvTcSmem {
  using L = KvTc<kD, kSplit>;
  static constexpr int kFixed = L::kQBytes + 2 * L::kPBytes + (int)sizeof(typename L::Misc) + 1024;
  static constexpr int kFit = (232448 - kFixed) / (L::kTileBytes * (kSep ? 2 : 1));
  static constexpr int kStages = kFit < kTcRing ? kFit : kTcRing;
  static constexpr int kBytes = kFixed + kStages * L::kTileBytes * (kSep ? 2 : 1);
  // with values of their own one tile of each is enough: keys are free after the first product
  static_assert(kStages >= (kSep ? 1 : 2), "shared memory over 227 KB");
};

// 8 codes (code i in bits 4i..4i+3) -> 8 f16
__device__ __forceinline__ uint4 e2m1x8_to_f16(uint32_t w) {
  uint4 v;
  asm("{ .reg .b8 a, b, c, d; mov.b32 {a, b, c, d}, %4; cvt.rn.f16x2.e2m1x2 %0, a;"
      " cvt.rn.f16x2.e2m1x2 %1, b; cvt.rn.f16x2.e2m1x2 %2, c; cvt.rn.f16x2.e2m1x2 %3, d; }"
      : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
      : "r"(w));
  return v;
}
__device__ __forceinline__ uint32_t hmul2_u(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// One block of 32 codes into four 16-byte pieces of a tile row, piece j at
// row + at[j].  seen = false: zeros.  Returns false where the scale byte has no
// exact f16 form.  Lanes with on = false write nothing.
__device__ __forceinline__ bool decode_block(const uint4& c, uint32_t sb, bool seen, bool on,
                                             uint8_t* row, const uint32_t (&at)[4]) {
  const int k = int(sb) - kKvBias;
  const bool zero = !seen || sb == 0;
  const bool in = zero || (k >= -23 && k <= 13);
  // 2^k as f16, subnormal below 2^-14; the products with codes are exact
  const uint32_t one = k >= -14 ? uint32_t(k + 15) << 10 : 1u << ((k + 24) & 31);
  const uint32_t scale = zero || !in ? 0u : one | one << 16;
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  uint4 v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[j] = e2m1x8_to_f16(w[j]);
    v[j].x = hmul2_u(v[j].x, scale);
    v[j].y = hmul2_u(v[j].y, scale);
    v[j].z = hmul2_u(v[j].z, scale);
    v[j].w = hmul2_u(v[j].w, scale);
  }
  if (on) {
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(row + at[j]) = v[j];
  }
  return in || !on;
}

// Registers of this warpgroup from here on (every warp of it executes this).
template <int kRegs>
__device__ __forceinline__ void regs_more() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void regs_less() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
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
// 16 bytes of a query row -> 8 values (16-bit types) or 4 (f32)
__device__ __forceinline__ void kv_widen(const uint4& x, int dtype, float (&v)[8]) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (dtype == WH_DTYPE_BF16) {
      v[2 * j] = __uint_as_float(w[j] << 16);
      v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    } else {
      const float2 f = h2_to_f2(w[j]);
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  }
}
__device__ __forceinline__ void kv_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void kv_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void kv_put(__half* p, float v) { *p = __float2half_rn(v); }

template <int kD, bool kSplit, bool kSep, class Args>
__global__ void __launch_bounds__(kTcThreads, 1) kv_attend_tc_kernel(Args a, KvWork w) {
  using L = KvTc<kD, kSplit>;
  using Misc = typename L::Misc;
  constexpr int kN = kTcCols, kRn = L::kRn, kNh = L::kNh, kRh = L::kRh;
  constexpr int kStages = KvTcSmem<kD, kSplit, kSep>::kStages;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* smem = align_smem_1024(smem_raw);
  uint8_t* qs = smem;
  uint8_t* kring = qs + L::kQBytes;
  uint8_t* vring = kSep ? kring + kStages * L::kTileBytes : kring;
  uint8_t* ps = vring + kStages * L::kTileBytes;
  Misc& m = *reinterpret_cast<Misc*>(ps + 2 * L::kPBytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < kTcInfo; ++i) {
      mbar_init(&m.info_full[i], 1);
      mbar_init(&m.info_empty[i], kTcSoft + kTcDec + 1);
    }
    for (int i = 0; i < kTcRing; ++i) {
      mbar_init(&m.k_full[i], L::kFillers);
      mbar_init(&m.v_full[i], L::kFillers);
      mbar_init(&m.k_empty[i], 1);
      mbar_init(&m.v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&m.s_full[i], 1);
      mbar_init(&m.p_full[i], kTcSoft);
      mbar_init(&m.p_empty[i], 1);
    }
    mbar_init(&m.q_empty, 1);
    mbar_init(&m.o_empty, kTcSoft);
    mbar_init(&m.all_done, 1);
    for (int i = 0; i < kTcFrag; ++i) mbar_init(&m.q_full[i], kTcDec);
    for (int i = 0; i < kTcRedo; ++i) m.redo[i] = 0;
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

  tc::fence_before_sync();
  kv_place<kTcThreads>(a, w, m.at);
  tc::fence_after_sync();
  const uint32_t tmem = m.tmem;
  const int ntiles = m.at.ntiles();

  if (warp == kTcAddr) {
    // ---------------- addresses ----------------
    if (ntiles > 0) {
      KvWalk c(m.at);
      bool frag_first = true;
      int slot1 = 0, cont = 0;
      int run = 0;  // tiles of the fragment
      int key[2], blk[2];
      // this lane's two rows of tile jj: position (-1 past the last one seen) and block
      auto look_up = [&](int rr, const KvItem& x, int jj) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int v = jj * kKvTile + lane + 32 * k;
          key[k] = v >= x.seen ? -1 : kv_key(x.head, x.start, v);
          blk[k] = key[k] < 0 ? -1 : a.block_table[(long long)rr * a.max_blocks + kv_page_of(a.c, key[k])];
        }
      };
      look_up(c.r, c.it, c.j);
      for (int n = 0; n < ntiles; ++n) {
        const int slot = n % kTcInfo;
        if (n >= kTcInfo && !warp_wait(&m.info_empty[slot], ((n / kTcInfo) - 1) & 1, a.status)) break;
        // this tile's rows; the next tile's look-up starts before they are written down
        const int j_ = c.j, kvh_ = c.kvh, ht_ = c.ht;
        const long long at_ = c.at + w.lead;  // its tiles
        const KvItem x = c.it;
        const int last = Args::kTree ? max(c.len, 0) - 1 : 0;
        const int ck[2] = {key[0], key[1]}, cb[2] = {blk[0], blk[1]};
        const bool item_end = c.j + 1 == c.it.tiles || n + 1 == ntiles;  // of this CTA
        const bool frag_last = item_end || (L::kFold && ++run == L::kFold);
        if (n + 1 < ntiles) {
          if (++c.j == c.it.tiles) c.next(a, w);
          look_up(c.r, c.it, c.j);
        }
        KvTileInfo& f = m.info[slot];
        bool all = true;
        const int p1 = Args::kTree ? last : x.p0 + x.nt - 1;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          int b = cb[k];
          if (ck[k] >= 0 && (b < 0 || b >= a.c.blocks)) {
            flag(a.status, WH_DEV_BADARG);
            b = -1;
          }
          if (ck[k] < 0) b = -1;
          const int row = b < 0 ? 0 : kvh_ * a.c.page + (ck[k] - kv_page_of(a.c, ck[k]) * a.c.page);
          all = all && b >= 0 && (Args::kTree ? ck[k] < x.p0 : ck[k] <= x.p0) &&
                (a.window == 0 || ck[k] > p1 - a.window || ck[k] < a.first);
          f.row[lane + 32 * k] = make_int2(b, row);
        }
        all = __all_sync(0xffffffffu, all);
        if (lane == 0) {
          f.first = at_;
          f.tiles = x.tiles;
          f.t0 = x.t0;
          f.nt = x.nt;
          f.p0 = x.p0;
          f.kvh = kvh_;
          f.ht = ht_;
          f.head = x.head;
          f.start = x.start;
          f.u0 = j_ * kKvTile;
          if (Args::kTree) f.last = last;
          f.flags = (frag_first ? kFragFirst : 0) | (frag_last ? kFragLast : 0) |
                    (all ? 0 : kTileMasked) | (at_ >= m.at.begin ? kItemFirst : 0) |
                    (at_ + x.tiles <= m.at.end ? kItemLast : 0) | slot1 | cont |
                    (frag_last && !item_end ? kFragCut : 0);
        }
        frag_first = frag_last;
        if (frag_last) {
          run = 0;
          cont = item_end ? 0 : kFragCont;
          if (item_end) slot1 = kSlot1;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&m.info_full[slot]);
      }
    }
  } else if (warp == kTcMma) {
    // ---------------- MMA issuer ----------------
    constexpr uint32_t id_s = tc::idesc_f16(64, kN, false, false);
    constexpr uint32_t id_o = tc::idesc_f16(128, kN, true, true);
    const uint64_t dq = tc::desc_sw128(smem_u32(qs));
    const uint64_t dk = tc::desc_sw128(smem_u32(kring));
    // 64-wide heads: rows 64-127 of O^T repeat rows 0-63 and are not read
    const uint64_t dv = tc::desc_sw128_mn(smem_u32(vring), kD >= 128 ? kKvTile * 128 : 0);
    const uint64_t dp = tc::desc_sw128_mn(smem_u32(ps), 1024);
    auto ready = [&](uint64_t* bar, uint32_t phase) {
      return __all_sync(0xffffffffu, mbar_test_wait(bar, phase)) != 0;
    };
    int ns = 0, np = 0;     // next tile of the first, of the second product
    int begun = 0;          // fragments whose first product has begun
    int frags = 0;          // fragments whose second product has begun
    int fl_even = 0, fl_odd = 0;
    uint64_t since = 0;
    while (np < ntiles) {
      bool did = false;
      if (np < ns) {
        const int b = np & 1, vs = np % kStages;
        const bool first = (b ? fl_odd : fl_even) & kFragFirst;
        if (ready(&m.p_full[b], (np >> 1) & 1) &&
            (!kSep || ready(&m.v_full[vs], (np / kStages) & 1)) &&
            (!first || frags == 0 || ready(&m.o_empty, (frags - 1) & 1))) {
          tc::fence_after_sync();
          const uint64_t dv_ = dv + (uint32_t(vs) * L::kTileBytes >> 4);
          const uint64_t dp_ = dp + (uint32_t(b) * L::kPBytes >> 4);
          if (tc::elect_one()) {
#pragma unroll
            for (int blk = 0; blk < L::kBlocks; ++blk)
#pragma unroll
              for (int k = 0; k < kKvTile / 16; ++k)
                tc::mma_f16(tmem + L::kTmemO + blk * kN,
                            dv_ + ((blk * 2 * (kKvTile * 128) + k * 2048) >> 4),
                            dp_ + ((k * 2048) >> 4), id_o, k != 0 || !first);
            tc::commit(&m.p_empty[b]);
            tc::commit(kSep ? &m.v_empty[vs] : &m.k_empty[vs]);
          }
          __syncwarp();
          frags += first;
          ++np;
          did = true;
        }
      }
      // S^T of tile ns may overwrite that of ns - 2, whose weights are in use: read
      if (!did && ns < ntiles && ns < np + 2) {
        const int slot = ns % kTcInfo, ks = ns % kStages, b = ns & 1;
        if (ready(&m.info_full[slot], (ns / kTcInfo) & 1) &&
            ready(&m.k_full[ks], (ns / kStages) & 1) &&
            // A new fragment's queries are all there.  k_full does not say so where
            // half of the decode warps fill the keys (heads up to 128 wide); that
            // every warp has arrived also keeps q_empty within a phase of them.
            (!(m.info[slot].flags & kFragFirst) ||
             ready(&m.q_full[begun % kTcFrag], (begun / kTcFrag) & 1))) {
          const int fl = m.info[slot].flags;
          begun += fl & kFragFirst;
          (b ? fl_odd : fl_even) = fl;
          tc::fence_after_sync();
          const uint64_t dk_ = dk + (uint32_t(ks) * L::kTileBytes >> 4);
          if (tc::elect_one()) {
#pragma unroll
            for (int k = 0; k < kD / 16; ++k)
              tc::mma_f16(tmem + L::kTmemS + b * kN,
                          dk_ + (((k >> 2) * (kKvTile * 128) + (k & 3) * 32) >> 4),
                          dq + (((k >> 2) * (kN * 128) + (k & 3) * 32) >> 4), id_s, k != 0);
            tc::commit(&m.s_full[b]);
            if (kSep) tc::commit(&m.k_empty[ks]);
            if (fl & kFragLast) tc::commit(&m.q_empty);
            mbar_arrive(&m.info_empty[slot]);
          }
          __syncwarp();
          ++ns;
          did = true;
        }
      }
      if (did) {
        since = 0;
      } else if (since == 0) {
        since = globaltimer();
      } else if (globaltimer() - since > WH_WAIT_NS) {
        if (lane == 0) flag(a.status, WH_DEV_TIMEOUT);
        break;
      }
    }
    // every product has finished before TMEM is released
    if (tc::elect_one()) tc::commit(&m.all_done);
    __syncwarp();
    mbar_wait(&m.all_done, 0, a.status);
  } else if (warp >= kTcSoft) {
    // ---------------- decode ----------------
    regs_less<kTcDecRegs>();
    constexpr int kPer = L::kPer, kAhead = L::kAhead;
    const int dw = warp - kTcSoft, rg = dw & 7, dh = dw >> 3;
    const int r7 = lane & 7, pq = lane >> 3;
    const int key = rg * 8 + r7;  // this lane's row of every tile
    const bool on = kD >= 128 || pq < 2;
    const bool has_k = L::kUnits > 1 || dh == 0, has_v = kSep && (L::kUnits > 1 || dh == 1);
    const int unit0 = L::kUnits > 1 ? dh : 0;  // its units: unit0, unit0 + 2, ...
    uint32_t at[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) at[j] = (((pq & 1) * 4 + j) ^ r7) << 4;
    const uint32_t row_at = (pq >> 1) * (kKvTile * 128) + key * 128;
    struct Raw {
      uint4 k[kPer], v[kSep ? kPer : 1];
      uint32_t ks[kPer], vs[kSep ? kPer : 1];
      bool seen;
    };
    auto load = [&](int n, Raw& x) {
      const int slot = n % kTcInfo;
      if (!warp_wait(&m.info_full[slot], (n / kTcInfo) & 1, a.status)) return false;
      const int2 br = m.info[slot].row[key];
      x.seen = br.x >= 0;
      const bool go = x.seen && on;
      const long long co = br.x * a.c.block_stride + (long long)br.y * (kD / 2) + unit0 * 64 + pq * 16;
      const long long so = br.x * a.c.scale_block_stride + (long long)br.y * (kD / 32) + unit0 * 4 + pq;
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        if (has_k) {
          x.k[u] = go ? __ldg(reinterpret_cast<const uint4*>(a.c.keys + co + u * 128)) : make_uint4(0, 0, 0, 0);
          x.ks[u] = go ? __ldg(a.c.key_scales + so + u * 8) : 0;
        }
        if (kSep && has_v) {
          x.v[u] = go ? __ldg(reinterpret_cast<const uint4*>(a.c.values + co + u * 128)) : make_uint4(0, 0, 0, 0);
          x.vs[u] = go ? __ldg(a.c.value_scales + so + u * 8) : 0;
        }
      }
      return true;
    };
    // The item's queries as f16 rows; warp dw takes rows dw, dw + 16, ...
    auto load_q = [&](int t0, int nt, int kvh, int ht, int frag) {
      constexpr int kG = kD / (kSplit ? 4 : 8);     // 16-byte groups of a row
      constexpr int kLoads = kG > 32 ? kG / 32 : 1;  // of them a lane takes
      constexpr int kRows = kRn / kTcDec;
      constexpr int kElems = kSplit ? 4 : 8;
      constexpr int kBatch = kLoads >= 4 ? 1 : kRows < 4 / kLoads ? kRows : 4 / kLoads;
      const int rows = w.ht > 1 ? min(kRn, a.group - ht * kRn) : nt * a.group;
      const uint8_t* q = static_cast<const uint8_t*>(a.q);
#pragma unroll 1
      for (int b0 = 0; b0 < kRows; b0 += kBatch) {
      uint4 raw[kBatch][kLoads];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int row = dw + kTcDec * (b0 + b);
        const bool real = row < rows;
        const long long off = real ? (t0 + m.row_tok[row]) * a.q_token_stride +
                                         (kvh * a.group + ht * kRn + m.row_head[row]) * a.q_head_stride
                                   : 0;
#pragma unroll
        for (int g = 0; g < kLoads; ++g) {
          const int gi = lane + 32 * g;
          raw[b][g] = real && gi < kG ? *reinterpret_cast<const uint4*>(q + off * (kSplit ? 4 : 2) + gi * 16)
                                      : make_uint4(0, 0, 0, 0);
        }
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int row = dw + kTcDec * (b0 + b);
        // the largest magnitude, as an integer: a NaN or infinity is at least 0x7f800000
        float v[kLoads][8];
        uint32_t top = 0;
#pragma unroll
        for (int g = 0; g < kLoads; ++g) {
          if (kSplit) {
            const uint32_t x[4] = {raw[b][g].x, raw[b][g].y, raw[b][g].z, raw[b][g].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) v[g][e] = __uint_as_float(x[e]);
          } else {
            kv_widen(raw[b][g], a.dtype, v[g]);
          }
#pragma unroll
          for (int e = 0; e < kElems; ++e) top = max(top, __float_as_uint(v[g][e]) & 0x7fffffffu);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        const bool fin = top < 0x7f800000u;
        // 2^14 <= top * mul < 2^15; below 2^-100 the row's scores vanish anyway
        const int ex = max(int(top >> 23) - 127, -100);
        const float mul = fin ? exp2i(14 - ex) : 0.0f;
        if (!fin) {
#pragma unroll
          for (int g = 0; g < kLoads; ++g)
#pragma unroll
            for (int e = 0; e < kElems; ++e) v[g][e] = 0.0f;
        }
        if (lane == 0) {
          if (!fin) m.redo[frag % kTcRedo] = 1;
          m.fac[frag % kTcFrag][row] = a.scale * kLog2e * exp2i(max(ex - 18, -126));
        }
        const int r0 = kSplit ? 2 * row : row;
#pragma unroll
        for (int g = 0; g < kLoads; ++g) {
          const int gi = lane + 32 * g;
          if (gi >= kG) continue;
          uint32_t hi[4], lo[2];
#pragma unroll
          for (int e = 0; e < kElems / 2; ++e) {
            const float x = v[g][2 * e] * mul, y = v[g][2 * e + 1] * mul;
            const __half2 h = __floats2half2_rn(x, y);
            hi[e] = half2_bits(h);
            if (kSplit) lo[e] = half2_bits(__floats2half2_rn(x - __low2float(h), y - __high2float(h)));
          }
          if (kSplit) {  // 4 columns: half a 16-byte piece
            uint8_t* chunk = qs + (gi >> 4) * (kN * 128);
            const int c16 = (gi >> 1) & 7, sub = (gi & 1) * 8;
            *reinterpret_cast<uint2*>(chunk + r0 * 128 + ((c16 ^ (r0 & 7)) << 4) + sub) = make_uint2(hi[0], hi[1]);
            *reinterpret_cast<uint2*>(chunk + (r0 + 1) * 128 + ((c16 ^ ((r0 + 1) & 7)) << 4) + sub) =
                make_uint2(lo[0], lo[1]);
          } else {
            uint8_t* chunk = qs + (gi >> 3) * (kN * 128);
            *reinterpret_cast<uint4*>(chunk + r0 * 128 + (((gi & 7) ^ (r0 & 7)) << 4)) =
                make_uint4(hi[0], hi[1], hi[2], hi[3]);
          }
        }
      }
      }
    };
    int frag = -1;
    auto begin_item = [&](int t0, int nt, int kvh, int ht) {
      ++frag;
      if (frag > 0 && !warp_wait(&m.q_empty, (frag - 1) & 1, a.status)) return false;
      // the mark four fragments on is the one four fragments back, whose rows are out
      if (dw == 0 && lane == 0) m.redo[(frag + 4) % kTcRedo] = 0;
      load_q(t0, nt, kvh, ht, frag);
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&m.q_full[frag % kTcFrag]);
      return true;
    };
    auto step = [&](int n, const Raw& x) {
      const int slot = n % kTcInfo, st = n % kStages;
      const KvTileInfo& f = m.info[slot];
      if (n > 0 && (f.flags & kFragFirst) && !begin_item(f.t0, f.nt, f.kvh, f.ht)) return false;
      __syncwarp();
      if (lane == 0) mbar_arrive(&m.info_empty[slot]);
      bool in = true;
      if (has_k) {
        if (n >= kStages && !warp_wait(&m.k_empty[st], ((n / kStages) - 1) & 1, a.status)) return false;
        uint8_t* row = kring + st * L::kTileBytes + row_at;
#pragma unroll
        for (int u = 0; u < kPer; ++u)
          in = decode_block(x.k[u], x.ks[u], x.seen, on, row + (unit0 + 2 * u) * (2 * kKvTile * 128), at) && in;
        tc::fence_proxy_async_smem();
        if (!in) m.redo[frag % kTcRedo] = 1;
        __syncwarp();
        if (lane == 0) mbar_arrive(&m.k_full[st]);
      }
      if (kSep && has_v) {
        if (n >= kStages && !warp_wait(&m.v_empty[st], ((n / kStages) - 1) & 1, a.status)) return false;
        uint8_t* row = vring + st * L::kTileBytes + row_at;
#pragma unroll
        for (int u = 0; u < kPer; ++u)
          in = decode_block(x.v[u], x.vs[u], x.seen, on, row + (unit0 + 2 * u) * (2 * kKvTile * 128), at) && in;
        tc::fence_proxy_async_smem();
        if (!in) m.redo[frag % kTcRedo] = 1;
        __syncwarp();
        if (lane == 0) mbar_arrive(&m.v_full[st]);
      }
      return true;
    };
    Raw raw[kAhead];
    // the first item's queries while the first rows are looked up
    bool ok = true;
    if (ntiles > 0) ok = begin_item(m.at.item.t0, m.at.item.nt, m.at.kvh, m.at.ht);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (ok && u < ntiles) ok = load(u, raw[u]);
    for (int n0 = 0; ok && n0 < ntiles; n0 += kAhead) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int n = n0 + u;
        if (ok && n < ntiles) ok = step(n, raw[u]);
        if (ok && n + kAhead < ntiles) ok = load(n + kAhead, raw[u]);
      }
    }
  } else {
    // ---------------- softmax, epilogue ----------------
    regs_more<kTcSoftRegs>();
    constexpr int kMax = L::kMax;
    const float inf = __int_as_float(0x7f800000);
    const int quad = warp & 3, half = warp >> 2, bar = 1 + half;
    const int g8 = lane >> 2, c4 = lane & 3;
    const int key0 = quad * 16 + g8;  // this thread's keys: key0 and key0 + 8
    // query row of the thread's entry e
    auto row_of = [&](int e) {
      return half * kRh + (kSplit ? 4 * e + c4 : 8 * (e >> 1) + 2 * c4 + (e & 1));
    };
    const uint32_t tmem_w = tmem + ((uint32_t)(quad * 32) << 16) + half * kNh;
    // Tile n's second product is in O^T.  Once tile n's scores are there, that of
    // n - 2 is (it was issued before them), so the phase of p_empty is never
    // more than one ahead of the one asked for.
    auto product_done = [&](int n) { return warp_wait(&m.p_empty[n & 1], (n >> 1) & 1, a.status); };
    // log2 weight = score * fac + off, off = kLift - the row's running maximum
    float fac[kMax], off[kMax], sum[kMax];
    uint32_t live = 0;  // bit e: the row has seen a key
    int frag = -1;
    int redo = 0;  // the item's rows are to be computed again
    bool ok = true;
    for (int n = 0; n < ntiles; ++n) {
      const int slot = n % kTcInfo, b = n & 1;
      // A wait that runs out clears ok; the next barrier carries that to the
      // half's four warps, which leave together.
      ok = ok && warp_wait(&m.info_full[slot], (n / kTcInfo) & 1, a.status);
      const KvTileInfo& f = m.info[slot];
      const int flags = ok ? f.flags : 0;
      if (flags & kFragFirst) {
        ++frag;
        live = 0;
        ok = ok && warp_wait(&m.q_full[frag % kTcFrag], (frag / kTcFrag) & 1, a.status);
#pragma unroll
        for (int e = 0; e < kMax; ++e) {
          fac[e] = m.fac[frag % kTcFrag][row_of(e)];
          off[e] = 0.0f;
          sum[e] = 0.0f;
        }
      }
      ok = ok && warp_wait(&m.s_full[b], (n >> 1) & 1, a.status);
      tc::fence_after_sync();
      uint32_t raw[16];
      tc::ld_16x256b(tmem_w + L::kTmemS + b * kN, raw);
      tc::wait_ld_of(raw);
      // log2 weights: s[e][0] of key0, s[e][1] of key0 + 8
      float s[kMax][2];
#pragma unroll
      for (int e = 0; e < kMax; ++e)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (kSplit)
            s[e][k] = fmaf(__uint_as_float(raw[4 * e + 2 * k]) + __uint_as_float(raw[4 * e + 2 * k + 1]),
                           fac[e], off[e]);
          else
            s[e][k] = fmaf(__uint_as_float(raw[4 * (e >> 1) + 2 * k + (e & 1)]), fac[e], off[e]);
        }
      if (flags & kTileMasked) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int u = f.u0 + key0 + 8 * k;
          const int i = kv_key(f.head, f.start, u);
          const bool real = f.row[key0 + 8 * k].x >= 0;
#pragma unroll
          for (int e = 0; e < kMax; ++e) {
            const int tok = m.row_tok[row_of(e)];
            bool seen = real;
            if constexpr (Args::kTree) {  // rows past the item's repeat its last token
              seen = seen && kv_tree_sees(a, f.t0 + min(tok, f.nt - 1), i, f.p0, f.last);
            } else {
              const int p = f.p0 + tok;
              seen = seen && i <= p && (a.window == 0 || i > p - a.window || i < a.first);
            }
            if (!seen) s[e][k] = -inf;
          }
        }
      }
      // The running maxima may lag: while no weight is past 2^(kLift + kLag)
      // they stay, and the half's warps need only agree on that.
      float most = -inf;
#pragma unroll
      for (int e = 0; e < kMax; ++e) most = fmaxf(most, fmaxf(s[e][0], s[e][1]));
      bool stay = ok && !(flags & kFragFirst) && most <= kLift + kLag;
      // A row that has seen nothing yet (its tiles so far lay in blocks outside the
      // pool) takes its maximum from the first keys that it sees.
      if (live != (1u << kMax) - 1) {
#pragma unroll
        for (int e = 0; e < kMax; ++e)
          stay = stay && ((live >> e & 1) || fmaxf(s[e][0], s[e][1]) == -inf);
      }
      tc::fence_before_sync();
      if (!bar_and(bar, 128, stay)) {
        // the tile's maxima, over the warp's 16 keys, then over the warps
#pragma unroll
        for (int e = 0; e < kMax; ++e) {
          float t = fmaxf(s[e][0], s[e][1]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
          if (g8 == 0) m.red[0][quad][row_of(e)] = t;
        }
        if (!bar_and(bar, 128, ok)) break;
#pragma unroll
        for (int e = 0; e < kMax; ++e) {
          // by: how far the row's log2 weights move so that the largest so far is kLift.
          // A row that has seen nothing has off = 0 and no sum; one that has, moves down only.
          const int r = row_of(e);
          const float t = fmaxf(fmaxf(m.red[0][0][r], m.red[0][1][r]), fmaxf(m.red[0][2][r], m.red[0][3][r]));
          const bool none = t == -inf, was = live >> e & 1;
          const float by = none ? 0.0f : fminf(kLift - t, was ? 0.0f : inf);
          const float sh = ex2(was ? by : 0.0f);
          live |= none ? 0u : 1u << e;
          off[e] += by;
          s[e][0] += by;
          s[e][1] += by;
          sum[e] *= sh;
          if (quad == 0 && g8 == 0) m.shrink[r] = sh;
        }
        if (!(flags & kFragFirst)) ok = product_done(n - 1);
        tc::fence_after_sync();
        if (!bar_and(bar, 128, ok)) break;
        if (!(flags & kFragFirst)) {
          // O^T shrinks too, now that the previous tile's product is in it
#pragma unroll 1
          for (int c0 = 0; c0 < kNh; c0 += 16)
#pragma unroll 1
            for (int blk = 0; blk < L::kBlocks; ++blk) {
              uint32_t o[16];
              tc::ld_32x32b_x16(tmem_w + L::kTmemO + blk * kN + c0, o);
              tc::wait_ld_of(o);
#pragma unroll
              for (int e = 0; e < 16; ++e)
                o[e] = __float_as_uint(__uint_as_float(o[e]) *
                                       m.shrink[half * kRh + (kSplit ? (c0 + e) >> 1 : c0 + e)]);
              tc::st_32x32b_x16(tmem_w + L::kTmemO + blk * kN + c0, o);
            }
          tc::wait_st();
          tc::fence_before_sync();
          if (!bar_and(bar, 128, ok)) break;  // shrink may be written again
        }
      }
      // weights; their buffer is free: the scores' product was issued after the one that read it
      uint8_t* pt = ps + b * L::kPBytes;
#pragma unroll
      for (int e = 0; e < kMax; ++e) {
        s[e][0] = ex2(s[e][0]);
        s[e][1] = ex2(s[e][1]);
        sum[e] += s[e][0] + s[e][1];
      }
#pragma unroll
      for (int j = 0; j < kNh / 8; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t bits;
          if (kSplit) {
            const float p = s[j][k];
            const __half hi = __float2half_rn(p);
            bits = half2_bits(__halves2half2(hi, __float2half_rn((p - __half2float(hi)) * kLoUp)));
          } else {
            bits = half2_bits(__floats2half2_rn(s[kSplit ? 0 : 2 * j][k], s[kSplit ? 0 : 2 * j + 1][k]));
          }
          const int key = key0 + 8 * k, piece = half * (kNh / 8) + j;
          *reinterpret_cast<uint32_t*>(pt + key * 128 + ((piece ^ (key & 7)) << 4) + 4 * c4) = bits;
        }
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&m.p_full[b]);

      if (flags & kFragLast) {
        // ---- the fragment's sums, then its rows: out, or a partial slot ----
#pragma unroll
        for (int e = 0; e < kMax; ++e) {
          float t = sum[e];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
          if (g8 == 0) {
            m.red[1][quad][row_of(e)] = t;
            if (quad == 0) m.top[row_of(e)] = live >> e & 1 ? kLift - off[e] : -inf;
          }
        }
        ok = product_done(n);
        tc::fence_after_sync();
        if (!bar_and(bar, 128, ok)) break;
        const bool cut = L::kFold && (flags & kFragCut), cont = L::kFold && (flags & kFragCont);
        const bool whole = (flags & kItemFirst) && (flags & kItemLast) && !cut;
        redo = (cont ? redo : 0) | m.redo[frag % kTcRedo];
        const int rows = w.ht > 1 ? min(kRn, a.group - f.ht * kRn) : f.nt * a.group;
        const int row = half * kRh + quad * 32 + lane;
        if (quad * 32 + lane < kRh && row >= rows) m.out_row[row] = 0;
        const int part = 2 * blockIdx.x + (flags & kSlot1 ? 1 : 0);
        if (quad * 32 + lane < kRh && row < rows) {
          const int h = f.kvh * a.group + f.ht * kRn + m.row_head[row];
          const int t = f.t0 + m.row_tok[row];
          float l = (m.red[1][0][row] + m.red[1][1][row]) + (m.red[1][2][row] + m.red[1][3][row]);
          float top = m.top[row];
          float os = 1.0f / 16.0f;  // the tiles hold 16 times the values
          float keep = 0.0f;        // by what the earlier fragments' sums are multiplied
          if (cont) {  // this thread wrote them
            const float2 x = w.part_ml[(long long)part * kRn + row];
            const float to = fmaxf(top, x.x), base = to == -inf ? 0.0f : to;
            const float now = top == -inf ? 0.0f : ex2(top - base);
            keep = x.x == -inf ? 0.0f : ex2(x.x - base);
            os *= now;
            l = l * now + x.y * keep;
            top = to;
          }
          if (whole) {
            float z = l;
            if (a.sink) {
              const float sk = a.sink[h] * kLog2e;
              const float to = fmaxf(top, sk), base = to == -inf ? 0.0f : to;
              const float sh = top == -inf ? 0.0f : ex2(top - base);
              os *= sh;
              keep *= sh;
              z = l * sh + ex2(sk - base + kLift);
            }
            os = z == 0.0f ? 0.0f : os / z;
            keep = z == 0.0f ? 0.0f : keep / z;
            m.out_row[row] = t * a.out_token_stride + h * a.out_head_stride;
          } else {
            w.part_ml[(long long)part * kRn + row] = make_float2(top, l);
            m.out_row[row] = ((long long)part * kRn + row) * kD;
            if (row == 0) w.part_redo[part] = redo;
          }
          m.out_scale[row] = os;
          m.shrink[row] = keep;
          if ((flags & kItemFirst) && !cut) {  // where the item's parts lie
            const int parts =
                whole ? 1 : KvCut(w, m.at.total).cta_of(f.first + f.tiles - 1) - (int)blockIdx.x + 1;
            w.meta[(long long)t * a.heads + h] =
                make_int4(blockIdx.x, parts, (flags & kSlot1 ? 1 : 0) | row << 1, redo);
          }
        }
        if (!bar_and(bar, 128, ok)) break;
        const int dim = quad * 32 + lane;
        // eight rows at a time, a 128-row block of O^T after the other
        auto sums = [&](int r0, int blk, float (&v)[8]) {
          const uint32_t at = tmem_w + L::kTmemO + (r0 - half * kRh) * (kSplit ? 2 : 1) + blk * kN;
          if (kSplit) {
            uint32_t o[16];
            tc::ld_32x32b_x16(at, o);
            tc::wait_ld_of(o);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = fmaf(__uint_as_float(o[2 * e + 1]), 1.0f / kLoUp, __uint_as_float(o[2 * e]));
          } else {
            uint32_t o[8];
            tc::ld_32x32b_x8(at, o);
            tc::wait_ld_of(o);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(o[e]);
          }
        };
        auto write = [&](auto* out) {
          if (kD < 128 && quad * 32 >= kD) return;
#pragma unroll 1
          for (int r0 = half * kRh; r0 < half * kRh + kRh; r0 += 8) {
            if (r0 >= rows) break;
            long long to[8];
            float by[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              to[e] = m.out_row[r0 + e] + dim;
              by[e] = m.out_scale[r0 + e];
            }
            const int live = rows - r0;
#pragma unroll 1
            for (int blk = 0; blk < L::kBlocks; ++blk) {
              float v[8];
              sums(r0, blk, v);
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (e < live) kv_put(out + to[e] + blk * 128, v[e] * by[e]);
            }
          }
        };
        // The same with what this thread has left in the partial slot, which goes on from
        // there (f32 queries: so does the output).
        auto add = [&](float* out) {
          if (kD < 128 && quad * 32 >= kD) return;
#pragma unroll 1
          for (int r0 = half * kRh; r0 < half * kRh + kRh; r0 += 8) {
            if (r0 >= rows) break;
            const float* at = w.part_o + ((long long)part * kRn + r0) * kD + dim;
            const int live = rows - r0;
            float old[L::kBlocks][8];
#pragma unroll
            for (int blk = 0; blk < L::kBlocks; ++blk)
#pragma unroll
              for (int e = 0; e < 8; ++e) old[blk][e] = e < live ? at[e * kD + blk * 128] : 0.0f;
#pragma unroll
            for (int blk = 0; blk < L::kBlocks; ++blk) {
              float v[8];
              sums(r0, blk, v);
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (e < live)
                  out[m.out_row[r0 + e] + dim + blk * 128] =
                      fmaf(old[blk][e], m.shrink[r0 + e], v[e] * m.out_scale[r0 + e]);
            }
          }
        };
        // rows to be computed again are left alone: out may be q, which that still reads
        if (cont) {
          if (!whole || !redo) add(whole ? static_cast<float*>(a.out) : w.part_o);
        } else if (!whole) {
          write(w.part_o);
        } else if (!redo) {
          if (kSplit)
            write(static_cast<float*>(a.out));
          else if (a.dtype == WH_DTYPE_BF16)
            write(static_cast<__nv_bfloat16*>(a.out));
          else
            write(static_cast<__half*>(a.out));
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&m.o_empty);
        if (!bar_and(bar, 128, ok)) break;  // sums and row tables may be written again
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

template <int kD, bool kSplit, bool kSep, class Args>
static cudaError_t launch_attend_tc(const Args& a, const KvWork& w, cudaStream_t s, bool pdl) {
  const size_t smem = KvTcSmem<kD, kSplit, kSep>::kBytes;
  if (w.rn != KvTc<kD, kSplit>::kRn) return cudaErrorInvalidValue;
  const cudaError_t e = ensure_smem(kv_attend_tc_kernel<kD, kSplit, kSep, Args>, smem);
  if (e != cudaSuccess) return e;
  return launch_pdl(kv_attend_tc_kernel<kD, kSplit, kSep, Args>, dim3(w.ctas), kTcThreads, smem, s, pdl, a, w);
}

}  // namespace wh
