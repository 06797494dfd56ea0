// fp8_gemm.cu -- FP8 E4M3 x UE8M0(128 x 128) matrix products of many tokens on
// the 5th-generation tensor cores.
//
//   y[t][r] = sum_c W[r][c] 2^(S[r/128][c/128] - 127) aq(x[t])[c]
//
// aq is the framework's FP8 act quant (common.cuh) per block of 32, 64 or 128
// values: both operands are E4M3 codes with a power-of-two scale, so a
// kind::mxf8f6f4 product is exact and only the sums round.  Two launches:
// fp8_quant_kernel writes the tokens' codes and their scale bytes in the order
// in which the product's scale copies read them; then the product, by clusters that
// share a tile's K (fp8_gemm_kernel: few tiles, a token or two quantised on the way) or
// by pairs of CTAs (fp8_gemm_pair_kernel: many).
//
// The weight is the M operand (128 rows of it a tile), so that one token costs
// N = 16 columns and not 128 rows.  Its scale is one byte for a tile of 128 x 128: 512
// equal bytes in the tensor core's layout, copied from a table of 256 such rows.
//
// Measured, quantisation included (inputs of three calls in turn): 8192 tokens x 4096 x
// 8192 in bf16 233 us (2360 TFLOP/s), in f32 270 (315 after a second of such calls, at the clock
// of 1.44 GHz that the power limit then leaves); 2048 in bf16 72; 509 in bf16 24.5; one token x
// 4096 x 4096 6.7.  The quantisation of 8192 x 8192 f32 is 57 us of it (51 at the copy's rate), its
// product 200: the tensor pipe is active in 77 % of the cycles, at a clock that the power limit
// holds at 1.55 GHz.
#include <cuda_bf16.h>

#include "kvcache.cuh"
#include "mm_steps.cuh"
#include "tc.cuh"

namespace wh {

struct Fp8GemmArgs {
  const uint8_t* scale;  // [ceil(rows/128)][ktiles]
  const uint8_t* sf_rows;  // wh_ctx's: 512 times each byte
  const uint8_t* xsf;    // [ntiles][ktiles][512, or 1024 for tiles of more than 128 tokens]
  void* y;
  long long ldy;
  int rows, tokens, ktiles;
  int dtype;   // of y
  int fold;    // K tiles that a sum runs through the tensor core before it is added in f32 (kMmFold)
  int mtiles, ntiles;
  bool boxes;  // y is written in boxes (its rows start on 16 bytes)
  // a call that quantises inside the product
  const void* x;
  long long ldx;
  int cols, lanes;  // lanes: 8 values each, of a block
  uint32_t* status;
};

// ---------------------------------------------------------------------------
// act quant: a thread takes 8 values, a block of 32/64/128 is 4/8/16 lanes.
// Reads tokens * cols values, writes a byte each and a scale byte for 32.
// ---------------------------------------------------------------------------
struct Fp8QuantArgs {
  const void* x;
  long long ldx;
  int tokens, cols, ktiles;
  int tile, shift;  // tokens of the product's tile; their logarithm, of 224 none
  uint8_t* xq;   // [tokens][cols]
  uint8_t* xsf;
};
constexpr int kQuantThreads = 256;

// v * inv (a power of two) as one rounded to the nearest E4M3, ties to even, has to be for the
// act quant's ties to the lower: the f32 below it, so that a tie is none any more.  For
// that to reach no tie itself, an f32's last bit goes into the one above it first (16-bit
// types have none).  A zero becomes -0.
template <bool kF32>
__device__ __forceinline__ float fp8_below(float v, float inv) {
  if (kF32) {
    const uint32_t u = __float_as_uint(v);
    v = __uint_as_float((u & ~1u) | (u << 1 & 2u));
  }
  return __fmaf_rd(v, inv, -7.888609052210118e-31f);  // 2^-100
}

// An amax's scale byte k + 127, and 2^-k (aq_block_scale)
__device__ __forceinline__ float fp8_block_scale(float amax, uint32_t& byte) {
  const uint32_t u = __float_as_uint(fmaxf(amax, 1.0e-4f)), e = u >> 23;
  byte = e == 255 ? 255 : e - 8 + (u > c_aq_top[e]);  // an infinite block's is 255, the product's NaN
  return e == 255 ? 0.0f : __uint_as_float((254 - byte) << 23);
}
// 8 values of a block that `lanes` lanes share -> codes (NaN of a NaN); byte: the block's
// scale.  Every lane of the warp calls it.  Instructions count: with the rounding by cases
// (grouped.cu) and a division a block 50 a value, and 8192 x 8192 f32 took 118 us.
template <bool kF32>
__device__ __forceinline__ uint2 fp8_quant8(const float (&v)[8], int lanes, uint32_t& byte) {
  float m = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[j]));  // passes over NaN
  for (int o = 1; o < lanes; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float inv = fp8_block_scale(m, byte);
  uint2 w;
  auto two = [&](int j) { return e4m3x2_rn(fp8_below<kF32>(v[j], inv), fp8_below<kF32>(v[j + 1], inv)); };
  w.x = two(0) | two(2) << 16;
  w.y = two(4) | two(6) << 16;
  return w;
}

// kLanes: 4, 8 or 16 a block
template <class T, int kLanes>
__global__ void __launch_bounds__(kQuantThreads) fp8_quant_kernel(Fp8QuantArgs a) {
  pdl_wait_prior();
  pdl_launch_dependents();  // what came before is complete: the product may start on its weights
  const int part = blockIdx.x * kQuantThreads + threadIdx.x, col = part * 8;
  const bool in = part < a.ktiles * 16, on = col < a.cols;  // cols is a multiple of 16
  for (uint32_t t = blockIdx.y; t < (uint32_t)a.tokens; t += gridDim.y) {
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (on) kv_load8(static_cast<const T*>(a.x) + t * a.ldx + col, v);
    uint32_t byte;
    const uint2 w = fp8_quant8<std::is_same<T, float>::value>(v, kLanes, byte);
    if (on) *reinterpret_cast<uint2*>(a.xq + (long long)t * a.cols + col) = w;
    if (in && (part & 3) == 0) {  // groups past the row's end get 2^0
      const uint32_t nt = a.shift ? t >> a.shift : t / 224, r = t - nt * a.tile;
      uint8_t* at = a.xsf + ((long long)nt * a.ktiles + (part >> 4)) * (a.tile > 128 ? 1024 : 512) + (r >> 7) * 512 +
                    (r & 31) * 16 + (r >> 5 & 3) * 4;
      at[(part >> 2) & 3] = on ? uint8_t(byte) : 127;
    }
  }
}
template <class T>
static cudaError_t launch_fp8_quant(const Fp8QuantArgs& a, int lanes, dim3 grid, cudaStream_t s, bool pdl) {
  return lanes == 4   ? launch_pdl(fp8_quant_kernel<T, 4>, grid, kQuantThreads, 0, s, pdl, a)
         : lanes == 8 ? launch_pdl(fp8_quant_kernel<T, 8>, grid, kQuantThreads, 0, s, pdl, a)
                      : launch_pdl(fp8_quant_kernel<T, 16>, grid, kQuantThreads, 0, s, pdl, a);
}

// ---------------------------------------------------------------------------
// product
// ---------------------------------------------------------------------------
constexpr int kMmWeight = 128 * 128;  // a weight tile: 128 rows x 128 K
constexpr int kMmEpi = 8;             // epilogue warps: TMEM quadrant w % 4, column half w / 4
constexpr int kMmMma = kMmEpi, kMmWeights = kMmEpi + 1, kMmTokens = kMmEpi + 2;
constexpr int kMmThreads = (kMmEpi + 3) * 32;
// A sum that runs through the tensor core is cut off with each instruction of 32 columns, always
// downwards.  Measured with terms of one sign, relative to the sum (of mixed signs: to its
// largest partial sum, so cancellation enlarges it relative to the result): 1024 columns lose
// 1.9e-6 on average and 3.6e-6 at most, 8192 lose 1.4e-5 to 1.9e-5, 32768 7.8e-5, 393216 1.1e-3.
// f32 outputs are therefore added in f32 after kMmFold K tiles (1024 columns), 16-bit ones
// after kMmFold16 (8192 columns): a twenty-fifth of f16's rounding, 2^-11.  32768 columns would be
// a sixth, and were no faster (509 tokens x 4096 x 32768 bf16 76.8 us, by 8192 columns 76.7).
constexpr int kMmFold = 8, kMmFold16 = 64;
constexpr int kMmBox = 16;   // tokens of an output box
constexpr int kMmMost = 1 << 30;  // rows, columns, tokens: rounded up to tiles they fit an int
constexpr int kMmShare = 8;  // most CTAs that share a tile's K

template <int kN>
struct Mm {
  static_assert(kN <= 128, "one block of scales a tile");
  static constexpr int kTokens = kN * 128;             // bytes of a token tile
  static constexpr int kStage = kMmWeight + kTokens;
  static constexpr int kSfb = 512, kSf = kSfb + 512;   // the tokens' scales, the weight's
  static constexpr int kStages = kN >= 128 ? 6 : 4;
  static constexpr int kAcc = 2;                       // accumulator sets
  static constexpr int kSfCols = 8;                    // TMEM columns of a set of scales
  static constexpr int kNeed = kAcc * kN + 2 * kSfCols;
  static constexpr int kCols = kNeed <= 64 ? 64 : kNeed <= 128 ? 128 : kNeed <= 256 ? 256 : 512;
  static constexpr int kPer = kN / 2;                  // columns of an epilogue warp
  struct Misc {
    uint64_t full[kStages], empty[2 * kStages], acc_full[kAcc], acc_empty[kAcc], done;
    uint32_t tmem;
  };
  static constexpr int kBytes = 1024 + kStages * (kStage + kSf) + (int)sizeof(Misc);
  static_assert(kBytes <= 232448 && kNeed <= 512, "shared memory or TMEM");
  static_assert(kN * 128 * 4 <= kStages * kStage, "a partial sum fits the ring");
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr, uint32_t rank) {
  float4 v;
  asm volatile("{ .reg .b32 a; mapa.shared::cluster.u32 a, %4, %5; ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a]; }"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr), "r"(rank)
               : "memory");
  return v;
}
// asks L2 for a box
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int32_t c0, int32_t c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ void mm_put(void* y, long long at, int dtype, float v) {
  if (dtype == WH_DTYPE_F32)
    static_cast<float*>(y)[at] = v;
  else if (dtype == WH_DTYPE_BF16)
    static_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(y)[at] = __float2half_rn(v);
}

__device__ __forceinline__ void mm_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void mm_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void mm_put(__half* p, float v) { *p = __float2half_rn(v); }
// 2-D tiled store; the box may reach past the tensor's ends.  What lies past the end of a row is
// left out by 16 bytes: up to there zeros are written behind a row that ends in between.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int32_t c0, int32_t c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ void bulk_stores_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// at most the last of this thread's groups of bulk stores still reads shared memory
__device__ __forceinline__ void bulk_stores_read() { asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory"); }
__device__ __forceinline__ void bulk_stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// Row `row` of tokens n0 .. as mm_store writes it, by the four warps of a column half together: 16
// tokens x 128 rows at a time through shared memory (two buffers at outs, in turn), written by
// bulk stores.  All four call it (mm_tile).  Whole lines: a
// warp's own stores are 64 or 128 bytes at a token, which took 6.7 us a tile of 128 x 224
// in bf16, more than its products over 1024 columns.
template <class T, int kPer>
__device__ __forceinline__ void mm_store_boxes(const Fp8GemmArgs& a, const CUtensorMap* ymap, uint8_t* outs,
                                               int& turn, int row, int n0, const float (&acc)[kPer]) {
  const int warp = threadIdx.x >> 5, bar = 1 + (warp >> 2), in = row & 127, row0 = row - in;
  if (row0 >= a.rows) return;  // the whole half
#pragma unroll
  for (int c = 0; c < kPer; c += kMmBox, turn ^= 1) {
    T* box = reinterpret_cast<T*>(outs + turn * (kMmBox * 128 * 4));
    if (in == 0) bulk_stores_read();  // of the box before the last one, which lay here
    asm volatile("bar.sync %0, 128;" ::"r"(bar) : "memory");
#pragma unroll
    for (int e = 0; e < kMmBox; ++e) mm_put(box + e * 128 + in, acc[c + e]);
    tc::fence_proxy_async_smem();
    asm volatile("bar.sync %0, 128;" ::"r"(bar) : "memory");
    if (in == 0) {  // a group for each box, so that the wait above counts boxes
      if (n0 + c < a.tokens) tma_store_2d(ymap, box, row0, n0 + c);
      bulk_stores_commit();
    }
  }
}

// Whether all four warps of a column half say so (named barrier `bar`)
__device__ __forceinline__ bool mm_all_of_half(int bar, bool ok) {
  uint32_t all;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %2, 0;\n bar.red.and.pred q, %1, 128, p;\n"
      " selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(all)
      : "r"(bar), "r"((uint32_t)ok)
      : "memory");
  return all != 0;
}

// A place in a ring of kCount stages
template <int kCount>
struct MmRing {
  int s = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++s == kCount) {
      s = 0;
      phase ^= 1;
    }
  }
};

// A warp's kPer accumulator columns, added to acc (or into it, the first time)
template <int kPer>
__device__ __forceinline__ void mm_sum(uint32_t at, float (&acc)[kPer], bool first) {
  if constexpr (kPer < 16) {
    uint32_t v[8];
    tc::ld_32x32b_x8(at, v);
    tc::wait_ld_of(v);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = first ? __uint_as_float(v[e]) : acc[e] + __uint_as_float(v[e]);
  } else {
#pragma unroll
    for (int c = 0; c < kPer; c += 32) {
      uint32_t v[16], u[16];
      tc::ld_32x32b_x16(at + c, v);
      if (c + 16 < kPer) tc::ld_32x32b_x16(at + c + 16, u);
      tc::wait_ld_of(v);
      if (c + 16 < kPer) tc::wait_ld_of(u);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        acc[c + e] = first ? __uint_as_float(v[e]) : acc[c + e] + __uint_as_float(v[e]);
        if (c + 16 < kPer)
          acc[(c + 16 + e) % kPer] = first ? __uint_as_float(u[e]) : acc[(c + 16 + e) % kPer] + __uint_as_float(u[e]);
      }
    }
  }
}
// Row `row` of tokens n0 ..: a warp's lanes are neighbours in y
template <int kPer>
__device__ __forceinline__ void mm_store(const Fp8GemmArgs& a, int row, int n0, const float (&acc)[kPer]) {
#pragma unroll
  for (int c = 0; c < kPer; ++c)
    if (row < a.rows && n0 + c < a.tokens) mm_put(a.y, (n0 + c) * a.ldy + row, a.dtype, acc[c]);
}

// The scale bytes of a row of weight tiles, 32 of which a warp reads at a time,
// ahead of their use.
struct MmScales {
  const uint8_t* row;
  int k0, k1;
  uint32_t mine, next;
  __device__ __forceinline__ MmScales(const uint8_t* row_, int k0_, int k1_) : row(row_), k0(k0_), k1(k1_) {
    mine = read(k0);
    next = read(k0 + 32);
  }
  __device__ __forceinline__ uint32_t read(int k) const {
    const int i = k + (threadIdx.x & 31);
    return i < k1 ? __ldg(row + i) : 0;
  }
  // for K tiles in order; the whole warp calls it
  __device__ __forceinline__ uint32_t at(int kt) {
    if (kt - k0 >= 32) {
      k0 += 32;
      mine = next;
      next = read(k0 + 32);
    }
    return __shfl_sync(0xffffffffu, mine, kt - k0);
  }
};

// One tile a cluster: its CTAs share the tile's K and add their sums through
// distributed shared memory, in the order of their ranks.  X: the epilogue's warps
// quantise the tokens (of type X) themselves, a K tile each, while the weight arrives;
// void: fp8_quant_kernel has.  The columns of tokens past the last one hold what the
// shared memory held, and nothing of them is stored.
template <int kN, class X>
__global__ void __launch_bounds__(kMmThreads, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                    Fp8GemmArgs a) {
  using L = Mm<kN>;
  constexpr int kStages = L::kStages, kAcc = L::kAcc, kPer = L::kPer;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* ring = align_smem_1024(smem_raw);
  uint8_t* sfs = ring + kStages * L::kStage;
  typename L::Misc& m = *reinterpret_cast<typename L::Misc*>(sfs + kStages * L::kSf);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr bool kQuant = !std::is_same<X, void>::value;
  static_assert(!kQuant || kN == 16, "few tokens");
  using Free = MmFree<kStages, kQuant ? 2 * kStages : kStages>;
  const int rank = (int)cluster_rank(), share = (int)cluster_size();

  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&m.full[i], 2);
      mbar_init(&m.empty[i], 1);
      mbar_init(&m.empty[kStages + i], 1);
    }
    for (int i = 0; i < kAcc; ++i) {
      mbar_init(&m.acc_full[i], 1);
      mbar_init(&m.acc_empty[i], kMmEpi);
    }
    mbar_init(&m.done, 1);
    fence_barrier_init();
  }
  if (warp == kMmMma) {
    tc::tmem_alloc(&m.tmem, L::kCols);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = m.tmem;
  const int tile = blockIdx.x / share, mt = tile % a.mtiles, n0 = tile / a.mtiles * kN;
  // this CTA's K tiles
  const int k0 = int((long long)a.ktiles * rank / share), k1 = int((long long)a.ktiles * (rank + 1) / share);

  // Loads: a warp for the weight and its scales, one for the tokens' codes and theirs
  // (a copy costs its issuing warp some 50 to 100 cycles; elect_one keeps its operands in
  // uniform registers, without which it is several hundred).
  if (warp == kMmWeights) {
    int g = 0;
    MmRing<kStages> at;
    bool ok = true;
    if (tc::elect_one()) {
      prefetch_tensormap(&wmap);
      // What came before need not be complete here: nothing is read, L2 is only asked for it.
      if (kQuant)
        for (int kt = k0; kt < min(k1, k0 + kStages); ++kt) tma_prefetch_2d(&wmap, kt * 128, mt * 128);
    }
    __syncwarp();
    if (kQuant) pdl_wait_prior();
    MmScales sc(a.scale + (long long)mt * a.ktiles, k0, k1);
    for (int kt = k0; kt < k1; ++kt, ++g, at.next()) {
      const int s = at.s;
      const uint32_t byte = sc.at(kt);
      if (g >= kStages) ok = mbar_wait_warp(&m.empty[Free::bar(g - kStages)], Free::parity(g - kStages), a.status);
      if (!ok) break;
      if (tc::elect_one()) {
        mbar_arrive_expect_tx(&m.full[s], kMmWeight + 512);
        tma_load_2d(ring + s * L::kStage, &wmap, &m.full[s], kt * 128, mt * 128);
        bulk_load(sfs + s * L::kSf + L::kSfb, a.sf_rows + byte * 512, 512, &m.full[s]);
      }
      __syncwarp();
    }
    pdl_wait_prior();
    // no copy may be in flight when the CTA exits
    for (int i = max(0, g - kStages); i < g; ++i)
      if (!mbar_drain(&m.full[i % kStages], (i / kStages) & 1, a.status)) break;
  } else if (!kQuant && warp == kMmTokens) {
    int g = 0;
    MmRing<kStages> at;
    bool ok = true;
    if (tc::elect_one()) prefetch_tensormap(&xmap);
    __syncwarp();
    pdl_wait_prior();
    const uint8_t* sf = a.xsf + (long long)(tile / a.mtiles) * a.ktiles * 512;
    for (int kt = k0; kt < k1; ++kt, ++g, at.next()) {
      const int s = at.s;
      if (g >= kStages) ok = mbar_wait_warp(&m.empty[Free::bar(g - kStages)], Free::parity(g - kStages), a.status);
      if (!ok) break;
      if (tc::elect_one()) {
        mbar_arrive_expect_tx(&m.full[s], L::kTokens + L::kSfb);
        tma_load_2d(ring + s * L::kStage + kMmWeight, &xmap, &m.full[s], kt * 128, n0);
        bulk_load(sfs + s * L::kSf, sf + (long long)kt * 512, 512, &m.full[s]);
      }
      __syncwarp();
    }
    for (int i = max(0, g - kStages); i < g; ++i)
      if (!mbar_drain(&m.full[i % kStages], (i / kStages) & 1, a.status)) break;
  } else if (warp == kMmMma) {
    // ---------------- MMA ----------------
    int chunk = 0;
    MmRing<kStages> at;
    bool ok = true;
    for (int c0 = k0; ok && c0 < k1; c0 += a.fold, ++chunk) {
      const int b = chunk % kAcc;
      if (chunk >= kAcc) ok = mbar_wait_warp(&m.acc_empty[b], ((chunk / kAcc) - 1) & 1, a.status);
      if (!ok) break;
      tc::fence_after_sync();
      const uint32_t acc = tmem + b * kN;
      const int c1 = min(k1, c0 + a.fold);
      for (int kt = c0; kt < c1; ++kt, at.next()) {
        const int s = at.s;
        ok = mbar_wait_warp(&m.full[s], at.phase, a.status);
        if (!ok) break;
        tc::fence_after_sync();
        if (tc::elect_one()) {
          const uint32_t wsf = tmem + kAcc * kN + (kt & 1) * L::kSfCols, xsf = wsf + 4;
          const uint32_t sf = smem_u32(sfs + s * L::kSf);
          tc::cp_sf_block(wsf, tc::desc_sf_block(sf + L::kSfb));
          tc::cp_sf_block(xsf, tc::desc_sf_block(sf));
          const uint64_t dw = tc::desc_sw128(smem_u32(ring + s * L::kStage));
          const uint64_t dx = tc::desc_sw128(smem_u32(ring + s * L::kStage + kMmWeight));
#pragma unroll
          for (int k = 0; k < 4; ++k)
            tc::mma_mxf8(acc, dw + 2 * k, dx + 2 * k, tc::idesc_mxf8(kN, k, k), wsf | (uint32_t(k) << 30),
                         xsf | (uint32_t(k) << 30), kt != c0 || k != 0);
          tc::commit(&m.empty[Free::bar(kt - k0)]);
        }
        __syncwarp();
      }
      if (ok && tc::elect_one()) tc::commit(&m.acc_full[b]);
      __syncwarp();
    }
    // every product has finished before TMEM is released
    if (tc::elect_one()) tc::commit(&m.done);
    __syncwarp();
    mbar_wait(&m.done, 0, a.status);
  } else if (warp < kMmEpi) {
    pdl_wait_prior();
    const int quad = warp & 3, half = warp >> 2;
    const uint32_t at_acc = tmem + ((uint32_t)(quad * 32) << 16) + half * kPer;
    float acc[kPer];
    bool ok = true;
    int c0 = k0, chunk = 0;  // the next sum to be taken from the tensor core
    auto take = [&] {
      const int b = chunk % kAcc;
      ok = __all_sync(0xffffffffu, mbar_wait(&m.acc_full[b], (chunk / kAcc) & 1, a.status));
      if (!ok) return;
      tc::fence_after_sync();
      mm_sum<kPer>(at_acc + b * kN, acc, c0 == k0);
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&m.acc_empty[b]);
      c0 += a.fold;
      ++chunk;
    };
    if constexpr (kQuant) {
      // ---------------- the tokens' codes: every eighth K tile, two tokens at a time ----------------
      const int part = lane & 15;
      const X* x = static_cast<const X*>(a.x);
      auto load = [&](int kt, int t, KvRaw8<X>& raw) {
        const int col = kt * 128 + part * 8;
        const bool on = t < a.tokens && kt < k1 && col < a.cols;
        if (on) raw.load(x + t * a.ldx + col);
        return on;
      };
      KvRaw8<X> next;
      bool next_on = load(k0 + warp, lane >> 4, next);
      for (int g = warp; ok && k0 + g < k1; g += kMmEpi) {
        const int kt = k0 + g, s = g % kStages;
        // The product goes on to sum `chunk` + 2 only after sum `chunk` has been taken, for
        // which it has (or gets from the other warps) all of the codes.
        while (ok && kt - c0 >= kAcc * a.fold) take();
        // two warps fill a stage in turn (MmFree)
        static_assert(kMmEpi == 2 * L::kStages || !kQuant, "every second tile of a stage is this warp's");
        if (ok && g >= kStages)
          ok = mbar_wait_warp(&m.empty[Free::bar(g - kStages)], Free::parity(g - kStages), a.status);
        if (!ok) break;
        for (int p = 0; 2 * p < a.tokens; ++p) {
          const int t = 2 * p + (lane >> 4);
          const bool on = next_on, last = 2 * p + 2 >= a.tokens;
          float v[8];
          next.widen(v);
          next_on = load(last ? kt + kMmEpi : kt, last ? lane >> 4 : t + 2, next);
          if (!on) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.0f;
          }
          uint32_t byte;
          const uint2 w = fp8_quant8<std::is_same<X, float>::value>(v, a.lanes, byte);
          *reinterpret_cast<uint2*>(ring + s * L::kStage + kMmWeight + t * 128 + ((part >> 1 ^ (t & 7)) << 4) +
                                    (part & 1) * 8) = w;
          if ((part & 3) == 0) sfs[s * L::kSf + t * 16 + (part >> 2)] = on ? uint8_t(byte) : 127;
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&m.full[s]);
      }
    }
    // ---------------- epilogue ----------------
    while (ok && c0 < k1) take();
    // the ring is idle: every product that reads it has finished
    float* part = reinterpret_cast<float*>(ring) + half * kPer * 128 + quad * 32 + lane;
    if (ok) {
#pragma unroll
      for (int c = 0; c < kPer; ++c) part[c * 128] = acc[c];
    }
  }
  __syncwarp();
  cluster_sync_all();
  // this CTA's share of the tile, four rows of a token a thread, added in the order of the ranks
  for (int i = rank * kMmThreads + tid; i < kN * 32; i += share * kMmThreads) {
    const int row = mt * 128 + (i & 31) * 4, n = n0 + (i >> 5);
    if (row >= a.rows || n >= a.tokens) continue;
    const uint32_t from = smem_u32(ring) + i * 16;
    float4 v[kMmShare];
#pragma unroll
    for (int r = 0; r < kMmShare; ++r) v[r] = r < share ? ld_cluster4(from, r) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float4 sum = v[0];
#pragma unroll
    for (int r = 1; r < kMmShare; ++r)
      if (r < share) sum = make_float4(sum.x + v[r].x, sum.y + v[r].y, sum.z + v[r].z, sum.w + v[r].w);
    const long long to = n * a.ldy + row;
    if (a.boxes && row + 4 <= a.rows) {
      if (a.dtype == WH_DTYPE_F32)
        kv_store4(static_cast<float*>(a.y) + to, sum, 1.0f);
      else if (a.dtype == WH_DTYPE_BF16)
        kv_store4(static_cast<__nv_bfloat16*>(a.y) + to, sum, 1.0f);
      else
        kv_store4(static_cast<__half*>(a.y) + to, sum, 1.0f);
    } else {
      const float one[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (row + e < a.rows) mm_put(a.y, to + e, a.dtype, one[e]);
    }
  }
  cluster_sync_all();  // the others have read this CTA's sums
  pdl_launch_dependents();
  tc::fence_before_sync();
  __syncthreads();
  if (warp == kMmMma) tc::tmem_dealloc(tmem, L::kCols);
}

// ---------------------------------------------------------------------------
// The product on pairs of CTAs (cta_group::2): 256 weight rows x kN tokens a tile.
// Each CTA of a pair holds 128 of the rows and half of the tokens' codes, so a
// byte of shared memory feeds twice the operations, and both halves of the tile
// come from L2 once.  The even CTA's MMA warp issues for both; its barriers count
// both CTAs' bytes.
// ---------------------------------------------------------------------------
template <int kN>
struct MmPair {
  static constexpr int kTokens = kN / 2 * 128;
  static constexpr int kStage = kMmWeight + kTokens;
  static constexpr int kSfb = kN > 128 ? 1024 : 512;
  static constexpr int kSf = kSfb + 512;
  static constexpr int kStages = kN > 128 ? 6 : 7;
  static constexpr int kAcc = 2;
  static constexpr int kSfCols = kSfb / 128 + 4;
  static constexpr int kCols = 512;
  static constexpr int kPer = kN / 2;
  struct Misc {
    uint64_t full[kStages], empty[kStages], acc_full[kAcc], acc_empty[kAcc], done;
    uint32_t tmem;
  };
  // outputs on their way out: [column half][2][16 tokens][128 rows]
  static constexpr int kOut = 4 * kMmBox * 128 * 4;
  static constexpr int kBytes = 1024 + kStages * (kStage + kSf) + kOut + (int)sizeof(Misc);
  static_assert(kBytes <= 232448 && kAcc * kN + 2 * kSfCols <= kCols, "shared memory or TMEM");
  static_assert(kN % 32 == 0 && kTokens % 1024 == 0, "product shape, alignment of a stage");
};

__device__ __forceinline__ uint32_t map_to_rank(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
// arrive on a barrier of the cluster (an address of map_to_rank)
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// mbar_wait_warp on a barrier that the other CTA of the cluster arrives on
__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t* bar, uint32_t phase) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(phase)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_wait_warp_cluster(uint64_t* bar, uint32_t phase, uint32_t* status) {
  if (__all_sync(0xffffffffu, mbar_try_wait_cluster(bar, phase))) return true;
  const uint64_t start = globaltimer();
  while (!__all_sync(0xffffffffu, mbar_try_wait_cluster(bar, phase))) {
    if (__any_sync(0xffffffffu, globaltimer() - start > WH_WAIT_NS)) {
      if ((threadIdx.x & 31) == 0) flag(status, WH_DEV_TIMEOUT);
      return false;
    }
  }
  return true;
}
// 2-D tiled load into this CTA's shared memory that counts on a barrier of either
// CTA of the pair
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int32_t c0,
                                                 int32_t c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}

template <int kN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kMmThreads, 1)
    fp8_gemm_pair_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                         const __grid_constant__ CUtensorMap sfmap, const __grid_constant__ CUtensorMap wsfmap,
                         const __grid_constant__ CUtensorMap ymap, Fp8GemmArgs a) {
  using L = MmPair<kN>;
  constexpr int kStages = L::kStages, kAcc = L::kAcc, kPer = L::kPer;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* ring = align_smem_1024(smem_raw);
  uint8_t* sfs = ring + kStages * L::kStage;
  uint8_t* outs = sfs + kStages * L::kSf;
  typename L::Misc& m = *reinterpret_cast<typename L::Misc*>(outs + L::kOut);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)cluster_rank();

  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&m.full[i], 2);
      mbar_init(&m.empty[i], 1);
    }
    for (int i = 0; i < kAcc; ++i) {
      mbar_init(&m.acc_full[i], 1);
      mbar_init(&m.acc_empty[i], 2 * kMmEpi);
    }
    mbar_init(&m.done, 1);
    fence_barrier_init();
  }
  if (warp == kMmMma) {
    tc::tmem_alloc_pair(&m.tmem, L::kCols);
    tc::tmem_relinquish_pair();
  }
  __syncwarp();
  tc::fence_before_sync();
  cluster_sync_all();  // both CTAs' barriers are there
  tc::fence_after_sync();
  const uint32_t tmem = m.tmem;
  const int mpairs = (a.mtiles + 1) / 2, tiles = mpairs * a.ntiles;
  const int tile0 = blockIdx.x / 2, step = gridDim.x / 2;

  if (warp == kMmWeights) {
    // ---------------- loads ----------------
    int g = 0;
    MmRing<kStages> at;
    bool ok = true;
    if (tc::elect_one()) {
      prefetch_tensormap(&wmap);
      prefetch_tensormap(&wsfmap);
    }
    __syncwarp();
    for (int tile = tile0; ok && tile < tiles; tile += step) {
      const int mt = tile % mpairs * 2 + rank;
      MmScales sc(a.scale + (long long)min(mt, a.mtiles - 1) * a.ktiles, 0, a.ktiles);
      for (int kt = 0; kt < a.ktiles; ++kt, ++g, at.next()) {
        const int s = at.s;
        const uint32_t byte = sc.at(kt);
        if (g >= kStages) ok = mbar_wait_warp(&m.empty[s], at.phase ^ 1, a.status);
        if (!ok) break;
        if (tc::elect_one()) {
          // the other CTA's bytes may be counted before they are announced; the phase ends after both
          if (rank == 0) mbar_arrive_expect_tx(&m.full[s], 2 * (kMmWeight + 512));
          const uint32_t bar = map_to_rank(&m.full[s], 0);
          tma_load_2d_pair(ring + s * L::kStage, &wmap, bar, kt * 128, mt * 128);
          tma_load_2d_pair(sfs + s * L::kSf + L::kSfb, &wsfmap, bar, 0, byte);
        }
        __syncwarp();
      }
    }
    pdl_wait_prior();
    // no copy of either CTA may be in flight when the pair leaves
    if (rank == 0)
      for (int i = max(0, g - kStages); i < g; ++i)
        if (!mbar_drain(&m.full[i % kStages], (i / kStages) & 1, a.status)) break;
  } else if (warp == kMmTokens) {
    int g = 0;
    MmRing<kStages> at;
    bool ok = true;
    if (tc::elect_one()) {
      prefetch_tensormap(&xmap);
      prefetch_tensormap(&sfmap);
    }
    __syncwarp();
    pdl_wait_prior();
    for (int tile = tile0; ok && tile < tiles; tile += step) {
      const int n0 = tile / mpairs * kN;
      for (int kt = 0; kt < a.ktiles; ++kt, ++g, at.next()) {
        const int s = at.s;
        if (g >= kStages) ok = mbar_wait_warp(&m.empty[s], at.phase ^ 1, a.status);
        if (!ok) break;
        if (tc::elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(&m.full[s], 2 * (L::kTokens + L::kSfb));
          const uint32_t bar = map_to_rank(&m.full[s], 0);
          tma_load_2d_pair(ring + s * L::kStage + kMmWeight, &xmap, bar, kt * 128, n0 + rank * (kN / 2));
          tma_load_2d_pair(sfs + s * L::kSf, &sfmap, bar, 0, tile / mpairs * a.ktiles + kt);
        }
        __syncwarp();
      }
    }
    if (rank == 0)
      for (int i = max(0, g - kStages); i < g; ++i)
        if (!mbar_drain(&m.full[i % kStages], (i / kStages) & 1, a.status)) break;
  } else if (warp == kMmMma) {
    // ---------------- MMA, for both CTAs ----------------
    if (rank == 0) {
      int chunk = 0;
      MmRing<kStages> at;
      bool ok = true;
      for (int tile = tile0; ok && tile < tiles; tile += step)
        for (int c0 = 0; ok && c0 < a.ktiles; c0 += a.fold, ++chunk) {
          const int b = chunk % kAcc;
          if (chunk >= kAcc)
            ok = mbar_wait_warp_cluster(&m.acc_empty[b], ((chunk / kAcc) - 1) & 1, a.status);
          if (!ok) break;
          tc::fence_after_sync();
          const uint32_t acc = tmem + b * kN;
          const int c1 = min(a.ktiles, c0 + a.fold);
          for (int kt = c0; kt < c1; ++kt, at.next()) {
            const int s = at.s;
            ok = mbar_wait_warp_cluster(&m.full[s], at.phase, a.status);
            if (!ok) break;
            tc::fence_after_sync();
            if (tc::elect_one()) {
              const uint32_t wsf = tmem + kAcc * kN + (kt & 1) * L::kSfCols, xsf = wsf + 4;
              const uint32_t sf = smem_u32(sfs + s * L::kSf);
              tc::cp_sf_block_pair(wsf, tc::desc_sf_block(sf + L::kSfb));
              tc::cp_sf_block_pair(xsf, tc::desc_sf_block(sf));
              if (kN > 128) tc::cp_sf_block_pair(xsf + 4, tc::desc_sf_block(sf + 512));
              const uint64_t dw = tc::desc_sw128(smem_u32(ring + s * L::kStage));
              const uint64_t dx = tc::desc_sw128(smem_u32(ring + s * L::kStage + kMmWeight));
#pragma unroll
              for (int k = 0; k < 4; ++k)
                tc::mma_mxf8_pair(acc, dw + 2 * k, dx + 2 * k, tc::idesc_mxf8(kN, k, k, 256),
                                  wsf | (uint32_t(k) << 30), xsf | (uint32_t(k) << 30), kt != c0 || k != 0);
              tc::commit_pair(&m.empty[s]);
            }
            __syncwarp();
          }
          if (ok && tc::elect_one()) tc::commit_pair(&m.acc_full[b]);
          __syncwarp();
        }
      // every product has finished before TMEM is released
      if (tc::elect_one()) tc::commit_pair(&m.done);
      __syncwarp();
    }
    mbar_wait(&m.done, 0, a.status);
  } else {
    // ---------------- epilogue ----------------
    pdl_wait_prior();
    const int quad = warp & 3, half = warp >> 2;
    const uint32_t at = tmem + ((uint32_t)(quad * 32) << 16) + half * kPer;
    int chunk = 0, turn = 0;
    bool ok = true;
    for (int tile = tile0; ok && tile < tiles; tile += step) {
      float acc[kPer];
      auto sum = [&](bool first) {
        const int b = chunk % kAcc;
        if (!__all_sync(0xffffffffu, mbar_wait(&m.acc_full[b], (chunk / kAcc) & 1, a.status))) return false;
        tc::fence_after_sync();
        mm_sum<kPer>(at + b * kN, acc, first);
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_to_rank(&m.acc_empty[b], 0));
        ++chunk;
        return true;
      };
      auto agree = [&](bool fine) { return mm_all_of_half(1 + half, fine); };
      auto store = [&] {
        const int row = (tile % mpairs * 2 + rank) * 128 + quad * 32 + lane;
        const int n0 = tile / mpairs * kN + half * kPer;
        // a last tile whose rows end between two 16 bytes of y would zero what lies behind them
        const bool ends = (a.rows & (a.dtype == WH_DTYPE_F32 ? 3 : 7)) == 0 || (row | 127) < a.rows;
        if (!a.boxes || !ends) {
          mm_store<kPer>(a, row, n0, acc);
        } else if (a.dtype == WH_DTYPE_F32) {
          mm_store_boxes<float, kPer>(a, &ymap, outs + half * (L::kOut / 2), turn, row, n0, acc);
        } else if (a.dtype == WH_DTYPE_BF16) {
          mm_store_boxes<__nv_bfloat16, kPer>(a, &ymap, outs + half * (L::kOut / 2), turn, row, n0, acc);
        } else {
          mm_store_boxes<__half, kPer>(a, &ymap, outs + half * (L::kOut / 2), turn, row, n0, acc);
        }
      };
      ok = mm_tile(a.ktiles, a.fold, sum, agree, store);
    }
    bulk_stores_done();
  }
  __syncwarp();
  pdl_launch_dependents();
  tc::fence_before_sync();
  cluster_sync_all();  // the pair leaves together
  tc::fence_after_sync();
  if (warp == kMmMma) tc::tmem_dealloc_pair(tmem, L::kCols);
}

template <int kN, class X>
static cudaError_t launch_fp8_gemm(const CUtensorMap& wmap, const CUtensorMap& xmap, const Fp8GemmArgs& a,
                                   int ctas, int share, cudaStream_t s, bool pdl) {
  const size_t smem = Mm<kN>::kBytes;
  const cudaError_t e = ensure_smem(fp8_gemm_kernel<kN, X>, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kMmThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2]{};
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)share, 1, 1};
  int n = 1;
  if (pdl) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, fp8_gemm_kernel<kN, X>, wmap, xmap, a);
}

template <int kN>
static cudaError_t launch_fp8_gemm_pair(const CUtensorMap& wmap, const CUtensorMap& xmap, const CUtensorMap& sfmap,
                                        const CUtensorMap& wsfmap, const CUtensorMap& ymap, const Fp8GemmArgs& a,
                                        int ctas, cudaStream_t s, bool pdl) {
  const size_t smem = MmPair<kN>::kBytes;
  const cudaError_t e = ensure_smem(fp8_gemm_pair_kernel<kN>, smem);
  if (e != cudaSuccess) return e;
  return launch_pdl(fp8_gemm_pair_kernel<kN>, dim3(ctas), kMmThreads, smem, s, pdl, wmap, xmap, sfmap, wsfmap, ymap, a);
}

}  // namespace wh

// ---------------------------------------------------------------------------
// C entry points
// ---------------------------------------------------------------------------
namespace {

// u32 matrix of scale tiles [rows][wide]: box [1][words]
wh_status make_sf_map(CUtensorMap* map, const void* base, uint64_t rows, uint32_t wide, uint32_t words) {
  auto fn = encode_fn();
  if (!fn) return fail(WH_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {wide, rows};
  cuuint64_t strides[1] = {wide * 4ull};
  cuuint32_t box[2] = {words, 1};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(WH_ERR_CUDA, "cuTensorMapEncodeTiled (scales) failed");
  return WH_OK;
}

// y [tokens][rows]: box [kMmBox][128]
wh_status make_y_map(CUtensorMap* map, void* y, int size, uint64_t rows, uint64_t tokens, uint64_t ldy) {
  auto fn = encode_fn();
  if (!fn) return fail(WH_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {rows, tokens};
  cuuint64_t strides[1] = {ldy * size};
  cuuint32_t box[2] = {128, kMmBox};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, y, dims,
                        strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                        CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(WH_ERR_CUDA, "cuTensorMapEncodeTiled (y) failed");
  return WH_OK;
}

// How a call is cut: tokens of a tile; pairs of CTAs that walk tiles, or clusters of
// `share` CTAs with a tile each.  Measured (tokens x rows x cols, f32 up to 16 tokens, bf16 from
// there on; device us, a CUDA graph of calls over three inputs):
//  - one token: 4096 x 4096 in 1 / 2 / 4 / 8 shares 12.3 / 8.1 / 6.2 / 6.5, 4096 x 8192 22.2 / 13.4
//    / 9.2 / 8.7, 32768 x 1024 (256 tiles) in 1 / 2 shares 8.6 / 12.5: as many CTAs as two an SM
//    hold.  Behind fp8_quant_kernel, whose CTAs are in their way, as many clusters of 8
//    take longer (16 x 4096 x 4096 8.1, in 4 shares 7.3), so
//  - more tokens get one CTA an SM: 17 x 4096 x 4096 in 4 / 8 shares 7.4 / 8.3, 128 x 4096 x 4096
//    9.7 / 22.2 (clusters of 8 no longer all fit), 128 x 512 x 4096 (4 tiles) 8.7 / 8.5;
//  - shares or pairs: 256 x 4096 x 4096 in 2 shares 12.7, pairs 14.2; 509 in 1 share 19.0, pairs 15.2;
//    64 x 32768 x 1024 in 1 share 18.4, pairs 13.5;
//  - pairs of 128 / 224 tokens a tile: 509 x 4096 x 8192 23.7 / 28.0, 1024 40.3 / 46.9, 2048 75.3 / 71.8: a
//    tile of 224 costs up to four thirds of one of 128.
struct MmHow {
  int n, share;
  bool pair;
  bool quant;  // by the product itself
};
// Tokens that the product quantises itself: a launch less, but each CTA quantises them anew.
// Inside / by fp8_quant_kernel, device us: 4096 x 4096 1 token 6.5 / 6.4, 2 6.6 / 6.3, 4 6.9 / 6.4, 8
// 7.9 / 6.7; 4096 x 8192 1 token 8.7 / 10.4, 2 8.9 / 10.3; 512 x 4096 1 token 5.0 / 5.2, 32768 x 1024 8.6 / 9.0.
// A call from Python, by the host: 12.3 / 16.8, for the launch and its scratch.
constexpr int kMmInside = 2;
MmHow mm_how(const wh_ctx* c, int rows, int cols, int tokens) {
  MmHow h{};
  const int mtiles = (rows + 127) / 128, mpairs = (mtiles + 1) / 2, ktiles = (cols + 127) / 128, sms = c->num_sms;
  h.n = tokens <= 16 ? 16 : tokens <= 32 ? 32 : tokens <= 64 ? 64 : 128;
  h.share = 1;
  h.quant = tokens <= kMmInside;
  const long long tiles = (long long)mtiles * ((tokens + h.n - 1) / h.n);
  auto fits = [&](int share) {
    return share * 2 <= ktiles && tiles * share <= (h.quant ? 2 * sms : share == 8 ? sms / 2 : sms);
  };
  while (h.share < kMmShare && fits(2 * h.share)) h.share *= 2;
  h.pair = tokens > 32 && h.share == 1;
  if (h.pair) {
    const long long wide = (long long)mpairs * ((tokens + 223) / 224), narrow = (long long)mpairs * ((tokens + 127) / 128);
    const int pairs = sms / 2;
    h.n = (wide + pairs - 1) / pairs * 4 <= (narrow + pairs - 1) / pairs * 3 ? 224 : 128;
  }
  return h;
}
// Bytes of the tokens' scales in whole tiles, whatever their size: a tile of 224 tokens
// has 1024 bytes a K tile, smaller ones have 512 and a call has at most one of them that
// is smaller than 128.
size_t mm_sf_bytes(int cols, int tokens) {
  const size_t wide = ((size_t)tokens + 223) / 224 * 1024, narrow = ((size_t)tokens + 127) / 128 * 512;
  return std::max(wide, narrow) * (((size_t)cols + 127) / 128);
}

}  // namespace

extern "C" {

size_t wh_fp8_gemm_scratch_bytes(int cols, int tokens) {
  if (cols < 1 || tokens <= kMmInside) return 0;
  return align256((size_t)tokens * cols) + mm_sf_bytes(cols, tokens);
}

wh_status wh_fp8_gemm(wh_ctx* c, const uint8_t* weight, const uint8_t* scale, int rows, int cols,
                      int scale_rows, int scale_cols, const void* x, int dtype, int tokens,
                      long long ldx, void* y, int y_dtype, long long ldy, int act_quant_block,
                      void* scratch, size_t scratch_bytes, wh_stream_t stream) {
  if (wh_status st = kv_device_check(c)) return st;
  int size, y_size;
  if (!kv_dtype_size(dtype, &size) || !kv_dtype_size(y_dtype, &y_size))
    return fail(WH_ERR_UNSUPPORTED, "FP8 GEMM: dtype");
  if (rows < 1 || cols < 1) return fail(WH_ERR_EMPTY_SHAPE, "FP8 GEMM: rows, cols");
  if (rows > kMmMost || cols > kMmMost || tokens > kMmMost)
    return fail(WH_ERR_UNSUPPORTED, "FP8 GEMM: rows, cols or tokens > 2^30");
  if (scale_rows != (rows + 127) / 128 || scale_cols != (cols + 127) / 128)
    return fail(WH_ERR_INVALID_SHAPE, "FP8 GEMM: a scale for each block of 128 x 128");
  if (cols % 16 != 0) return fail(WH_ERR_UNSUPPORTED, "FP8 GEMM: cols % 16 != 0");
  if (tokens < 0) return fail(WH_ERR_INVALID_SHAPE, "FP8 GEMM: tokens");
  if (act_quant_block != 32 && act_quant_block != 64 && act_quant_block != 128)
    return fail(WH_ERR_UNSUPPORTED, "FP8 GEMM: act_quant_block 32, 64 or 128");
  if (tokens == 0) return WH_OK;
  if (tokens > 1 && (ldx < cols || ldy < rows))
    return fail(WH_ERR_INVALID_SHAPE, "FP8 GEMM: rows of x or y overlap");
  if (!weight || !scale || !x || !y || (!scratch && tokens > kMmInside))
    return fail(WH_ERR_INVALID_POINTER, "FP8 GEMM: null pointer");
  if (!aligned(weight, 16) || !aligned(scratch, 16))
    return fail(WH_ERR_INVALID_POINTER, "FP8 GEMM: weight and scratch must be 16-byte aligned");
  if (!kv_rows_aligned(x, tokens > 1 ? ldx : 0, 0, size))
    return fail(WH_ERR_INVALID_POINTER, "FP8 GEMM: rows of x must start on 16 bytes");
  if (!aligned(y, y_size)) return fail(WH_ERR_INVALID_POINTER, "FP8 GEMM: y is not aligned");
  if (scratch_bytes < wh_fp8_gemm_scratch_bytes(cols, tokens))
    return fail(WH_ERR_SCRATCH_TOO_SMALL, "FP8 GEMM: scratch too small");
  const MmHow h = mm_how(c, rows, cols, tokens);
  uint8_t* xq = static_cast<uint8_t*>(scratch);
  uint8_t* xsf = xq + align256((size_t)tokens * cols);
  CUtensorMap wmap, xmap;
  if (wh_status st = make_u8_map(&wmap, weight, rows, cols, 128)) return st;
  if (h.quant)
    xmap = wmap;  // not used
  else if (wh_status st = make_u8_map(&xmap, xq, tokens, cols, h.pair ? h.n / 2 : h.n))
    return st;
  const cudaStream_t s = (cudaStream_t)stream;
  const int ktiles = (cols + 127) / 128;
  const int chunks = (ktiles * 16 + kQuantThreads - 1) / kQuantThreads;
  const int shift = h.n == 16 ? 4 : h.n == 32 ? 5 : h.n == 64 ? 6 : h.n == 128 ? 7 : 0, lanes = act_quant_block / 8;
  const Fp8QuantArgs qa{x, ldx, tokens, cols, ktiles, h.n, shift, xq, xsf};
  if ((long long)tokens * chunks > 0x7fffffffLL) return fail(WH_ERR_UNSUPPORTED, "FP8 GEMM: tokens * cols too large");
  const dim3 grid(chunks, std::min(tokens, 65535));
  if (h.quant)
    ;
  else if (dtype == WH_DTYPE_F32)
    WH_CUDA(launch_fp8_quant<float>(qa, lanes, grid, s, c->pdl()));
  else if (dtype == WH_DTYPE_BF16)
    WH_CUDA(launch_fp8_quant<__nv_bfloat16>(qa, lanes, grid, s, c->pdl()));
  else
    WH_CUDA(launch_fp8_quant<__half>(qa, lanes, grid, s, c->pdl()));
  const bool boxes = aligned(y, 16) && ldy * y_size % 16 == 0;
  const Fp8GemmArgs a{scale, c->sf_rows, xsf, y, ldy, rows, tokens, ktiles, y_dtype,
                      y_dtype == WH_DTYPE_F32 ? kMmFold : kMmFold16, (rows + 127) / 128,
                      (tokens + h.n - 1) / h.n, boxes, x, ldx, cols, lanes, c->status};
  if ((long long)a.mtiles * a.ntiles > 0x7fffffffLL / 8)
    return fail(WH_ERR_UNSUPPORTED, "FP8 GEMM: rows * tokens too large");
  const bool pdl = c->pdl();
  const int tiles = a.mtiles * a.ntiles, split = tiles * h.share;
  cudaError_t e;
  if (h.pair) {
    CUtensorMap sfmap, wsfmap, ymap;
    const uint32_t words = h.n > 128 ? 256 : 128;
    if (wh_status st = make_sf_map(&sfmap, xsf, (uint64_t)a.ntiles * ktiles, words, words)) return st;
    if (wh_status st = make_sf_map(&wsfmap, c->sf_rows, 256, 128, 128)) return st;
    if (!boxes)
      ymap = xmap;  // not used
    else if (wh_status st = make_y_map(&ymap, y, y_size, rows, tokens, ldy))
      return st;
    const int ctas = std::min((a.mtiles + 1) / 2 * a.ntiles, c->num_sms / 2) * 2;
    e = h.n > 128 ? launch_fp8_gemm_pair<224>(wmap, xmap, sfmap, wsfmap, ymap, a, ctas, s, pdl)
                  : launch_fp8_gemm_pair<128>(wmap, xmap, sfmap, wsfmap, ymap, a, ctas, s, pdl);
  } else {
    e = h.n == 32   ? launch_fp8_gemm<32, void>(wmap, xmap, a, split, h.share, s, pdl)
        : h.n == 64 ? launch_fp8_gemm<64, void>(wmap, xmap, a, split, h.share, s, pdl)
        : h.n > 64  ? launch_fp8_gemm<128, void>(wmap, xmap, a, split, h.share, s, pdl)
        : !h.quant  ? launch_fp8_gemm<16, void>(wmap, xmap, a, split, h.share, s, pdl)
        : dtype == WH_DTYPE_F32  ? launch_fp8_gemm<16, float>(wmap, xmap, a, split, h.share, s, pdl)
        : dtype == WH_DTYPE_BF16 ? launch_fp8_gemm<16, __nv_bfloat16>(wmap, xmap, a, split, h.share, s, pdl)
                                 : launch_fp8_gemm<16, __half>(wmap, xmap, a, split, h.share, s, pdl);
  }
  if (e != cudaSuccess) return cuda_fail(e, "FP8 GEMM");
  return WH_OK;
}

}  // extern "C"
