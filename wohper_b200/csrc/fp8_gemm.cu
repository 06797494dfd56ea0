// fp8_gemm.cu -- FP8 E4M3 x UE8M0(128 x 128) matrix products of many tokens on
// the 5th-generation tensor cores.
//
//   y[t][r] = sum_c W[r][c] 2^(S[r/128][c/128] - 127) aq(x[t])[c]
//
// aq is the framework's FP8 act quant (common.cuh) per block of 32, 64 or 128
// values: both operands are E4M3 codes with a power-of-two scale, so a
// kind::mxf8f6f4 product is exact and only the sums round.  Two launches:
// fp8_quant_kernel writes the tokens' codes and their scale bytes in the order
// in which the product's scale copies read them; fp8_gemm_kernel multiplies.
//
// The weight is the M operand (128 rows of it a tile), so that one token costs
// N = 16 columns and not 128 rows, and a warp's 32 accumulator lanes are 32
// neighbouring outputs of a token.
#include <cuda_bf16.h>

#include "tc.cuh"

namespace wh {

struct Fp8GemmArgs {
  const uint8_t* scale;  // [ceil(rows/128)][ktiles]
  const uint8_t* xsf;    // [ceil(tokens/128)][ktiles][512], fp8_quant_kernel's
  void* y;
  long long ldy;
  int rows, tokens, ktiles;
  int dtype;   // of y
  int fold;    // K tiles that a sum runs through the tensor core before it is added in f32
  int mtiles, ntiles;
  uint32_t* status;
};

// ---------------------------------------------------------------------------
// act quant: a thread takes 8 values, a block of 32/64/128 is 4/8/16 lanes.
// Reads tokens * cols values, writes a byte each and a scale byte for 32.
// ---------------------------------------------------------------------------
struct Fp8QuantArgs {
  const void* x;
  long long ldx;
  int cols, ktiles;
  int lanes;   // 4, 8 or 16 a block
  int chunks;  // CTAs of a token
  uint8_t* xq;   // [tokens][cols]
  uint8_t* xsf;
};
constexpr int kQuantThreads = 256;

template <class T>
__global__ void __launch_bounds__(kQuantThreads) fp8_quant_kernel(Fp8QuantArgs a) {
  pdl_wait_prior();
  pdl_launch_dependents();  // what came before is complete: the product may start on its weights
  const int t = blockIdx.x / a.chunks;
  const int part = (blockIdx.x - t * a.chunks) * kQuantThreads + threadIdx.x, col = part * 8;
  if (part >= a.ktiles * 16) return;  // whole blocks leave
  const bool on = col < a.cols;  // cols is a multiple of 16
  float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (on) kv_load8(static_cast<const T*>(a.x) + t * a.ldx + col, v);
  float m = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[j]));  // passes over NaN
  const unsigned lane = threadIdx.x & 31;
  const unsigned group = ((1u << a.lanes) - 1) << (lane & ~(a.lanes - 1));
  for (int o = 1; o < a.lanes; o <<= 1) m = fmaxf(m, __shfl_xor_sync(group, m, o));
  const AqScale s = aq_block_scale(m, c_aq.thr);
  uint2 w;
  w.x = e4m3x2_ref(__fmul_rn(v[0], s.inv), __fmul_rn(v[1], s.inv)) |
        e4m3x2_ref(__fmul_rn(v[2], s.inv), __fmul_rn(v[3], s.inv)) << 16;
  w.y = e4m3x2_ref(__fmul_rn(v[4], s.inv), __fmul_rn(v[5], s.inv)) |
        e4m3x2_ref(__fmul_rn(v[6], s.inv), __fmul_rn(v[7], s.inv)) << 16;
  if (on) *reinterpret_cast<uint2*>(a.xq + (long long)t * a.cols + col) = w;
  // an infinite block's scale byte is 255, the product's NaN; groups past the row's end get 2^0
  if ((part & 3) == 0) {
    uint8_t* at = a.xsf + ((long long)(t >> 7) * a.ktiles + (part >> 4)) * 512 + (t & 31) * 16 + ((t & 127) >> 5) * 4;
    at[(part >> 2) & 3] = on ? uint8_t(__float_as_uint(s.scale) >> 23) : 127;
  }
}

// ---------------------------------------------------------------------------
// product
// ---------------------------------------------------------------------------
constexpr int kMmWeight = 128 * 128;  // a weight tile: 128 rows x 128 K
constexpr int kMmEpi = 8;             // epilogue warps: TMEM quadrant w % 4, column half w / 4
constexpr int kMmLoad = kMmEpi, kMmMma = kMmEpi + 1;
constexpr int kMmThreads = (kMmEpi + 2) * 32;

template <int kN>
struct Mm {
  static constexpr int kTokens = kN * 128;             // bytes of a token tile
  static constexpr int kStage = kMmWeight + kTokens;
  static constexpr int kSfb = kN > 128 ? 1024 : 512;
  static constexpr int kSf = kSfb + 512;
  static constexpr int kStages = kN >= 256 ? 4 : kN >= 128 ? 6 : 4;
  static constexpr int kAcc = kN > 128 ? 1 : 2;        // accumulator sets
  static constexpr int kSfCols = kSfb / 128 + 4;       // TMEM columns of a set of scales
  static constexpr int kNeed = kAcc * kN + 2 * kSfCols;
  static constexpr int kCols = kNeed <= 64 ? 64 : kNeed <= 128 ? 128 : kNeed <= 256 ? 256 : 512;
  static constexpr int kPer = kN / 2;                  // columns of an epilogue warp
  struct Misc {
    uint64_t full[kStages], empty[kStages], acc_full[kAcc], acc_empty[kAcc], done;
    uint32_t tmem;
  };
  static constexpr int kBytes = 1024 + kStages * (kStage + kSf) + (int)sizeof(Misc);
  static_assert(kBytes <= 232448 && kNeed <= 512, "shared memory or TMEM");
  static_assert(kN > 128 || kN * 128 * 4 <= kStages * kStage, "a partial sum fits the ring");
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
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
  float v;
  asm volatile("{ .reg .b32 a; mapa.shared::cluster.u32 a, %1, %2; ld.shared::cluster.f32 %0, [a]; }"
               : "=f"(v)
               : "r"(addr), "r"(rank)
               : "memory");
  return v;
}
__device__ __forceinline__ void mm_put(void* y, long long at, int dtype, float v) {
  if (dtype == WH_DTYPE_F32)
    static_cast<float*>(y)[at] = v;
  else if (dtype == WH_DTYPE_BF16)
    static_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(y)[at] = __float2half_rn(v);
}

// kSplit: the CTAs of a cluster share one tile's K and add their sums through
// distributed shared memory, in the order of their ranks; otherwise each CTA
// walks tiles, weight tiles of the same tokens next to one another.
template <int kN, bool kSplit>
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
  const int rank = kSplit ? (int)cluster_rank() : 0, share = kSplit ? (int)cluster_size() : 1;

  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&m.full[i], 1);
      mbar_init(&m.empty[i], 1);
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
  const int tiles = a.mtiles * a.ntiles;
  const int tile0 = kSplit ? blockIdx.x / share : blockIdx.x, step = kSplit ? tiles : gridDim.x;
  // this CTA's K tiles
  const int k0 = kSplit ? int((long long)a.ktiles * rank / share) : 0;
  const int k1 = kSplit ? int((long long)a.ktiles * (rank + 1) / share) : a.ktiles;

  if (warp == kMmLoad) {
    // ---------------- loads ----------------
    int g = 0;
    bool ok = true, waited = false;
    if (lane == 0) {
      prefetch_tensormap(&wmap);
      prefetch_tensormap(&xmap);
    }
    int ahead = 0;  // stages whose weights are on their way before the tokens' codes are there
    auto weights = [&](int s, int tile, int kt) {
      uint8_t* st = ring + s * L::kStage;
      const uint32_t b = a.scale[(long long)(tile % a.mtiles) * a.ktiles + kt] * 0x01010101u;
      *reinterpret_cast<uint4*>(sfs + s * L::kSf + L::kSfb + lane * 16) = make_uint4(b, b, b, b);
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive_expect_tx(&m.full[s], kMmWeight + L::kTokens + L::kSfb);
        tma_load_2d(st, &wmap, &m.full[s], kt * 128, tile % a.mtiles * 128);
      }
    };
    auto tokens = [&](int s, int tile, int kt) {
      if (lane == 0) {
        uint8_t* st = ring + s * L::kStage + kMmWeight;
        uint8_t* sf = sfs + s * L::kSf;
        const int n0 = tile / a.mtiles * kN;
        tma_load_2d(st, &xmap, &m.full[s], kt * 128, n0);
        const uint8_t* src = a.xsf + ((long long)(n0 >> 7) * a.ktiles + kt) * 512;
        bulk_load(sf, src, 512, &m.full[s]);
        if (kN > 128) bulk_load(sf + 512, src + (long long)a.ktiles * 512, 512, &m.full[s]);
      }
    };
    if (tile0 < tiles) {
      ahead = min(kStages, k1 - k0);
      for (int i = 0; i < ahead; ++i) weights(i, tile0, k0 + i);
    }
    pdl_wait_prior();
    for (int tile = tile0; ok && tile < tiles; tile += step)
      for (int kt = k0; kt < k1; ++kt, ++g) {
        const int s = g % kStages;
        if (g >= ahead) {
          if (g >= kStages) ok = __all_sync(0xffffffffu, mbar_wait(&m.empty[s], ((g / kStages) - 1) & 1, a.status));
          if (!ok) break;
          weights(s, tile, kt);
        }
        tokens(s, tile, kt);
      }
    // no copy may be in flight when the CTA exits
    for (int i = max(0, g - kStages); i < g; ++i)
      if (!mbar_drain(&m.full[i % kStages], (i / kStages) & 1, a.status)) break;
  } else if (warp == kMmMma) {
    // ---------------- MMA ----------------
    int g = 0, chunk = 0;
    bool ok = true;
    for (int tile = tile0; ok && tile < tiles; tile += step)
      for (int c0 = k0; ok && c0 < k1; c0 += a.fold, ++chunk) {
        const int b = chunk % kAcc;
        if (chunk >= kAcc) ok = __all_sync(0xffffffffu, mbar_wait(&m.acc_empty[b], ((chunk / kAcc) - 1) & 1, a.status));
        if (!ok) break;
        tc::fence_after_sync();
        const uint32_t acc = tmem + b * kN;
        const int c1 = min(k1, c0 + a.fold);
        for (int kt = c0; kt < c1; ++kt, ++g) {
          const int s = g % kStages;
          ok = __all_sync(0xffffffffu, mbar_wait(&m.full[s], (g / kStages) & 1, a.status));
          if (!ok) break;
          tc::fence_after_sync();
          if (tc::elect_one()) {
            const uint32_t wsf = tmem + kAcc * kN + (g & 1) * L::kSfCols, xsf = wsf + 4;
            const uint32_t sf = smem_u32(sfs + s * L::kSf);
            tc::cp_sf_block(wsf, tc::desc_sf_block(sf + L::kSfb));
            tc::cp_sf_block(xsf, tc::desc_sf_block(sf));
            if (kN > 128) tc::cp_sf_block(xsf + 4, tc::desc_sf_block(sf + 512));
            const uint64_t dw = tc::desc_sw128(smem_u32(ring + s * L::kStage));
            const uint64_t dx = tc::desc_sw128(smem_u32(ring + s * L::kStage + kMmWeight));
#pragma unroll
            for (int k = 0; k < 4; ++k)
              tc::mma_mxf8(acc, dw + 2 * k, dx + 2 * k, tc::idesc_mxf8(kN, k, k), wsf | (uint32_t(k) << 30),
                           xsf | (uint32_t(k) << 30), kt != c0 || k != 0);
            tc::commit(&m.empty[s]);
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
  } else {
    // ---------------- epilogue ----------------
    pdl_wait_prior();
    const int quad = warp & 3, half = warp >> 2;
    const uint32_t at = tmem + ((uint32_t)(quad * 32) << 16) + half * kPer;
    int chunk = 0;
    bool ok = true;
    for (int tile = tile0; ok && tile < tiles; tile += step) {
      float acc[kPer];
      for (int c0 = k0; c0 < k1; c0 += a.fold, ++chunk) {
        const int b = chunk % kAcc;
        ok = __all_sync(0xffffffffu, mbar_wait(&m.acc_full[b], (chunk / kAcc) & 1, a.status));
        if (!ok) break;
        tc::fence_after_sync();
        constexpr int kOne = kPer < 16 ? 8 : 16;
#pragma unroll
        for (int c = 0; c < kPer; c += kOne) {
          uint32_t v[kOne];
          if constexpr (kOne == 8)
            tc::ld_32x32b_x8(at + b * kN + c, v);
          else
            tc::ld_32x32b_x16(at + b * kN + c, v);
          tc::wait_ld_of(v);
#pragma unroll
          for (int e = 0; e < kOne; ++e)
            acc[c + e] = c0 == k0 ? __uint_as_float(v[e]) : acc[c + e] + __uint_as_float(v[e]);
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&m.acc_empty[b]);
      }
      if (!ok) break;
      const int row = tile % a.mtiles * 128 + quad * 32 + lane;
      const int n0 = tile / a.mtiles * kN + half * kPer;
      if (kSplit) {
        // the ring is idle: every product that reads it has finished
        float* part = reinterpret_cast<float*>(ring) + half * kPer * 128 + quad * 32 + lane;
#pragma unroll
        for (int c = 0; c < kPer; ++c) part[c * 128] = acc[c];
      } else {
#pragma unroll
        for (int c = 0; c < kPer; ++c)
          if (row < a.rows && n0 + c < a.tokens) mm_put(a.y, (n0 + c) * a.ldy + row, a.dtype, acc[c]);
      }
    }
  }
  if (kSplit) {
    __syncwarp();
    cluster_sync_all();
    // this CTA's columns of the tile, added in the order of the ranks
    const int n0 = tile0 / a.mtiles * kN;
    for (int i = rank * kMmThreads + tid; i < kN * 128; i += share * kMmThreads) {
      const int row = tile0 % a.mtiles * 128 + (i & 127), n = n0 + (i >> 7);
      if (row >= a.rows || n >= a.tokens) continue;
      const uint32_t at = smem_u32(ring) + i * 4;
      float v = 0.0f;
      for (int r = 0; r < share; ++r) v += ld_cluster(at, r);
      mm_put(a.y, n * a.ldy + row, a.dtype, v);
    }
    cluster_sync_all();  // the others have read this CTA's sums
  }
  pdl_launch_dependents();
  tc::fence_before_sync();
  __syncthreads();
  if (warp == kMmMma) tc::tmem_dealloc(tmem, L::kCols);
}

template <int kN, bool kSplit>
static cudaError_t launch_fp8_gemm(const CUtensorMap& wmap, const CUtensorMap& xmap, const Fp8GemmArgs& a,
                                   int ctas, int share, cudaStream_t s, bool pdl) {
  const size_t smem = Mm<kN>::kBytes;
  const cudaError_t e = ensure_smem(fp8_gemm_kernel<kN, kSplit>, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kMmThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2]{};
  int n = 0;
  if (kSplit) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim = {(unsigned)share, 1, 1};
    ++n;
  }
  if (pdl) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, fp8_gemm_kernel<kN, kSplit>, wmap, xmap, a);
}

}  // namespace wh

// ---------------------------------------------------------------------------
// C entry points
// ---------------------------------------------------------------------------
namespace {

// How a call is cut: tokens of a tile, CTAs that share a tile's K.
struct MmHow {
  int n, share;
};
MmHow mm_how(const wh_ctx* c, int rows, int cols, int tokens) {
  MmHow h{256, 1};
  if (tokens <= 128) {
    h.n = tokens <= 16 ? 16 : tokens <= 32 ? 32 : tokens <= 64 ? 64 : 128;
    const int mtiles = (rows + 127) / 128, ktiles = (cols + 127) / 128;
    while (h.share < 8 && mtiles * h.share * 2 <= c->num_sms && h.share * 4 <= ktiles) h.share *= 2;
  } else {
    const long long tiles = (long long)((rows + 127) / 128) * ((tokens + 255) / 256);
    if (tiles < c->num_sms) h.n = 128;
  }
  return h;
}
size_t mm_sf_bytes(int cols, int tokens) {
  // whole tiles of 256 tokens
  return (size_t)((tokens + 255) / 256 * 2) * ((cols + 127) / 128) * 512;
}

}  // namespace

extern "C" {

size_t wh_fp8_gemm_scratch_bytes(int cols, int tokens) {
  if (cols < 1 || tokens < 1) return 0;
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
  if (scale_rows != (rows + 127) / 128 || scale_cols != (cols + 127) / 128)
    return fail(WH_ERR_INVALID_SHAPE, "FP8 GEMM: a scale for each block of 128 x 128");
  if (cols % 16 != 0) return fail(WH_ERR_UNSUPPORTED, "FP8 GEMM: cols % 16 != 0");
  if (tokens < 0) return fail(WH_ERR_INVALID_SHAPE, "FP8 GEMM: tokens");
  if (act_quant_block != 32 && act_quant_block != 64 && act_quant_block != 128)
    return fail(WH_ERR_UNSUPPORTED, "FP8 GEMM: act_quant_block 32, 64 or 128");
  if (tokens == 0) return WH_OK;
  if (tokens > 1 && (ldx < cols || ldy < rows))
    return fail(WH_ERR_INVALID_SHAPE, "FP8 GEMM: rows of x or y overlap");
  if (!weight || !scale || !x || !y || !scratch)
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
  if (wh_status st = make_u8_map(&xmap, xq, tokens, cols, h.n)) return st;
  const cudaStream_t s = (cudaStream_t)stream;
  const int ktiles = (cols + 127) / 128;
  const int chunks = (ktiles * 16 + kQuantThreads - 1) / kQuantThreads;
  const Fp8QuantArgs qa{x, ldx, cols, ktiles, act_quant_block / 8, chunks, xq, xsf};
  const long long blocks = (long long)tokens * chunks;
  if (blocks > 0x7fffffffLL) return fail(WH_ERR_UNSUPPORTED, "FP8 GEMM: tokens * cols too large");
  const dim3 grid((unsigned)blocks);
  if (dtype == WH_DTYPE_F32)
    WH_CUDA(launch_pdl(fp8_quant_kernel<float>, grid, kQuantThreads, 0, s, c->pdl(), qa));
  else if (dtype == WH_DTYPE_BF16)
    WH_CUDA(launch_pdl(fp8_quant_kernel<__nv_bfloat16>, grid, kQuantThreads, 0, s, c->pdl(), qa));
  else
    WH_CUDA(launch_pdl(fp8_quant_kernel<__half>, grid, kQuantThreads, 0, s, c->pdl(), qa));
  const Fp8GemmArgs a{scale, xsf, y, ldy, rows, tokens, ktiles, y_dtype,
                      y_dtype == WH_DTYPE_F32 ? 8 : 1 << 20, (rows + 127) / 128,
                      (tokens + h.n - 1) / h.n, c->status};
  if ((long long)a.mtiles * a.ntiles > 0x7fffffffLL)
    return fail(WH_ERR_UNSUPPORTED, "FP8 GEMM: rows * tokens too large");
  const int tiles = a.mtiles * a.ntiles;
  const bool pdl = c->pdl();
  const int split = tiles * h.share, walk = std::min(tiles, c->num_sms);
  const cudaError_t e = tokens <= 16    ? launch_fp8_gemm<16, true>(wmap, xmap, a, split, h.share, s, pdl)
                        : tokens <= 32  ? launch_fp8_gemm<32, true>(wmap, xmap, a, split, h.share, s, pdl)
                        : tokens <= 64  ? launch_fp8_gemm<64, true>(wmap, xmap, a, split, h.share, s, pdl)
                        : tokens <= 128 ? launch_fp8_gemm<128, true>(wmap, xmap, a, split, h.share, s, pdl)
                        : h.n == 128    ? launch_fp8_gemm<128, false>(wmap, xmap, a, walk, 1, s, pdl)
                                        : launch_fp8_gemm<256, false>(wmap, xmap, a, walk, 1, s, pdl);
  if (e != cudaSuccess) return cuda_fail(e, "FP8 GEMM");
  return WH_OK;
}

}  // extern "C"
