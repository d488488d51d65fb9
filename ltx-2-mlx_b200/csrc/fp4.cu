// fp4.cu -- 4-bit floating point (mxfp4, nvfp4): quantizing and reading back
// matrices, and the product of two quantized operands on the block-scaled
// tensor cores (tcgen05.mma kind::mxf4 / kind::mxf4nvf4).
//
// The reference's cache quantizers name both formats beside mxfp8
// (loader/transformer_cache.py:797-811: mxfp4 -> group 32, nvfp4 -> group 16);
// the numerics are in fp4.cuh.  A matrix is held in one of two forms that
// differ only in where its scale bytes lie: row-major [rows, K / group] in the
// weight cache, and the MMA's atom layout (fp4.cuh) in an ltxq_fp4_act and in
// the packed weight scales.
#include "common.cuh"
#include "fp4.cuh"
#include "gemm_epilogue.cuh"

namespace ltxq {

ltxq_status check_qweight(const ltxq_qweight& w, bool need_data, int64_t* R, int64_t* L);
bool fp4_rows_supported(int64_t M, const ltxq_qweight& w);
ltxq_status launch_fp4_rows(const void* x, bool quantize, const ltxq_fp4_act* packed, const ltxq_qweight& w,
                            const gemm::Params& p, cudaStream_t stream);

namespace fp4 {

// ---------------------------------------------------------------- quantize / read back

// Both ways: one thread per 16 elements of a row, memory-bound (2 bytes of
// values and 0.53 to 0.56 of codes and scales per element).  A CTA's 256 threads
// take a row side by side (width a power of two, 16 to 256: several short rows
// per CTA, a long one in steps), so that no index is divided out: with a flat
// 64-bit index 16384 x 4096 took 35 us to quantize.

// kAtomsOut: rows run over whole K stages, whose groups past the row's end get
// scale 0 (the GEMM reads their codes as zeros); otherwise scales go row-major.
template <int F, bool kAtomsOut, bool kDiv>
__global__ void __launch_bounds__(256) quantize_kernel(const uint16_t* __restrict__ x, int64_t rows, int K,
                                                       int64_t row_stride, float g, int log_width,
                                                       uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  chain_trigger();  // the product of what it writes
  constexpr int kGroup = Traits<F>::kGroup;
  const int chunks = kAtomsOut ? (K + kStageK - 1) / kStageK * (kStageK / 16) : K / 16;
  const int64_t row_tiles = (rows + 127) / 128;
  const float inv_g = F == kNv && !kDiv ? __frcp_rn(g) : 1.f;
  const int width = 1 << log_width;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 >> log_width) + (threadIdx.x >> log_width);
  const uint16_t* xr = x + row * row_stride;
  uint8_t* cr = codes + row * (K / 2);
  for (int c0 = 0; c0 < chunks; c0 += width) {  // every lane takes part in the shuffles of every step
    const int c = c0 + (threadIdx.x & (width - 1));
    const bool live = row < rows && c < chunks;
    const bool data = live && c * 16 < K;
    uint32_t u[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (data) {
      const uint4* src = reinterpret_cast<const uint4*>(xr + c * 16);
      const uint4 a = __ldg(src), b = __ldg(src + 1);
      u[0] = a.x; u[1] = a.y; u[2] = a.z; u[3] = a.w;
      u[4] = b.x; u[5] = b.y; u[6] = b.z; u[7] = b.w;
    }
    uint32_t am = amax16(u);
    GroupScale gs;
    if (F == kMx) {  // a group is two neighbouring lanes (an even number of chunks per row)
      am = max(am, __shfl_xor_sync(0xffffffffu, am, 1));
      gs = mx_group(am);
    } else {
      const float a = __uint_as_float(am << 16);
      gs = nv_group(kDiv ? __fdiv_rn(a, g) : __fmul_rn(a, inv_g), am < 0x7F80u, inv_g);
    }
    if (data) *reinterpret_cast<uint2*>(cr + c * 8) = encode16<F, kDiv>(u, gs, g);
    const uint32_t byte = data ? gs.byte : 0u;
    const int group = c * 16 / kGroup;
    if (kAtomsOut) {
      // four neighbouring groups are one word of an atom; a row starts at a multiple of 16 threads
      const int lane = threadIdx.x & 31;
      uint32_t w;
      if (F == kNv) {
        w = byte << (8 * (lane & 3));
        w |= __shfl_xor_sync(0xffffffffu, w, 1);
        w |= __shfl_xor_sync(0xffffffffu, w, 2);
      } else {
        w = byte << (8 * ((lane >> 1) & 3));
        w |= __shfl_xor_sync(0xffffffffu, w, 2);
        w |= __shfl_xor_sync(0xffffffffu, w, 4);
      }
      if (live && (lane & (F == kNv ? 3 : 7)) == 0)
        *reinterpret_cast<uint32_t*>(scales + atom_offset<F>(row, group, row_tiles)) = w;
    } else if (data && (F == kNv || (threadIdx.x & 1) == 0)) {
      scales[row * (K / kGroup) + group] = static_cast<uint8_t>(byte);
    }
  }
}

template <int F, bool kAtomsIn>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* __restrict__ codes,
                                                         const uint8_t* __restrict__ scales, int64_t rows, int K,
                                                         float g, int log_width, uint16_t* __restrict__ out) {
  chain_trigger();  // the product of what it writes
  constexpr int kGroup = Traits<F>::kGroup;
  const int64_t row_tiles = (rows + 127) / 128;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 >> log_width) + (threadIdx.x >> log_width);
  if (row >= rows) return;
  const uint8_t* cr = codes + row * (K / 2);
  const uint8_t* sr = scales + row * (K / kGroup);
  uint16_t* orow = out + row * K;
  for (int c = threadIdx.x & ((1 << log_width) - 1); c < K / 16; c += 1 << log_width) {
    const int group = c * 16 / kGroup;
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(cr + c * 8));
    const uint32_t s2 = scale_bf16x2<F>(kAtomsIn ? __ldg(scales + atom_offset<F>(row, group, row_tiles)) : __ldg(sr + group));
    uint32_t a[4], b[4];
    decode_word(w.x, s2, a);
    decode_word(w.y, s2, b);
    if (F == kNv && g != 1.f) {  // one more product in fp32, rounded to bf16
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        a[k] = pack_bf16x2(__fmul_rn(lo_bf16(a[k]), g), __fmul_rn(hi_bf16(a[k]), g));
        b[k] = pack_bf16x2(__fmul_rn(lo_bf16(b[k]), g), __fmul_rn(hi_bf16(b[k]), g));
      }
    }
    uint4* dst = reinterpret_cast<uint4*>(orow + c * 16);
    dst[0] = make_uint4(a[0], a[1], a[2], a[3]);
    dst[1] = make_uint4(b[0], b[1], b[2], b[3]);
  }
}

// Row-major scales [N, G] -> the atom layout, one thread per byte; groups past
// the row's end and rows of the last tile past N get scale 0.
template <int F>
__global__ void __launch_bounds__(256) pack_scales_kernel(const uint8_t* __restrict__ s, int64_t N, int64_t G,
                                                          int64_t Gp, uint8_t* __restrict__ out) {
  const int64_t row_tiles = (N + 127) / 128;
  const int64_t total = row_tiles * 128 * Gp;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t row = i / Gp, gi = i - row * Gp;
    out[atom_offset<F>(row, gi, row_tiles)] = row < N && gi < G ? s[row * G + gi] : uint8_t(0);
  }
}

// a row's threads, as a power of two from 16 to 256, and the CTAs of that
struct RowGrid {
  int log_width;
  unsigned grid;
};
static RowGrid row_grid(int64_t rows, int64_t chunks) {
  int lw = 4;
  while (lw < 8 && (1 << lw) < chunks) ++lw;
  const int64_t per = 256 >> lw;
  return RowGrid{lw, static_cast<unsigned>((rows + per - 1) / per)};
}

static unsigned grid_for(int64_t work) {
  const int64_t want = (work + 255) / 256;
  const int64_t cap = static_cast<int64_t>(num_sms()) * 32;
  return static_cast<unsigned>(want < 1 ? 1 : (want < cap ? want : cap));
}

static bool power_of_two(float g) {
  uint32_t b;
  memcpy(&b, &g, sizeof(b));
  return (b & 0x7FFFFFu) == 0;
}

}  // namespace fp4

// global_scale as the formats take it: 1 for mxfp4; finite and within
// [2^-64, 2^64] for nvfp4, so that its reciprocal and its products with a
// scale stay in range.  0 stands for 1 (a zeroed descriptor).
ltxq_status fp4_global_scale(int32_t mode, float g, float* out, const char* what) {
  *out = 1.f;
  if (g == 0.f || g == 1.f) return LTXQ_OK;
  if (mode != LTXQ_NVFP4) return fail(LTXQ_ERR_INVALID, std::string(what) + ": mxfp4 has no global_scale");
  if (!(g >= 5.421010862427522e-20f && g <= 1.8446744073709552e19f))
    return fail(LTXQ_ERR_INVALID, std::string(what) + ": global_scale must be within [2^-64, 2^64]");
  *out = g;
  return LTXQ_OK;
}

// The weight cache's row-major form (the caller checked the descriptor, sizes below 2^30).
ltxq_status launch_fp4_quantize_rows(const uint16_t* x, int64_t R, int64_t L, int32_t mode, float g, uint8_t* codes,
                                     uint8_t* scales, cudaStream_t s) {
  const fp4::RowGrid r = fp4::row_grid(R, L / 16);
  const int K = static_cast<int>(L);
  if (mode == LTXQ_MXFP4)
    fp4::quantize_kernel<fp4::kMx, false, false><<<r.grid, 256, 0, s>>>(x, R, K, L, g, r.log_width, codes, scales);
  else if (fp4::power_of_two(g))
    fp4::quantize_kernel<fp4::kNv, false, false><<<r.grid, 256, 0, s>>>(x, R, K, L, g, r.log_width, codes, scales);
  else
    fp4::quantize_kernel<fp4::kNv, false, true><<<r.grid, 256, 0, s>>>(x, R, K, L, g, r.log_width, codes, scales);
  return launch_check("fp4 quantize launch");
}

ltxq_status launch_fp4_dequantize_rows(const uint8_t* codes, const uint8_t* scales, int64_t R, int64_t L, int32_t mode,
                                       float g, uint16_t* out, cudaStream_t s) {
  const fp4::RowGrid r = fp4::row_grid(R, L / 16);
  const int K = static_cast<int>(L);
  if (mode == LTXQ_MXFP4)
    fp4::dequantize_kernel<fp4::kMx, false><<<r.grid, 256, 0, s>>>(codes, scales, R, K, g, r.log_width, out);
  else
    fp4::dequantize_kernel<fp4::kNv, false><<<r.grid, 256, 0, s>>>(codes, scales, R, K, g, r.log_width, out);
  return launch_check("fp4 dequantize launch");
}

// ---------------------------------------------------------------- GEMM of two quantized operands

namespace fp4 {

// Persistent kernel, clusters of two CTAs (tcgen05 cta_group::2).  A tile is
// 256 kBlocks tokens x BN features: CTA r holds kBlocks blocks of 128 token
// rows (operand A, TMEM lanes = tokens) and BN / 2 weight rows (operand B).  Codes
// of a 256-K stage (128-byte swizzle) arrive by TMA on one barrier of the
// leader, scale atoms on one of each CTA's own.  With tokens on the lanes
// an epilogue thread holds consecutive features of one row.
//
// The MMA reads its scales from tensor memory: of rows m and 32 + m, 64 + m,
// 96 + m on lane m, the same in all four lane quarters.  Four warps per CTA,
// one per quarter, move them there through registers (tcgen05.st), one stage
// ahead in the other of two buffers, while the MMAs of a stage run.  Copying
// them with tcgen05.cp from the MMA's thread instead takes the tensor pipe's
// own time: at 9216 x 16384 x 4096 nvfp4 the MMAs alone took
// 213 us, the copies alone 190 more, and the kernel 414.
constexpr int BM = 128;       // tokens per block and CTA (MMA M = 256 for the pair)
constexpr int BKB = kStageK / 2;  // bytes of one operand row in a stage
constexpr uint32_t kTmemCols = 512;
constexpr int kGroupM = 16;  // token tiles that walk the feature tiles together (L2 reuse of the weight)

template <int F, int kBlocks, int BN>
struct Plan {
  static constexpr int BNC = BN / 2;  // weight rows per CTA
  static constexpr int AP = Traits<F>::kAtoms;
  static constexpr int kA = kBlocks * BM * BKB;       // this CTA's token rows
  static constexpr int kB = BNC * BKB;                // this CTA's weight rows
  static constexpr int kSfa = kBlocks * AP * kAtom;   // its tokens' scales
  static constexpr int kSfb = 2 * AP * kAtom;         // the two 128-feature row tiles that BN features touch
  static constexpr int kStage = kA + kB + kSfa + kSfb;
  static constexpr uint32_t kStageTx = 2u * (kA + kB);  // both CTAs' codes land on the leader's barrier
  static constexpr int kEpiWarps = 8;  // per lane quarter: one for each block, or two for the columns of one
  static constexpr int kParts = 2 / kBlocks;
  static constexpr int kSfWarp0 = kEpiWarps;  // four warps that bring scales to TMEM
  static constexpr int kTmaWarp = kEpiWarps + 4, kMmaWarp = kEpiWarps + 5;
  static constexpr int kThreads = 32 * (kEpiWarps + 6);
  static constexpr int kAccBufs = kBlocks == 1 ? 2 : 1;
  static constexpr int kStagesRaw = (227 * 1024 - 1024 - 512 - gemm::kGeluTabBytes) / kStage;
  static constexpr int kStages = kStagesRaw > 8 ? 8 : kStagesRaw;
  static constexpr int kBOff = kStages * kA;
  static constexpr int kSfaOff = kBOff + kStages * kB;
  static constexpr int kSfbOff = kSfaOff + kStages * kSfa;
  static constexpr int kBarOff = kSfbOff + kStages * kSfb;
  static constexpr int kTabOff = kBarOff + 512;
  static constexpr int kSmem = 1024 + kTabOff + gemm::kGeluTabBytes;
  // TMEM: accumulators, then two buffers of scales: block b, atom a at 4 (b AP + a);
  // behind them the weight's two row tiles of atom a side by side at 8 a
  static constexpr uint32_t kSfCol = 2 * BN;
  static constexpr uint32_t kSfbOffCol = 4 * kBlocks * AP;
  static constexpr uint32_t kSfCols = (kSfbOffCol + 8 * AP + 15) / 16 * 16;  // stores are 16 columns wide
  static_assert(kSfCol + 2 * kSfCols <= kTmemCols, "TMEM columns");
  // a tile starts 0 or 64 features into a row tile, 0 or 2 columns into its scales: the MMA faults on odd columns
  static_assert(BN % 64 == 0 && BN <= 192, "tile width");
  static_assert(kStages >= 4, "pipeline depth");
  static_assert(kSmem <= 227 * 1024, "shared memory budget");
  static_assert(kA % 1024 == 0 && kB % 1024 == 0, "128B-swizzle atoms need 1024-byte alignment");
  static_assert((3 * kStages + 8) * 8 + 8 <= 512, "barrier area");
};

// Instruction descriptor of kind::mxf4 / kind::mxf4nvf4: E2M1 A and B, K-major,
// fp32 accumulators; scales E8M0 (two bytes of a scale word per MMA, sf_id 0
// or 2) or E4M3 (all four, sf_id 0).
template <int F>
__host__ __device__ constexpr uint32_t idesc_fp4(uint32_t M, uint32_t N, uint32_t sf_id) {
  return (sf_id << 4) | (1u << 7) | (1u << 10) | ((N >> 3) << 17) | ((F == kMx ? 1u : 0u) << 23) | ((M >> 4) << 24) |
         (sf_id << 29);
}

template <int F>
__device__ __forceinline__ void mma_fp4_pair(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                             uint32_t sfb, uint32_t accumulate) {
  if (F == kNv)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
}

struct GemmArgs {
  int x_tiles, w_tiles;  // row tiles of the two scale layouts
  float alpha;           // product of the operands' global scales
  int chained;           // host: launched behind the kernel that quantizes x
};

template <int F, int kBlocks, int BN>
__global__ void __launch_bounds__(Plan<F, kBlocks, BN>::kThreads, 1)
    qgemm_fp4_pair_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_sfx,
                          const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_sfw,
                          const GemmArgs a, const gemm::Params p) {
  using P = Plan<F, kBlocks, BN>;
  constexpr int S = P::kStages;
  constexpr int AP = P::AP;
  constexpr int kRows = kBlocks * BM;  // token rows per CTA
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + P::kBarOff);
  uint64_t* full = bars;                   // leader: the stage's codes landed in both CTAs
  uint64_t* empty = bars + S;              // stage consumed by the MMAs (commit, to both CTAs)
  uint64_t* sf_full = bars + 2 * S;        // this CTA's scales of the stage landed
  uint64_t* acc_full = bars + 3 * S;       // [kAccBufs]
  uint64_t* acc_empty = bars + 3 * S + 2;  // [kAccBufs], leader: both CTAs' epilogues have read the accumulator
  uint64_t* sf_ready = bars + 3 * S + 4;   // [2], leader: both CTAs' scales are in TMEM
  uint64_t* sf_empty = bars + 3 * S + 6;   // [2] scales in TMEM consumed (commit, to both CTAs)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 3 * S + 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint16_t* gtab = reinterpret_cast<uint16_t*>(smem + P::kTabOff);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int num_kb = (p.K + kStageK - 1) / kStageK;
  const int n_t = (p.N + BN - 1) / BN;
  const int m_t = (p.M + 2 * kRows - 1) / (2 * kRows);
  const int tiles = n_t * m_t;
  const int cluster_id = static_cast<int>(blockIdx.x >> 1);
  const int n_clusters = static_cast<int>(gridDim.x >> 1);
  // tile t -> this CTA's first token row m0, the tile's first feature n0
  auto coords = [&](int t, int& m0, int& n0) {
    const int span = kGroupM * n_t;
    const int grp = t / span;
    const int rem_m = m_t - grp * kGroupM;
    const int gm = rem_m < kGroupM ? rem_m : kGroupM;
    const int w = t - grp * span;
    n0 = (w / gm) * BN;
    m0 = (grp * kGroupM + w % gm) * (2 * kRows) + static_cast<int>(rank) * kRows;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&sf_full[s], 1);
    }
    for (int b = 0; b < P::kAccBufs; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * P::kEpiWarps);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sf_ready[b], 8);  // four warps of each CTA
      mbar_init(&sf_empty[b], 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == P::kMmaWarp) {
    tmem_alloc_pair(tmem_slot, kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();  // barriers of both CTAs initialized, TMEM allocated
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t leader_full = mapa_shared(smem_u32(full), 0);
  const uint32_t leader_acc_empty = mapa_shared(smem_u32(acc_empty), 0);
  const uint32_t leader_sf_ready = mapa_shared(smem_u32(sf_ready), 0);

  if (warp == P::kTmaWarp) {
    if (lane == 0) {
      tma_prefetch_desc(&tmap_x);
      tma_prefetch_desc(&tmap_sfx);
      tma_prefetch_desc(&tmap_w);
      tma_prefetch_desc(&tmap_sfw);
      chain_wait();  // activations quantized by the kernel before this one
      bool ok = true;
      int g = 0;
      for (int t = cluster_id; t < tiles && ok; t += n_clusters) {
        int m0, n0;
        coords(t, m0, n0);
        for (int kb = 0; kb < num_kb; ++kb, ++g) {
          const int s = g % S;
          if (!mbar_wait(&empty[s], ((g / S) & 1) ^ 1, abort_flag, p.err)) {
            ok = false;
            break;
          }
          if (leader) mbar_arrive_expect_tx(&full[s], P::kStageTx);
          const uint32_t bar = leader_full + 8u * s;
          tma_load_2d_pair(smem + s * P::kA, &tmap_x, bar, kb * BKB, m0);
          tma_load_2d_pair(smem + P::kBOff + s * P::kB, &tmap_w, bar, kb * BKB, n0 + static_cast<int>(rank) * P::BNC);
          mbar_arrive_expect_tx(&sf_full[s], P::kSfa + P::kSfb);
          tma_load_2d(smem + P::kSfaOff + s * P::kSfa, &tmap_sfx, &sf_full[s], 0, (kb * a.x_tiles + m0 / BM) * AP);
          tma_load_2d(smem + P::kSfbOff + s * P::kSfb, &tmap_sfw, &sf_full[s], 0, (kb * a.w_tiles + n0 / 128) * AP);
        }
      }
      if (*abort_flag) {
        // give copies already in flight time to land before smem is released
        const uint64_t t0 = globaltimer();
        while (globaltimer() - t0 < 50000ull) {
        }
      }
    }
  } else if (warp == P::kMmaWarp) {
    if (leader && lane == 0) {
      bool ok = true;
      int it = 0, g = 0;
      for (int t = cluster_id; t < tiles && ok; t += n_clusters, ++it) {
        int m0, n0;
        coords(t, m0, n0);
        const int buf = it % P::kAccBufs;
        if (!mbar_wait(&acc_empty[buf], ((it / P::kAccBufs) & 1) ^ 1, abort_flag, p.err)) break;
        tc_fence_after();
        const uint32_t skip = static_cast<uint32_t>(n0 & 127) / 32;  // where the tile starts within its row tile
        for (int kb = 0; kb < num_kb; ++kb, ++g) {
          const int s = g % S;
          const int sb = g & 1;
          if (!mbar_wait(&full[s], (g / S) & 1, abort_flag, p.err) ||
              !mbar_wait(&sf_ready[sb], (g >> 1) & 1, abort_flag, p.err)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sf = tmem + P::kSfCol + static_cast<uint32_t>(sb) * P::kSfCols;
          const uint32_t aaddr = smem_u32(smem + s * P::kA);
          const uint32_t baddr = smem_u32(smem + P::kBOff + s * P::kB);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const int atom = F == kNv ? kk : kk >> 1;
            const uint32_t id = F == kNv ? 0u : 2u * (kk & 1);
            const uint32_t idesc = idesc_fp4<F>(2 * BM, BN, id);
            const uint32_t sfb = (id << 30) | (sf + P::kSfbOffCol + 8u * atom + skip);
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
              const uint32_t d = tmem + static_cast<uint32_t>((kBlocks == 1 ? buf : b) * BN);
              const uint32_t sfa = (id << 30) | (sf + 4u * (b * AP + atom));
              mma_fp4_pair<F>(d, smem_desc_sw128(aaddr + b * (BM * BKB) + kk * 32), smem_desc_sw128(baddr + kk * 32),
                              idesc, sfa, sfb, (kb | kk) != 0 ? 1u : 0u);
            }
          }
          mma_commit_pair(&empty[s], 0x3);
          mma_commit_pair(&sf_empty[sb], 0x3);
        }
        if (!ok) break;
        mma_commit_pair(&acc_full[buf], 0x3);
      }
      if (*abort_flag) {
        // give MMAs already issued time to complete before TMEM is released
        const uint64_t t0 = globaltimer();
        while (globaltimer() - t0 < 50000ull) {
        }
      }
    }
  } else if (warp >= P::kSfWarp0) {
    // ------------------------------------------------ scales, shared memory -> this warp's lane quarter of TMEM
    const uint32_t t_lane = static_cast<uint32_t>((warp & 3) * 32) << 16;
    bool ok = true;
    int g = 0;
    for (int t = cluster_id; t < tiles && ok; t += n_clusters) {
      for (int kb = 0; kb < num_kb; ++kb, ++g) {
        const int s = g % S, sb = g & 1;
        if (!mbar_wait_warp(&sf_full[s], (g / S) & 1, abort_flag, p.err)) {
          ok = false;
          break;
        }
        // an atom is 32 rows of 16 bytes: a lane's row is its four columns
        const uint8_t* sfa = smem + P::kSfaOff + s * P::kSfa + lane * 16;
        const uint8_t* sfb = smem + P::kSfbOff + s * P::kSfb + lane * 16;
        uint32_t r[P::kSfCols] = {};
#pragma unroll
        for (int i = 0; i < kBlocks * AP; ++i) {
          const uint4 v = *reinterpret_cast<const uint4*>(sfa + i * kAtom);
          r[4 * i] = v.x; r[4 * i + 1] = v.y; r[4 * i + 2] = v.z; r[4 * i + 3] = v.w;
        }
#pragma unroll
        for (int i = 0; i < 2 * AP; ++i) {  // row tile i / AP, atom i % AP
          const uint4 v = *reinterpret_cast<const uint4*>(sfb + i * kAtom);
          const int c = P::kSfbOffCol + 8 * (i % AP) + 4 * (i / AP);
          r[c] = v.x; r[c + 1] = v.y; r[c + 2] = v.z; r[c + 3] = v.w;
        }
        if (!mbar_wait_warp(&sf_empty[sb], ((g >> 1) & 1) ^ 1, abort_flag, p.err)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t dst = tmem + t_lane + P::kSfCol + static_cast<uint32_t>(sb) * P::kSfCols;
#pragma unroll
        for (uint32_t c = 0; c < P::kSfCols; c += 16) tmem_st_32x32b_x16(dst + c, r + c);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(leader_sf_ready + 8u * static_cast<uint32_t>(sb));
      }
    }
  } else {
    // ------------------------------------------------ epilogue warps
    const int q = warp & 3;     // TMEM lane quarter of this warp
    const int blk = kBlocks == 2 ? warp >> 2 : 0;   // its block of token rows
    const int part = kBlocks == 2 ? 0 : warp >> 2;  // its share of the columns
    const uint32_t t_lane = static_cast<uint32_t>(q * 32) << 16;
    const bool gated = p.epi == LTXQ_EPI_GATED_RESIDUAL || p.epi == LTXQ_EPI_GATE_THEN_ADD;
    const bool two_round = p.epi == LTXQ_EPI_GATE_THEN_ADD || p.gate.dtype == LTXQ_BF16;
    if (p.epi == LTXQ_EPI_GELU) {
      gemm::gelu_tab_fill(gtab, threadIdx.x, 32 * P::kEpiWarps);  // while the first tile's main loop runs
      gemm::named_bar_sync(1, 32 * P::kEpiWarps);
    }
    for (int t = cluster_id, it = 0; t < tiles; t += n_clusters, ++it) {
      int m0, n0;
      coords(t, m0, n0);
      const int buf = it % P::kAccBufs;
      if (!mbar_wait_warp(&acc_full[buf], (it / P::kAccBufs) & 1, abort_flag, p.err)) break;
      tc_fence_after();
      const uint32_t tacc = tmem + t_lane + static_cast<uint32_t>((kBlocks == 1 ? buf : blk) * BN);
      const int m0w = m0 + blk * BM + q * 32;  // first token of this warp
#pragma unroll 1
      for (int c = part; c < BN / 32; c += P::kParts) {
        if (n0 + c * 32 >= p.N) break;  // uniform
        uint32_t v[32], u[4][4];
        tmem_ld_32x32b_x32(tacc + c * 32, v);
        tmem_wait_ld();
        gemm::epi_pack32(a.alpha, v, u);
        gemm::epi_rows32(p, u, m0w, n0 + c * 32, gated, two_round, gtab);
      }
      tc_fence_before();
      __syncwarp();  // each warp for itself: a barrier of all would have no limit if one of them gave up
      if (lane == 0) mbar_arrive_cluster(leader_acc_empty + 8u * static_cast<uint32_t>(buf));
    }
  }

  tc_fence_before();
  cluster_sync_all();  // no CTA leaves while its peer may still signal or read it
  if (warp == P::kMmaWarp) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, kTmemCols);
  }
}

// ---------------------------------------------------------------- host side

static size_t align_up(size_t v) { return (v + 255) & ~size_t(255); }

struct Sizes {
  int64_t stages, row_tiles;
  size_t codes, scales;
};
static Sizes sizes(int64_t rows, int64_t K, int32_t mode) {
  Sizes s{};
  s.stages = (K + kStageK - 1) / kStageK;
  s.row_tiles = (rows + 127) / 128;
  s.codes = static_cast<size_t>(rows) * static_cast<size_t>(K / 2);
  s.scales = static_cast<size_t>(s.stages * s.row_tiles) * (mode == LTXQ_NVFP4 ? 4 : 2) * kAtom;
  return s;
}

static bool is_fp4(int32_t mode) { return mode == LTXQ_MXFP4 || mode == LTXQ_NVFP4; }

static ltxq_status check_act(const ltxq_fp4_act* a, int64_t M, int64_t K, float* g, const char* what) {
  if (!a || !a->codes || !a->scales) return fail(LTXQ_ERR_INVALID, std::string(what) + ": NULL pointer");
  if (!is_fp4(a->mode)) return fail(LTXQ_ERR_INVALID, std::string(what) + ": mode must be mxfp4 or nvfp4");
  if (M < 0 || K <= 0) return fail(LTXQ_ERR_INVALID, std::string(what) + ": bad shape");
  if (K % 32 != 0) return fail(LTXQ_ERR_UNSUPPORTED, std::string(what) + ": K must be a multiple of 32");
  if (M > 0x7FFFFFFF / 2 || K > 0x7FFFFFFF / 2)
    return fail(LTXQ_ERR_UNSUPPORTED, std::string(what) + ": dimension too large");
  if ((reinterpret_cast<uintptr_t>(a->codes) | reinterpret_cast<uintptr_t>(a->scales)) & 15u)
    return fail(LTXQ_ERR_UNSUPPORTED, std::string(what) + ": codes / scales must be 16-byte aligned");
  return fp4_global_scale(a->mode, a->global_scale, g, what);
}

template <int F, int kBlocks, int BN>
static ltxq_status launch_pair(const ltxq_fp4_act& x, const ltxq_qweight& w, const GemmArgs& a, const gemm::Params& p,
                               cudaStream_t stream) {
  using PL = Plan<F, kBlocks, BN>;
  const Sizes sx = sizes(p.M, p.K, x.mode), sw = sizes(p.N, p.K, x.mode);
  CUtensorMap tx, tsx, tw, tsw;
  if (ltxq_status st = encode_tmap_2d(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, x.codes, p.K / 2, p.M, p.K / 2, BKB,
                                      kBlocks * BM, CU_TENSOR_MAP_SWIZZLE_128B))
    return st;
  if (ltxq_status st = encode_tmap_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, w.weight, p.K / 2, p.N, p.K / 2, BKB, PL::BNC,
                                      CU_TENSOR_MAP_SWIZZLE_128B))
    return st;
  // scale atoms as rows of 128 words
  if (ltxq_status st = encode_tmap_2d(&tsx, CU_TENSOR_MAP_DATA_TYPE_UINT32, x.scales, 128, sx.scales / kAtom, kAtom, 128,
                                      kBlocks * PL::AP, CU_TENSOR_MAP_SWIZZLE_NONE))
    return st;
  if (ltxq_status st = encode_tmap_2d(&tsw, CU_TENSOR_MAP_DATA_TYPE_UINT32, w.mx_scales, 128, sw.scales / kAtom, kAtom,
                                      128, 2 * PL::AP, CU_TENSOR_MAP_SWIZZLE_NONE))
    return st;
  auto kern = qgemm_fp4_pair_kernel<F, kBlocks, BN>;
  static SmemAttr attr_done;
  if (ltxq_status st = attr_done.set(reinterpret_cast<const void*>(kern), PL::kSmem)) return st;
  const int tiles = ((p.M + 2 * kBlocks * BM - 1) / (2 * kBlocks * BM)) * ((p.N + BN - 1) / BN);
  const int max_clusters = num_sms() / 2;
  const int clusters = tiles < max_clusters ? tiles : max_clusters;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * clusters);
  cfg.blockDim = dim3(PL::kThreads);
  cfg.dynamicSmemBytes = PL::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1] = chained_attr();
  cfg.attrs = attr;
  cfg.numAttrs = a.chained ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tx, tsx, tw, tsw, a, p);
  if (e == cudaSuccess) note_launch();
  return cuda_check(e, "fp4 block-scaled GEMM launch");
}

// Behind the kernel that quantizes x the product is chained: 751 x 2048 x 2048
// 11.3 us in all, was 12.1; 9216 x 16384 x 4096 nvfp4 355, was 375.
// 512 x 192 tiles where they fill every cluster once (fewest bytes per MMA: 282
// us against 324 with 256 x 192 at 9216 x 16384 x 4096), else 256 x 192.
// (256 x 128, 48 tiles instead of 33 at 751 x 2048 x 2048: 11.4 us, as before.)
template <int F>
static ltxq_status launch_gemm(const ltxq_fp4_act& x, const ltxq_qweight& w, const GemmArgs& a, const gemm::Params& p,
                               cudaStream_t stream) {
  const int64_t n_t = (p.N + 191) / 192;
  const int clusters = num_sms() / 2;
  return (p.M + 511) / 512 * n_t >= clusters ? launch_pair<F, 2, 192>(x, w, a, p, stream)
                                             : launch_pair<F, 1, 192>(x, w, a, p, stream);
}

}  // namespace fp4

// Bytes of workspace a product over `w` needs for its quantized activations
// (codes, then scale atoms), or 0 where `w` does not compute in fp4.
size_t fp4_workspace_bytes(int64_t M, const ltxq_qweight& w) {
  if (w.compute != LTXQ_COMPUTE_FP4 || !fp4::is_fp4(w.mode) || w.layout != LTXQ_LAYOUT_STD) return 0;
  if (fp4_rows_supported(M, w)) return 0;  // the few-row kernel quantizes as it reads
  if (M <= 0 || w.k_in <= 0 || w.k_in % 32 != 0) return 0;
  const fp4::Sizes s = fp4::sizes(M, w.k_in, w.mode);
  return fp4::align_up(s.codes) + fp4::align_up(s.scales);
}

ltxq_status launch_qlinear_fp4(const ltxq_fp4_act& x, int64_t M, const ltxq_qweight& w, const gemm::Params& p,
                               cudaStream_t stream, bool chained) {
  float gx, gw;
  if (ltxq_status st = fp4::check_act(&x, M, w.k_in, &gx, "qlinear_fp4")) return st;
  if (ltxq_status st = fp4_global_scale(w.mode, w.global_scale, &gw, "qlinear_fp4")) return st;
  if (x.mode != w.mode) return fail(LTXQ_ERR_INVALID, "qlinear_fp4: x and the weight have different formats");
  if (fp4_rows_supported(M, w)) {
    gemm::Params q = p;
    q.alpha = gx * gw;
    return launch_fp4_rows(nullptr, false, &x, w, q, stream);
  }
  if (!w.mx_scales || (reinterpret_cast<uintptr_t>(w.mx_scales) & 15u))
    return fail(LTXQ_ERR_INVALID, "qlinear_fp4: mx_scales (ltxq_fp4_pack_weight_scales) is NULL or not 16-byte aligned");
  fp4::GemmArgs a{static_cast<int>((M + 127) / 128), static_cast<int>((w.n_out + 127) / 128), gx * gw, chained ? 1 : 0};
  return w.mode == LTXQ_NVFP4 ? fp4::launch_gemm<fp4::kNv>(x, w, a, p, stream)
                              : fp4::launch_gemm<fp4::kMx>(x, w, a, p, stream);
}

ltxq_status launch_fp4_quantize(const void* x, int64_t M, int64_t K, int64_t row_stride, const ltxq_fp4_act& o, float g,
                                cudaStream_t s) {
  const fp4::RowGrid r = fp4::row_grid(M, (K + fp4::kStageK - 1) / fp4::kStageK * (fp4::kStageK / 16));
  auto* src = static_cast<const uint16_t*>(x);
  auto* c = static_cast<uint8_t*>(o.codes);
  auto* sc = static_cast<uint8_t*>(o.scales);
  const int k = static_cast<int>(K);
  if (o.mode == LTXQ_MXFP4)
    fp4::quantize_kernel<fp4::kMx, true, false><<<r.grid, 256, 0, s>>>(src, M, k, row_stride, g, r.log_width, c, sc);
  else if (fp4::power_of_two(g))
    fp4::quantize_kernel<fp4::kNv, true, false><<<r.grid, 256, 0, s>>>(src, M, k, row_stride, g, r.log_width, c, sc);
  else
    fp4::quantize_kernel<fp4::kNv, true, true><<<r.grid, 256, 0, s>>>(src, M, k, row_stride, g, r.log_width, c, sc);
  return launch_check("fp4 quantize launch");
}

// From bf16 activations: quantize x into the workspace, then the product.
// The caller checked shapes, alignment and the epilogue and that the
// workspace holds fp4_workspace_bytes(M, w).
ltxq_status launch_qlinear_fp4_from_bf16(const void* x, int64_t M, const ltxq_qweight& w, const gemm::Params& p,
                                         void* workspace, cudaStream_t stream) {
  const fp4::Sizes s = fp4::sizes(M, w.k_in, w.mode);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const ltxq_fp4_act a{ws, ws + fp4::align_up(s.codes), w.mode, 1.0f};
  if (ltxq_status st = launch_fp4_quantize(x, M, w.k_in, w.k_in, a, 1.0f, stream)) return st;
  return launch_qlinear_fp4(a, M, w, p, stream, true);
}

}  // namespace ltxq

extern "C" {

size_t ltxq_fp4_sizes(int64_t rows, int64_t K, int32_t mode, size_t* codes_bytes, size_t* scale_bytes) {
  if (rows <= 0 || K <= 0 || K % 32 != 0 || !ltxq::fp4::is_fp4(mode)) return 0;
  const ltxq::fp4::Sizes s = ltxq::fp4::sizes(rows, K, mode);
  if (codes_bytes) *codes_bytes = s.codes;
  if (scale_bytes) *scale_bytes = s.scales;
  return static_cast<size_t>(s.row_tiles);
}

ltxq_status ltxq_fp4_quantize(const void* x, int64_t M, int64_t K, int64_t row_stride, const ltxq_fp4_act* out,
                              void* stream) {
  using namespace ltxq;
  float g;
  if (ltxq_status st = fp4::check_act(out, M, K, &g, "fp4_quantize")) return st;
  if (!x) return fail(LTXQ_ERR_INVALID, "fp4_quantize: x is NULL");
  if (row_stride < K) return fail(LTXQ_ERR_INVALID, "fp4_quantize: row_stride < K");
  if (row_stride % 8 != 0 || (reinterpret_cast<uintptr_t>(x) & 15u))
    return fail(LTXQ_ERR_UNSUPPORTED, "fp4_quantize: rows of x must be 16-byte aligned");
  if (M == 0) return LTXQ_OK;
  return launch_fp4_quantize(x, M, K, row_stride, *out, g, static_cast<cudaStream_t>(stream));
}

ltxq_status ltxq_fp4_dequantize(const ltxq_fp4_act* a, int64_t M, int64_t K, void* out, void* stream) {
  using namespace ltxq;
  float g;
  if (ltxq_status st = fp4::check_act(a, M, K, &g, "fp4_dequantize")) return st;
  if (!out) return fail(LTXQ_ERR_INVALID, "fp4_dequantize: out is NULL");
  if (reinterpret_cast<uintptr_t>(out) & 15u) return fail(LTXQ_ERR_UNSUPPORTED, "fp4_dequantize: out not 16-byte aligned");
  if (M == 0) return LTXQ_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const fp4::RowGrid r = fp4::row_grid(M, K / 16);
  const int k = static_cast<int>(K);
  auto* c = static_cast<const uint8_t*>(a->codes);
  auto* sc = static_cast<const uint8_t*>(a->scales);
  auto* o = static_cast<uint16_t*>(out);
  if (a->mode == LTXQ_MXFP4)
    fp4::dequantize_kernel<fp4::kMx, true><<<r.grid, 256, 0, s>>>(c, sc, M, k, g, r.log_width, o);
  else
    fp4::dequantize_kernel<fp4::kNv, true><<<r.grid, 256, 0, s>>>(c, sc, M, k, g, r.log_width, o);
  return launch_check("fp4 dequantize launch");
}

size_t ltxq_fp4_weight_scales_size(const ltxq_qweight* w) {
  if (!w || w->layout != LTXQ_LAYOUT_STD) return 0;
  size_t bytes = 0;
  return ltxq_fp4_sizes(w->n_out, w->k_in, w->mode, nullptr, &bytes) ? bytes : 0;
}

ltxq_status ltxq_fp4_pack_weight_scales(const ltxq_qweight* w, void* out, void* stream) {
  using namespace ltxq;
  if (!w || !out || !w->scales) return fail(LTXQ_ERR_INVALID, "fp4_pack_weight_scales: NULL argument");
  if (!ltxq_fp4_weight_scales_size(w))
    return fail(LTXQ_ERR_UNSUPPORTED, "fp4_pack_weight_scales: mxfp4 / nvfp4 weights, standard layout, K % 32 == 0");
  if (reinterpret_cast<uintptr_t>(out) & 15u)
    return fail(LTXQ_ERR_UNSUPPORTED, "fp4_pack_weight_scales: out must be 16-byte aligned");
  int64_t R, L;
  if (ltxq_status st = check_qweight(*w, false, &R, &L)) return st;
  const int64_t G = L / w->group_size;
  const int64_t Gp = (L + fp4::kStageK - 1) / fp4::kStageK * (fp4::kStageK / w->group_size);
  const unsigned grid = fp4::grid_for((R + 127) / 128 * 128 * Gp);
  auto* sc = static_cast<const uint8_t*>(w->scales);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (w->mode == LTXQ_MXFP4)
    fp4::pack_scales_kernel<fp4::kMx><<<grid, 256, 0, s>>>(sc, R, G, Gp, static_cast<uint8_t*>(out));
  else
    fp4::pack_scales_kernel<fp4::kNv><<<grid, 256, 0, s>>>(sc, R, G, Gp, static_cast<uint8_t*>(out));
  return launch_check("fp4 pack scales launch");
}

ltxq_status ltxq_qlinear_fp4(const ltxq_fp4_act* x, int64_t M, const ltxq_qweight* w, const ltxq_epilogue* epi,
                             void* out, void* stream) {
  using namespace ltxq;
  if (!x || !w) return fail(LTXQ_ERR_INVALID, "qlinear_fp4: NULL argument");
  if (M < 0) return fail(LTXQ_ERR_INVALID, "qlinear_fp4: M < 0");
  if (!fp4::is_fp4(w->mode) || w->layout != LTXQ_LAYOUT_STD)
    return fail(LTXQ_ERR_UNSUPPORTED, "qlinear_fp4: the weight must be mxfp4 or nvfp4 in the standard layout");
  float gx, gw;
  if (ltxq_status st = fp4::check_act(x, M, w->k_in, &gx, "qlinear_fp4")) return st;
  if (ltxq_status st = fp4_global_scale(w->mode, w->global_scale, &gw, "qlinear_fp4")) return st;
  // one fp32 factor of the sums, with room for the 2^8 of decoded weights (fp4.cuh)
  if (gx * gw < 0x1p-96f || gx * gw > 0x1p96f)
    return fail(LTXQ_ERR_UNSUPPORTED, "qlinear_fp4: the product of the global scales must be within [2^-96, 2^96]");
  gemm::Params p{};
  if (ltxq_status st = qlinear_params(x->codes, M, *w, epi, out, &p)) return st;
  if (M == 0) return LTXQ_OK;
  return launch_qlinear_fp4(*x, M, *w, p, static_cast<cudaStream_t>(stream), false);
}

}  // extern "C"
