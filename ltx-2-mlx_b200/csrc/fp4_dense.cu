// fp4_dense.cu -- products of many bf16 rows with an mxfp4 / nvfp4 weight: the
// weight dequantized into the workspace (exact in bf16), then a dense bf16
// product on the tensor cores.
//
// The fused kernel (qgemm.cu) converts every weight tile again for each 256
// tokens, and its conversion warps, which feed the MMA through tensor memory,
// bound it at 780 to 1090 TFLOP/s.  From a few tiles of tokens on, converting
// the weight once (2.5 bytes moved per element) and running both operands by
// TMA costs less: 3456 x 4096 x 4096 takes 88 us, the fused kernel 117.
//
// Persistent kernel, clusters of two CTAs (tcgen05 cta_group::2), tiles of 256
// tokens x 256 features: CTA r holds token rows [m0 + 128 r, +128) (operand A,
// TMEM lanes = tokens) and 128 weight rows (operand B); a 64-K stage of both
// arrives by TMA on one barrier of the leader.  Two accumulators let the
// epilogue of one tile run while the next accumulates.  At 3456 x 4096 x
// 4096 the MMAs keep the tensor pipe busy 79 % of the kernel's cycles.  Narrower tiles, which fill the last wave
// better, were slower throughout (each byte from L2 feeds fewer MMAs: 192
// features 117 us and 128 features 151 us where 256 take 97); instead the last
// wave's tiles are split along K by the pair kernels' schedule (qgemm.cu).  The
// kernel sets itself up while the weight is still being dequantized (1536 x 2048
// x 2048 19.3 us, was 20.2); the split tiles' sum is launched plainly behind it
// (chained too, 3456 x 4096 x 4096 took 100.6 us instead of 88.6).
#include "common.cuh"
#include "fp4.cuh"
#include "gemm_epilogue.cuh"

namespace ltxq {

ltxq_status launch_fp4_dequantize_rows(const uint8_t* codes, const uint8_t* scales, int64_t R, int64_t L, int32_t mode,
                                       float g, uint16_t* out, cudaStream_t s);

namespace dense {

constexpr int BM = 128;  // tokens per CTA
constexpr int BN = 256;  // features per tile
constexpr int BK = 64;   // K per stage (128 bytes of a row)
constexpr uint32_t kTmemCols = 512;
constexpr int kEpiWarps = 8, kTmaWarp = 8, kMmaWarp = 9, kThreads = 320;  // two epilogue warps per lane quarter
constexpr int kGroupM = 16;  // token tiles that walk the feature tiles together (L2 reuse of the weight)

struct Plan {
  static constexpr int kA = BM * BK * 2;
  static constexpr int kB = BN / 2 * BK * 2;
  static constexpr int kStage = kA + kB;
  static constexpr int kStagesRaw = (227 * 1024 - 1024 - 512 - gemm::kGeluTabBytes) / kStage;
  static constexpr int kStages = kStagesRaw > 8 ? 8 : kStagesRaw;
  static constexpr int kBOff = kStages * kA;
  static constexpr int kBarOff = kStages * kStage;
  static constexpr int kTabOff = kBarOff + 512;
  static constexpr int kSmem = 1024 + kTabOff + gemm::kGeluTabBytes;
  static_assert(2 * BN <= static_cast<int>(kTmemCols), "two accumulators");
  static_assert(kA % 1024 == 0 && kB % 1024 == 0, "128B-swizzle atoms need 1024-byte alignment");
  static_assert(kSmem <= 227 * 1024, "shared memory budget");
};

__global__ void __launch_bounds__(kThreads, 1)
    gemm_bf16_pair_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
                          const gemm::Params p) {
  using P = Plan;
  constexpr int S = P::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + P::kBarOff);
  uint64_t* full = bars;
  uint64_t* empty = bars + S;
  uint64_t* acc_full = bars + 2 * S;       // [2]
  uint64_t* acc_empty = bars + 2 * S + 2;  // [2], leader: both CTAs' epilogues have read the accumulator
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint16_t* gtab = reinterpret_cast<uint16_t*>(smem + P::kTabOff);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int num_kb = (p.K + BK - 1) / BK;
  const int n_t = (p.N + BN - 1) / BN;
  const int m_t = (p.M + 2 * BM - 1) / (2 * BM);
  const int tiles = n_t * m_t;
  // unit u < dp: whole tile u; else K range sp of tile dp + (u - dp) / splits
  const int dp = p.dp_tiles, splits = p.splits, units = dp + (tiles - dp) * splits;
  const int cluster_id = static_cast<int>(blockIdx.x >> 1);
  const int n_clusters = static_cast<int>(gridDim.x >> 1);
  auto unit = [&](int u, int& m0, int& n0, int& sp, int& kb_lo, int& kb_hi) {
    int t = u;
    sp = -1;
    kb_lo = 0;
    kb_hi = num_kb;
    if (u >= dp) {
      t = dp + (u - dp) / splits;
      sp = (u - dp) - (t - dp) * splits;
      kb_lo = sp * num_kb / splits;
      kb_hi = (sp + 1) * num_kb / splits;
    }
    const int span = kGroupM * n_t;
    const int grp = t / span;
    const int rem_m = m_t - grp * kGroupM;
    const int gm = rem_m < kGroupM ? rem_m : kGroupM;
    const int w = t - grp * span;
    n0 = (w / gm) * BN;
    m0 = (grp * kGroupM + w % gm) * (2 * BM) + static_cast<int>(rank) * BM;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * kEpiWarps);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc_pair(tmem_slot, kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();  // barriers of both CTAs initialized, TMEM allocated
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t leader_full = mapa_shared(smem_u32(full), 0);
  const uint32_t leader_acc_empty = mapa_shared(smem_u32(acc_empty), 0);

  if (warp == kTmaWarp) {
    if (lane == 0) {
      tma_prefetch_desc(&tmap_x);
      tma_prefetch_desc(&tmap_w);
      chain_wait();  // the weight, written by the kernel before this one
      bool ok = true;
      int g = 0;
      for (int u = cluster_id; u < units && ok; u += n_clusters) {
        int m0, n0, sp, kb_lo, kb_hi;
        unit(u, m0, n0, sp, kb_lo, kb_hi);
        for (int kb = kb_lo; kb < kb_hi; ++kb, ++g) {
          const int s = g % S;
          if (!mbar_wait(&empty[s], ((g / S) & 1) ^ 1, abort_flag, p.err)) {
            ok = false;
            break;
          }
          if (leader) mbar_arrive_expect_tx(&full[s], 2 * P::kStage);
          const uint32_t bar = leader_full + 8u * s;
          tma_load_2d_pair(smem + s * P::kA, &tmap_x, bar, kb * BK, m0);
          tma_load_2d_pair(smem + P::kBOff + s * P::kB, &tmap_w, bar, kb * BK, n0 + static_cast<int>(rank) * (BN / 2));
        }
      }
      if (*abort_flag) {
        // give copies already in flight time to land before smem is released
        const uint64_t t0 = globaltimer();
        while (globaltimer() - t0 < 50000ull) {
        }
      }
    }
  } else if (warp == kMmaWarp) {
    if (leader && lane == 0) {
      const uint32_t idesc = idesc_bf16_f32(2 * BM, BN);
      bool ok = true;
      int it = 0, g = 0;
      for (int u = cluster_id; u < units && ok; u += n_clusters, ++it) {
        int m0, n0, sp, kb_lo, kb_hi;
        unit(u, m0, n0, sp, kb_lo, kb_hi);
        const int buf = it & 1;
        if (!mbar_wait(&acc_empty[buf], ((it >> 1) & 1) ^ 1, abort_flag, p.err)) break;
        tc_fence_after();
        const uint32_t d = tmem + static_cast<uint32_t>(buf * BN);
        for (int kb = kb_lo; kb < kb_hi; ++kb, ++g) {
          const int s = g % S;
          if (!mbar_wait(&full[s], (g / S) & 1, abort_flag, p.err)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t aaddr = smem_u32(smem + s * P::kA);
          const uint32_t baddr = smem_u32(smem + P::kBOff + s * P::kB);
#pragma unroll
          for (int j = 0; j < BK / 16; ++j)
            mma_bf16_ss_pair(d, smem_desc_sw128(aaddr + j * 32), smem_desc_sw128(baddr + j * 32), idesc,
                             (kb != kb_lo || j != 0) ? 1u : 0u);
          mma_commit_pair(&empty[s], 0x3);
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
  } else {
    const int q = warp & 3;  // TMEM lane quarter
    const uint32_t t_lane = static_cast<uint32_t>(q * 32) << 16;
    const bool gated = p.epi == LTXQ_EPI_GATED_RESIDUAL || p.epi == LTXQ_EPI_GATE_THEN_ADD;
    const bool two_round = p.epi == LTXQ_EPI_GATE_THEN_ADD || p.gate.dtype == LTXQ_BF16;
    if (p.epi == LTXQ_EPI_GELU) {
      gemm::gelu_tab_fill(gtab, threadIdx.x, 32 * kEpiWarps);  // while the first tile's main loop runs
      gemm::named_bar_sync(1, 32 * kEpiWarps);
    }
    for (int u = cluster_id, it = 0; u < units; u += n_clusters, ++it) {
      int m0, n0, sp, kb_lo, kb_hi;
      unit(u, m0, n0, sp, kb_lo, kb_hi);
      const int buf = it & 1;
      if (!mbar_wait_warp(&acc_full[buf], (it >> 1) & 1, abort_flag, p.err)) break;
      tc_fence_after();
      const uint32_t tacc = tmem + t_lane + static_cast<uint32_t>(buf * BN);
      const int m0w = m0 + q * 32;  // first token of this warp
#pragma unroll 1
      for (int c = warp >> 2; c < BN / 32; c += 2) {
        if (n0 + c * 32 >= p.N) break;  // uniform
        uint32_t v[32];
        tmem_ld_32x32b_x32(tacc + c * 32, v);
        tmem_wait_ld();
        if (sp >= 0) {  // fp32 partial, tile-local [token][feature]
          float* dst = p.partial + (static_cast<size_t>((u - dp) / splits) * splits + sp) * (2 * BM * BN) +
                       (static_cast<int>(rank) * BM + q * 32 + lane) * BN + c * 32;
          if (m0w + lane < p.M) {
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              *reinterpret_cast<float4*>(dst + j) =
                  make_float4(__fmul_rn(__uint_as_float(v[j]), p.alpha), __fmul_rn(__uint_as_float(v[j + 1]), p.alpha),
                              __fmul_rn(__uint_as_float(v[j + 2]), p.alpha), __fmul_rn(__uint_as_float(v[j + 3]), p.alpha));
          }
          continue;
        }
        uint32_t u8[4][4];
        gemm::epi_pack32(p.alpha, v, u8);
        gemm::epi_rows32(p, u8, m0w, n0 + c * 32, gated, two_round, gtab);
      }
      tc_fence_before();
      __syncwarp();  // each warp for itself: a barrier of all would have no limit if one of them gave up
      if (lane == 0) mbar_arrive_cluster(leader_acc_empty + 8u * static_cast<uint32_t>(buf));
    }
  }

  tc_fence_before();
  cluster_sync_all();  // no CTA leaves while its peer may still signal or read it
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, kTmemCols);
  }
}

static ltxq_status launch(const void* x, const void* w, const gemm::Params& p, cudaStream_t stream) {
  using PL = Plan;
  CUtensorMap tx, tw;
  if (ltxq_status st = encode_tmap_2d(&tx, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, x, p.K, p.M, static_cast<uint64_t>(p.K) * 2,
                                      BK, BM, CU_TENSOR_MAP_SWIZZLE_128B))
    return st;
  if (ltxq_status st = encode_tmap_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, w, p.K, p.N, static_cast<uint64_t>(p.K) * 2,
                                      BK, BN / 2, CU_TENSOR_MAP_SWIZZLE_128B))
    return st;
  auto kern = gemm_bf16_pair_kernel;
  static SmemAttr attr_done;
  if (ltxq_status st = attr_done.set(reinterpret_cast<const void*>(kern), PL::kSmem)) return st;
  const int tiles = ((p.M + 2 * BM - 1) / (2 * BM)) * ((p.N + BN - 1) / BN);
  const int units = p.dp_tiles + (tiles - p.dp_tiles) * p.splits;
  const int max_clusters = num_sms() / 2;
  const int clusters = units < max_clusters ? units : max_clusters;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * clusters);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = PL::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1] = chained_attr();
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tx, tw, p);
  if (e == cudaSuccess) note_launch();
  if (ltxq_status st = cuda_check(e, "dense bf16 GEMM launch")) return st;
  return p.dp_tiles < tiles ? gemm::launch_splitk_reduce(p, stream) : LTXQ_OK;
}

}  // namespace dense

// Workspace of the dequantized weight and behind it of the split tiles' partial
// sums (from *weight_bytes on; without them no tile is split), or 0 where the
// fused kernel runs.
size_t fp4_dense_bytes(int64_t M, const ltxq_qweight& w, size_t* weight_bytes) {
  if ((w.mode != LTXQ_MXFP4 && w.mode != LTXQ_NVFP4) || w.layout != LTXQ_LAYOUT_STD || w.compute == LTXQ_COMPUTE_FP4)
    return 0;
  if (w.n_out <= 0 || w.k_in <= 0 || w.k_in % 32 != 0) return 0;
  // 768 tokens and 48 tiles: below, the conversion pass costs more than it saves (512 x 4096 x 4096: 36 us against the
  // fused kernel's 28; 1024 x 2048 x 2048, 32 tiles: 26 against 21; 768 x 4096 x 4096: 37 against 43, 1536 x 2048 x
  // 2048: 22 against 28, 3456 x 4096 x 4096: 91 against 117).  Wide outputs come out even at the limit (768 x 4096 x
  // 16384: 109 against 108, 1024 rows: 129 against 126)
  if (M < 768 || (M + 255) / 256 * ((w.n_out + 255) / 256) < 48) return 0;
  const size_t weight = (static_cast<size_t>(w.n_out) * static_cast<size_t>(w.k_in) * 2 + 255) & ~size_t(255);
  if (weight_bytes) *weight_bytes = weight;
  return weight + gemm::splitk_bytes(M, w.n_out, w.k_in);
}

// p as qlinear_params filled it, checked; workspace 256-byte aligned, of fp4_dense_bytes()
// or at least of their part for the weight.
ltxq_status launch_qlinear_fp4_dense(const void* x, const ltxq_qweight& w, gemm::Params p, void* workspace,
                                     size_t workspace_bytes, cudaStream_t stream) {
  if (ltxq_status st = launch_fp4_dequantize_rows(static_cast<const uint8_t*>(w.weight),
                                                  static_cast<const uint8_t*>(w.scales), w.n_out, w.k_in, w.mode, 1.f,
                                                  static_cast<uint16_t*>(workspace), stream))
    return st;
  size_t off = 0;
  const size_t all = fp4_dense_bytes(p.M, w, &off);
  gemm::Sched sc = gemm::plan_schedule(p.M, p.N, p.K);
  if (workspace_bytes < all) sc.dp = sc.tiles, sc.splits = 1;
  p.dp_tiles = sc.dp;
  p.splits = sc.splits;
  p.partial = sc.splits > 1 ? reinterpret_cast<float*>(static_cast<char*>(workspace) + off) : nullptr;
  return dense::launch(x, workspace, p, stream);
}

}  // namespace ltxq
