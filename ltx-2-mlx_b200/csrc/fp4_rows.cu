// fp4_rows.cu -- products of a few rows with an mxfp4 / nvfp4 weight: single
// tokens and short batches, bound by reading and decoding the weight once.
//
// out[m, n] = epilogue(sum_k x[m, k] w[n, k]), M <= 16 rows.  x is kept in
// shared memory as bf16 -- as given, or quantized to the weight's format and
// read back there (exact: E2M1 times a scale has 6 bits), or read from an
// FP4Tensor -- so both computes share one kernel and one set of products,
// bf16 x bf16 in fp32 (mma.sync m16n8k16, weight rows on the MMA's 16 rows,
// tokens on its 8 columns: with so few tokens the tensor pipe idles anyway, and
// the decoded weight goes from registers into it).
//
// One CTA of 16 warps per SM.  A CTA takes tiles of 16 features; a warp takes
// every 16th block of 128 K of each, so x is read once per CTA, any N and K
// spread over all SMs, and the warps' partial sums meet in shared memory once
// per kT tiles, added in warp order.  A thread owns 32 consecutive K of two rows
// of a block (16 bytes each, streaming loads; the MMA's K order is a permutation
// that x is laid out in too) and loads kT blocks ahead.
//
// One token through 4096 x 16384 (nvfp4) takes 17.3 us, 2.2 TB/s of weight.  No
// unit is full: the counters of a launch from cold caches show the integer pipe,
// on which the words are decoded, busy 36 % of the cycles and issue slots 38 %;
// of a warp's time 41 % goes to waiting for its loads, 11 % to the barriers
// around x and the partial sums, 11 % to the full pipe and 2 % to instructions
// that are not there yet.  So the loads and the decoding, 16 warps of an SM in
// step, overlap only in part.  Measured and not kept: the weight through shared
// memory, by cp.async or TMA, with the loops rolled (17.7 to 20.8 us), and fp16
// products, whose decoding takes the hardware half the cycles (11 per warp and
// word of 8 on a quarter of an SM, against 23) but whose x needs a scan of its
// range (17.7 us, 26 against 18 at 8 rows).
#include "common.cuh"
#include "fp4.cuh"
#include "gemm_epilogue.cuh"

namespace ltxq {
namespace fp4 {

constexpr int kRowWarps = 16, kRowThreads = 32 * kRowWarps;
constexpr int kBlockK = 128;  // K per block: 4 threads of 32
// tiles per round, each with a block per warp in flight: as many as registers hold
constexpr int row_tiles(int nt) { return nt == 1 ? 4 : 2; }
constexpr int kMaxRows = 16;

enum FillX { kCopy = 0, kQuantize = 1, kPacked = 2 };

struct RowArgs {
  const uint16_t* x;     // kCopy, kQuantize: bf16 [M, K]
  const uint8_t* codes;  // kPacked
  const uint8_t* x_scales;
  const uint8_t* w;
  const uint8_t* w_scales;
  float alpha;
};

// Byte of 16-byte chunk c of row m of x: the eight lanes of a load's phase (two
// rows, four chunks 64 bytes apart) spread over all banks.
__device__ __forceinline__ int x_byte(int m, int c, int pitch) {
  return m * pitch + 16 * (c ^ ((c >> 3) & 1) ^ ((m & 1) << 1));
}

// 16 values of x (piece c of row m) as bf16x2 words.  Every lane calls (the
// quantizer's shuffles); pieces per row are even, so an mxfp4 group is two
// neighbouring lanes.
template <int F, int kFill>
__device__ __forceinline__ void fetch16(const RowArgs& a, int M, int K, bool live, int m, int c, uint32_t (&u)[8]) {
  const bool data = live && c * 16 < K;
#pragma unroll
  for (int e = 0; e < 8; ++e) u[e] = 0;
  if (kFill != kPacked && data) {
    const uint4* src = reinterpret_cast<const uint4*>(a.x + static_cast<int64_t>(m) * K + c * 16);
    const uint4 lo = __ldg(src), hi = __ldg(src + 1);
    u[0] = lo.x; u[1] = lo.y; u[2] = lo.z; u[3] = lo.w;
    u[4] = hi.x; u[5] = hi.y; u[6] = hi.z; u[7] = hi.w;
  }
  if (kFill == kCopy) return;
  uint2 code = make_uint2(0, 0);
  uint32_t byte = 0;
  if (kFill == kQuantize) {
    uint32_t am = amax16(u);
    GroupScale gs;
    if (F == kMx) {
      am = max(am, __shfl_xor_sync(0xffffffffu, am, 1));
      gs = mx_group(am);
    } else {
      gs = nv_group(__uint_as_float(am << 16), am < 0x7F80u, 1.f);
    }
    code = encode16<F, false>(u, gs, 1.f);
    byte = gs.byte;
  } else if (data) {
    code = __ldg(reinterpret_cast<const uint2*>(a.codes + m * static_cast<int64_t>(K / 2) + c * 8));
    byte = __ldg(a.x_scales + atom_offset<F>(m, c * 16 / Traits<F>::kGroup, (M + 127) / 128));
  }
  if (!data) return;
  uint32_t lo[4], hi[4];
  const uint32_t s2 = scale_bf16x2<F>(byte);
  decode_word(code.x, s2, lo);
  decode_word(code.y, s2, hi);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    u[e] = lo[e];
    u[4 + e] = hi[e];
  }
}

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// kNT: groups of 8 tokens
template <int F, int kFill, int kNT>
__global__ void __launch_bounds__(kRowThreads, 1) rows_kernel(const RowArgs a, const gemm::Params p) {
  constexpr int kGroup = Traits<F>::kGroup;
  constexpr int kT = row_tiles(kNT);
  constexpr int kTok = 8 * kNT;
  extern __shared__ __align__(16) uint8_t smem_rows[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int K = p.K, M = p.M, N = p.N;
  const int blocks = (K + kBlockK - 1) / kBlockK;
  const int pitch = blocks * (kBlockK * 2);  // bytes of a row of x
  float* red = reinterpret_cast<float*>(smem_rows);  // [warp][tile][token][16 features]
  uint8_t* xs = smem_rows + kRowWarps * kT * kTok * 16 * 4;
  const int n_tiles = (N + 15) / 16;
  const int64_t row_bytes = K / 2, row_scales = K / kGroup;
  const int stride = static_cast<int>(gridDim.x), tile0 = static_cast<int>(blockIdx.x);

  uint4 w[kT][2];
  uint32_t s[kT][2];
  const uint32_t w_row = static_cast<uint32_t>(g * row_bytes), s_row = static_cast<uint32_t>(g * row_scales);
  // this thread's 32 K of block blk, rows g and g + 8 of a tile; past K zeros.  N is a multiple of 8: a tile without
  // its second half reads the first twice
  auto load = [&](int tile, int blk, uint4 (&wr)[2], uint32_t (&sr)[2]) {
    const int k = blk * kBlockK + 32 * t;
    const bool in = k < K;
    const uint32_t wo = w_row + (in ? k >> 1 : 0), so = s_row + (in ? k / kGroup : 0);
    const uint8_t* q = a.w + tile * (16 * row_bytes);
    const uint8_t* r = a.w_scales + tile * (16 * row_scales);
    const bool second = tile * 16 + 8 < N;
    const uint8_t* q2 = second ? q + 8 * row_bytes : q;
    const uint8_t* r2 = second ? r + 8 * row_scales : r;
    wr[0] = __ldcs(reinterpret_cast<const uint4*>(q + wo));
    wr[1] = __ldcs(reinterpret_cast<const uint4*>(q2 + wo));
    if (F == kNv) {  // two scales of 32 K
      sr[0] = __ldg(reinterpret_cast<const uint16_t*>(r + so));
      sr[1] = __ldg(reinterpret_cast<const uint16_t*>(r2 + so));
    } else {
      sr[0] = __ldg(r + so);
      sr[1] = __ldg(r2 + so);
    }
    if (!in) sr[0] = sr[1] = 0;
  };
  if (warp < blocks) {
#pragma unroll
    for (int i = 0; i < kT; ++i)
      if (tile0 + i * stride < n_tiles) load(tile0 + i * stride, warp, w[i], s[i]);
  }

  // x into shared memory, in 16-byte chunks of 8 values in split order; past K zeros
  {
    const int pieces = pitch / 32, total = M * pieces;  // of 16 values
#pragma unroll 1
    for (int i0 = 0; i0 < total; i0 += kRowThreads) {
      const int i = i0 + static_cast<int>(threadIdx.x);
      const bool live = i < total;
      const int m = live ? i / pieces : 0, c = live ? i - m * pieces : 0;
      uint32_t u[8];
      fetch16<F, kFill>(a, M, K, live, m, c, u);
      if (!live) continue;
      *reinterpret_cast<uint4*>(xs + x_byte(m, 2 * c, pitch)) = split_order(u[0], u[1], u[2], u[3]);
      *reinterpret_cast<uint4*>(xs + x_byte(m, 2 * c + 1, pitch)) = split_order(u[4], u[5], u[6], u[7]);
    }
  }
  __syncthreads();

  // this lane's row of x for each 8 tokens; lanes past the last row repeat it, their columns are not used
  const uint8_t* xrow[kNT];
  int xswz[kNT];
#pragma unroll
  for (int q = 0; q < kNT; ++q) {
    const int m = min(8 * q + g, M - 1);
    xrow[q] = xs + m * pitch + 64 * t;
    xswz[q] = (t >> 1) | ((m & 1) << 1);  // x_byte's exclusive-or for a lane's four chunks
  }

  for (int first = tile0; first < n_tiles; first += kT * stride) {
    float acc[kT][kNT][4];
#pragma unroll
    for (int i = 0; i < kT; ++i)
#pragma unroll
      for (int q = 0; q < kNT; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][q][e] = 0.f;
    for (int blk = warp; blk < blocks; blk += kRowWarps) {
      const bool last = blk + kRowWarps >= blocks;
      const int next_blk = last ? warp : blk + kRowWarps;
      uint4 xv[kNT][4];
#pragma unroll
      for (int q = 0; q < kNT; ++q)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          xv[q][j] = *reinterpret_cast<const uint4*>(xrow[q] + blk * (kBlockK * 2) + 16 * (j ^ xswz[q]));
#pragma unroll
      for (int i = 0; i < kT; ++i) {
        const int tile = first + i * stride;
        if (tile >= n_tiles) break;  // uniform
        uint32_t mul[2][2];  // [row half][first / second 16 of the 32 K]
        bool f0, f1;
        decode_mul2<F>(s[i][0], mul[0], f0);
        decode_mul2<F>(s[i][1], mul[1], f1);
        const bool fast = F == kNv || __all_sync(0xffffffffu, f0 && f1);
        const uint32_t v[2][4] = {{w[i][0].x, w[i][0].y, w[i][0].z, w[i][0].w},
                                  {w[i][1].x, w[i][1].y, w[i][1].z, w[i][1].w}};
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // word j: K 8j..8j+7 of this thread's 32, two MMAs of 4 per thread
          uint32_t wa[4], wb[4];
          decode_word1_split(v[0][j], fast ? mul[0][j >> 1] : 0x7E807E80u, wa);
          decode_word1_split(v[1][j], fast ? mul[1][j >> 1] : 0x7E807E80u, wb);
          if (F == kMx && !fast) {  // a scale above 2: 2^126 and the scale apart
            const uint32_t sa = scale_bf16x2<F>(s[i][0]), sb = scale_bf16x2<F>(s[i][1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              wa[e] = fma_bf16x2(wa[e], sa, 0x80008000u);
              wb[e] = fma_bf16x2(wb[e], sb, 0x80008000u);
            }
          }
#pragma unroll
          for (int q = 0; q < kNT; ++q) {
            mma_16816(acc[i][q], wa[0], wb[0], wa[1], wb[1], xv[q][j].x, xv[q][j].y);
            mma_16816(acc[i][q], wa[2], wb[2], wa[3], wb[3], xv[q][j].z, xv[q][j].w);
          }
        }
        // the next block of this tile, or the first one of the tile that follows it
        const int next = last ? tile + kT * stride : tile;
        if (next < n_tiles) load(next, next_blk, w[i], s[i]);
      }
    }
    // partial sums (zeros where a warp has no block): features g, g + 8 of tokens 2t, 2t + 1
#pragma unroll
    for (int i = 0; i < kT; ++i) {
#pragma unroll
      for (int q = 0; q < kNT; ++q) {
        float* d = red + ((warp * kT + i) * kTok + 8 * q + 2 * t) * 16 + g;
        d[0] = acc[i][q][0];
        d[16] = acc[i][q][1];
        d[8] = acc[i][q][2];
        d[24] = acc[i][q][3];
      }
    }
    __syncthreads();
    // 8 features of one token per thread
#pragma unroll 1
    for (int i = threadIdx.x; i < kT * M * 2; i += kRowThreads) {
      const int tl = i / (2 * M), r = i - tl * 2 * M, m = r >> 1;
      const int nf = (first + tl * stride) * 16 + (r & 1) * 8;
      if (nf >= N) continue;
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int wi = 0; wi < kRowWarps; ++wi) {
        const float4* q = reinterpret_cast<const float4*>(red + ((wi * kT + tl) * kTok + m) * 16 + (r & 1) * 8);
        const float4 q0 = q[0], q1 = q[1];
        v[0] += q0.x; v[1] += q0.y; v[2] += q0.z; v[3] += q0.w;
        v[4] += q1.x; v[5] += q1.y; v[6] += q1.z; v[7] += q1.w;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = rbf16(__fmul_rn(v[k], a.alpha));  // the first rounding point, bf16(x W^T)
      gemm::Epi8 epi;
      epi.init(p, nf);
      epi.store(p, v, m, nf, nullptr);
    }
    __syncthreads();
  }
}

// Shared memory for M rows of x.
static size_t rows_smem(int64_t M, int64_t K) {
  const int nt = M <= 8 ? 1 : 2;
  return static_cast<size_t>(M * ((K + kBlockK - 1) / kBlockK) * (kBlockK * 2) +
                             kRowWarps * row_tiles(nt) * nt * 8 * 16 * 4);
}
constexpr size_t kRowSmem = 227 * 1024;

template <int F, int kFill, int kNT>
static ltxq_status launch_rows(const RowArgs& a, const gemm::Params& p, cudaStream_t stream) {
  auto kern = rows_kernel<F, kFill, kNT>;
  static SmemAttr attr_done;
  if (ltxq_status st = attr_done.set(reinterpret_cast<const void*>(kern), kRowSmem)) return st;
  const int tiles = (p.N + 15) / 16, sms = num_sms();
  kern<<<tiles < sms ? tiles : sms, kRowThreads, rows_smem(p.M, p.K), stream>>>(a, p);
  return launch_check("fp4 rows launch");
}

template <int F, int kFill>
static ltxq_status launch_rows_n(const RowArgs& a, const gemm::Params& p, cudaStream_t stream) {
  return p.M <= 8 ? launch_rows<F, kFill, 1>(a, p, stream) : launch_rows<F, kFill, 2>(a, p, stream);
}

template <int F>
static ltxq_status launch_rows_f(int fill, const RowArgs& a, const gemm::Params& p, cudaStream_t stream) {
  return fill == kPacked     ? launch_rows_n<F, kPacked>(a, p, stream)
         : fill == kQuantize ? launch_rows_n<F, kQuantize>(a, p, stream)
                             : launch_rows_n<F, kCopy>(a, p, stream);
}

}  // namespace fp4

// Whether the few-row kernel runs M rows over `w`: up to 16, as long as x fits (16 x 6000, 8 x 12000, 4 x 24000).
bool fp4_rows_supported(int64_t M, const ltxq_qweight& w) {
  if (w.mode != LTXQ_MXFP4 && w.mode != LTXQ_NVFP4) return false;
  if (M <= 0 || M > fp4::kMaxRows || (reinterpret_cast<uintptr_t>(w.scales) & 1u)) return false;
  return fp4::rows_smem(M, w.k_in) <= fp4::kRowSmem;
}

// x: bf16 rows, quantized first where `quantize`; or NULL with `packed`, an
// FP4Tensor of the weight's format whose global scale the caller put into
// p.alpha.  p as qlinear_params filled it, checked.
ltxq_status launch_fp4_rows(const void* x, bool quantize, const ltxq_fp4_act* packed, const ltxq_qweight& w,
                            const gemm::Params& p, cudaStream_t stream) {
  fp4::RowArgs a{};
  const int fill = packed ? fp4::kPacked : quantize ? fp4::kQuantize : fp4::kCopy;
  a.x = static_cast<const uint16_t*>(x);
  if (packed) {
    a.codes = static_cast<const uint8_t*>(packed->codes);
    a.x_scales = static_cast<const uint8_t*>(packed->scales);
  }
  a.w = static_cast<const uint8_t*>(w.weight);
  a.w_scales = static_cast<const uint8_t*>(w.scales);
  a.alpha = w.mode == LTXQ_NVFP4 ? p.alpha / fp4::kDecodeScale<fp4::kNv> : p.alpha;
  return w.mode == LTXQ_NVFP4 ? fp4::launch_rows_f<fp4::kNv>(fill, a, p, stream)
                              : fp4::launch_rows_f<fp4::kMx>(fill, a, p, stream);
}

}  // namespace ltxq
