// gemm_epilogue.cuh -- pieces shared by the quantized GEMM kernels (qgemm.cu
// for the dequantizing path, mx.cu for the native block-scaled fp8 path):
// the launch parameters, the reference's GELU with its per-op bf16 rounding
// (exact table form), named barriers, the epilogue's row store with the gated
// residual fused, and the epilogue of 8 features of one token.
#pragma once

#include "common.cuh"

namespace ltxq {
namespace gemm {

struct Params {
  int M, N, K, gs;
  int vec_groups;  // group parameters of a row are 16-byte aligned blocks (see GroupCursor)
  const void* scales;
  const uint16_t* biases;
  const uint16_t* bias;
  int epi;
  VecArg gate;
  const uint16_t* residual;
  uint16_t* out;
  unsigned int* err;
  // pair-kernel schedule: output tiles [0, dp_tiles) are computed whole; each
  // later tile is split into `splits` K ranges whose fp32 partials go to
  // `partial` ([tile - dp_tiles][split][256 tokens][256 features], tile-local)
  // and are summed by splitk_reduce_kernel
  int dp_tiles;
  int splits;
  float* partial;
  float alpha;  // nvfp4: the tensor scale that multiplies the accumulator (1 elsewhere)
};

// output tiles of a pair kernel, how many stay whole, K splits of the rest
struct Sched {
  int tiles, dp, splits;
};
Sched plan_schedule(int64_t M, int64_t N, int64_t K);
size_t splitk_bytes(int64_t M, int64_t N, int64_t K);
ltxq_status launch_splitk_reduce(const Params& p, cudaStream_t stream);

// gelu_approx with the reference's per-op bf16 rounding (feed_forward.py:8-14;
// MLX evaluates each op of the expression on bf16 arrays, the constants
// 0.044715 and sqrt(2/pi) taking the bf16 values below).
__device__ __forceinline__ float gelu_ref(float x) {
  constexpr float c1 = 0.044677734375f;  // bf16(0.044715)
  constexpr float c2 = 0.796875f;        // bf16(sqrt(2/pi))
  const float x3 = rbf16(__fmul_rn(__fmul_rn(x, x), x));  // exact in fp32 for bf16 x
  float t = rbf16(__fmul_rn(c1, x3));
  t = rbf16(__fadd_rn(x, t));
  t = rbf16(__fmul_rn(c2, t));
  t = rbf16(tanhf(t));
  t = rbf16(__fadd_rn(1.0f, t));
  const float h = rbf16(__fmul_rn(0.5f, x));
  return rbf16(__fmul_rn(h, t));
}

// gelu_ref through a table.  Over all 65536 bf16 inputs gelu_ref(x) equals
// bf16(0.5 x) for |x| < 2^-9 (its 1 + tanh term rounds to 1), x for x >= 4
// (tanh rounds to 1), -0 for finite x <= -4 (1 + tanh rounds to 0) and NaN
// for -inf / NaN.  Between, the result is read from a table of gelu_ref
// values built by the kernel itself, so both forms give the same bits.
// Magnitudes [kGeluLo, kGeluLo + kGeluN) are tabulated, positive then negative.
constexpr uint32_t kGeluLo = 0x3B00u;  // 2^-9
constexpr uint32_t kGeluN = 0x4080u - kGeluLo;  // up to 4.0 (exclusive)
constexpr int kGeluTabBytes = static_cast<int>(2 * kGeluN * 2);

// b: bf16 bits (low 16), small: bf16 bits of bf16(0.5 b); returns the bf16
// bits of gelu_ref(b)
__device__ __forceinline__ uint32_t gelu_tab_sel(uint32_t b, uint32_t small, const uint16_t* tab) {
  const uint32_t mag = b & 0x7FFFu, neg = b >> 15;
  const uint32_t t = mag - kGeluLo;  // wraps for mag < kGeluLo
  const bool in_tab = t < kGeluN;
  const uint32_t tv = tab[in_tab ? t + neg * kGeluN : 0u];
  const uint32_t big = neg ? (mag >= 0x7F80u ? 0x7FC0u : 0x8000u) : b;
  return in_tab ? tv : (mag < kGeluLo ? small : big);
}

// gelu_ref on both halves of a bf16x2 word (one paired conversion for the
// small-input form)
__device__ __forceinline__ uint32_t gelu_tab_x2(uint32_t b2, const uint16_t* tab) {
  const uint32_t small2 = pack_bf16x2(__fmul_rn(0.5f, __uint_as_float(b2 << 16)),
                                      __fmul_rn(0.5f, __uint_as_float(b2 & 0xFFFF0000u)));
  return gelu_tab_sel(b2 & 0xFFFFu, small2 & 0xFFFFu, tab) | (gelu_tab_sel(b2 >> 16, small2 >> 16, tab) << 16);
}

// fills the table (n_threads threads, thread id tid); caller synchronizes
__device__ __forceinline__ void gelu_tab_fill(uint16_t* tab, int tid, int n_threads) {
  for (int i = tid; i < static_cast<int>(2 * kGeluN); i += n_threads) {
    const uint32_t neg = static_cast<uint32_t>(i) >= kGeluN;
    const uint32_t mag = kGeluLo + static_cast<uint32_t>(i) - (neg ? kGeluN : 0u);
    tab[i] = f32_to_bf16(gelu_ref(__uint_as_float(((neg << 15) | mag) << 16)));
  }
}

__device__ __forceinline__ void named_bar_sync(int id, int n) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory");
}

// Row side of the smem-A epilogue: u = bf16x2 words of 8 consecutive
// features (bias / GELU already applied); gated residual, then a 16-byte store.
__device__ __forceinline__ void epi_row_store(const Params& p, uint32_t (&u)[4], int m, int nf, const float (&g8b)[8],
                                              bool gated, bool two_round, bool gate_bcast) {
  const int64_t off = static_cast<int64_t>(m) * p.N + nf;
  if (gated) {
    const uint4 rv = __ldg(reinterpret_cast<const uint4*>(p.residual + off));
    const uint32_t rw[4] = {rv.x, rv.y, rv.z, rv.w};
    float g8[8];
    if (gate_bcast) {
#pragma unroll
      for (int k = 0; k < 8; ++k) g8[k] = g8b[k];
    } else {
      load_vec8(p.gate, vec_row(p.gate, m), nf, g8);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float p0 = __fmul_rn(lo_bf16(u[k]), g8[2 * k]);
      const float p1 = __fmul_rn(hi_bf16(u[k]), g8[2 * k + 1]);
      const float r0 = lo_bf16(rw[k]), r1 = hi_bf16(rw[k]);
      if (two_round) {
        const uint32_t pr = pack_bf16x2(p0, p1);
        u[k] = pack_bf16x2(__fadd_rn(r0, lo_bf16(pr)), __fadd_rn(r1, hi_bf16(pr)));
      } else {
        u[k] = pack_bf16x2(__fadd_rn(p0, r0), __fadd_rn(p1, r1));
      }
    }
  }
  *reinterpret_cast<uint4*>(p.out + off) = make_uint4(u[0], u[1], u[2], u[3]);
}

// Rows and pieces of a lane quad: lane j holds piece k of row j in u[k], and
// then piece j of row i in u[i].
__device__ __forceinline__ void quad_transpose(uint32_t (&u)[4][4]) {
  const int j = threadIdx.x & 3;
#pragma unroll
  for (int step = 1; step <= 2; ++step) {
    const bool up = j & step;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int lo = step == 1 ? 2 * k : k, hi = lo + step;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t r = __shfl_xor_sync(0xffffffffu, up ? u[lo][w] : u[hi][w], step);
        if (up) u[lo][w] = r;
        else u[hi][w] = r;
      }
    }
  }
}

// 32 accumulators of a token times alpha, rounded to bf16 (the first rounding
// point), as four 16-byte pieces
__device__ __forceinline__ void epi_pack32(float alpha, const uint32_t (&v)[32], uint32_t (&u)[4][4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int w = 0; w < 4; ++w)
      u[k][w] = pack_bf16x2(__fmul_rn(__uint_as_float(v[8 * k + 2 * w]), alpha),
                            __fmul_rn(__uint_as_float(v[8 * k + 2 * w + 1]), alpha));
}

// Epilogue of 32 features [n0, n0 + 32) of a warp's 32 tokens [m0, m0 + 32),
// lane = token, u as epi_pack32 leaves it: lane quads exchange 16-byte pieces,
// so that each store writes 64 contiguous bytes of 8 rows (a store of one piece
// of 32 rows takes four times the cycles: 9216 x 4096 x 16384 fp4 products 356
// us with those, 313 without); bias, GELU and the gated residual on that side.
__device__ __forceinline__ void epi_rows32(const Params& p, uint32_t (&u)[4][4], int m0, int n0, bool gated,
                                           bool two_round, const uint16_t* gtab) {
  const int lane = threadIdx.x & 31;
  quad_transpose(u);
  const int nf = n0 + 8 * (lane & 3);
  if (nf >= p.N) return;
  if (p.bias != nullptr) {
    const uint4 bv = __ldg(reinterpret_cast<const uint4*>(p.bias + nf));
    const uint32_t bw[4] = {bv.x, bv.y, bv.z, bv.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w)
        u[i][w] = pack_bf16x2(__fadd_rn(lo_bf16(u[i][w]), lo_bf16(bw[w])), __fadd_rn(hi_bf16(u[i][w]), hi_bf16(bw[w])));
  }
  if (p.epi == LTXQ_EPI_GELU) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) u[i][w] = gelu_tab_x2(u[i][w], gtab);
  }
  const bool gate_bcast = p.gate.rows_per_vec == 0;
  float g8[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (gated && gate_bcast) load_vec8(p.gate, vec_row(p.gate, 0), nf, g8);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + (lane & ~3) + i;
    if (m < p.M) epi_row_store(p, u[i], m, nf, g8, gated, two_round, gate_bcast);
  }
}

// Epilogue state of one thread for a fixed chunk of 8 features [nf, nf + 8):
// the linear bias and a broadcast gate are loaded once.  store() takes the
// bf16-rounded accumulators of one token (the reference's first rounding
// point) and applies bias / GELU / gated residual with the reference's
// rounding points, then writes 16 bytes.
struct Epi8 {
  float bias8[8];
  float g8[8];
  bool gated, two_round, gate_bcast;
  __device__ __forceinline__ void init(const Params& p, int nf) {
    gated = p.epi == LTXQ_EPI_GATED_RESIDUAL || p.epi == LTXQ_EPI_GATE_THEN_ADD;
    two_round = p.epi == LTXQ_EPI_GATE_THEN_ADD || p.gate.dtype == LTXQ_BF16;
    gate_bcast = p.gate.rows_per_vec == 0;
    if (p.bias != nullptr) {
      const uint4 bv = __ldg(reinterpret_cast<const uint4*>(p.bias + nf));
      const uint32_t bw[4] = {bv.x, bv.y, bv.z, bv.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        bias8[2 * k] = lo_bf16(bw[k]);
        bias8[2 * k + 1] = hi_bf16(bw[k]);
      }
    }
    if (gated && gate_bcast) load_vec8(p.gate, vec_row(p.gate, 0), nf, g8);
  }
  // conversions to bf16 are paired (cvt.rn.bf16x2.f32), never one value at a time
  __device__ __forceinline__ void store(const Params& p, const float (&a)[8], int m, int nf, const uint16_t* gtab) {
    uint32_t u[4];
    if (p.bias != nullptr) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        u[k] = pack_bf16x2(__fadd_rn(a[2 * k], bias8[2 * k]), __fadd_rn(a[2 * k + 1], bias8[2 * k + 1]));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) u[k] = pack_bf16x2(a[2 * k], a[2 * k + 1]);  // exact: a is bf16-valued
    }
    if (p.epi == LTXQ_EPI_GELU) {
      if (gtab != nullptr) {
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = gelu_tab_x2(u[k], gtab);
      } else {  // no table: the same function evaluated directly
#pragma unroll
        for (int k = 0; k < 4; ++k)
          u[k] = pack_bf16x2(gelu_ref(lo_bf16(u[k])), gelu_ref(hi_bf16(u[k])));
      }
    }
    const int64_t off = static_cast<int64_t>(m) * p.N + nf;
    if (gated) {
      const uint4 rv = __ldg(reinterpret_cast<const uint4*>(p.residual + off));
      const uint32_t rw[4] = {rv.x, rv.y, rv.z, rv.w};
      if (!gate_bcast) load_vec8(p.gate, vec_row(p.gate, m), nf, g8);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float p0 = __fmul_rn(lo_bf16(u[k]), g8[2 * k]);
        const float p1 = __fmul_rn(hi_bf16(u[k]), g8[2 * k + 1]);
        const float r0 = lo_bf16(rw[k]), r1 = hi_bf16(rw[k]);
        if (two_round) {
          const uint32_t pr = pack_bf16x2(p0, p1);
          u[k] = pack_bf16x2(__fadd_rn(r0, lo_bf16(pr)), __fadd_rn(r1, hi_bf16(pr)));
        } else {
          u[k] = pack_bf16x2(__fadd_rn(p0, r0), __fadd_rn(p1, r1));
        }
      }
    }
    *reinterpret_cast<uint4*>(p.out + off) = make_uint4(u[0], u[1], u[2], u[3]);
  }
};

}  // namespace gemm

ltxq_status qlinear_params(const void* x, int64_t M, const ltxq_qweight& w, const ltxq_epilogue* epi, void* out,
                           gemm::Params* params);

}  // namespace ltxq
