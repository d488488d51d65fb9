// fp4.cuh -- 4-bit floating point in groups, shared by the quantizers, the
// standalone dequantizers and the GEMMs, so that every reader and writer of a
// format agrees bit for bit.
//
// Elements are E2M1 (sign, 2 exponent bits, 1 mantissa bit: 0, 0.5, 1, 1.5,
// 2, 3, 4, 6), two per byte, the lower index in the low nibble.
//   mxfp4: 32 elements share an E8M0 scale 2^(s-127)      (s = 255: NaN)
//   nvfp4: 16 elements share an E4M3 scale, times one fp32 scale of the whole
//          tensor (global_scale, 1 where the cache layout has none)
//
// Quantizing a group (y = x / global_scale, amax = max|y|):
//   mxfp4: scale 2^e with the largest e for which 4 * 2^e <= amax, at least
//          2^-127 -- the OCP MX rule floor(log2(amax)) - emax(E2M1) that the
//          mxfp8 quantizer follows too (values of [6, 8) * 2^e saturate at 6)
//   nvfp4: scale = RNE_E4M3(amax / 6), saturating at 448; a scale that rounds
//          to zero stores zeros
//   code = RNE_E2M1(y / scale), ties to the even code, saturating at 6.
// E2M1 has neither infinity nor NaN: a group that holds one gets its scale's
// NaN code, so that every value read back from it is NaN.
#pragma once

#include "common.cuh"
#include "dequant.cuh"

namespace ltxq {
namespace fp4 {

enum Fmt { kMx = 0, kNv = 1 };

template <int F>
struct Traits {
  static constexpr int kGroup = F == kNv ? 16 : 32;  // elements per scale
  static constexpr int kAtoms = F == kNv ? 4 : 2;    // scale atoms (128 rows x 4 groups) per 256-element K stage
};

constexpr int kAtom = 512;    // bytes of a scale atom
constexpr int kStageK = 256;  // elements of K per GEMM stage (128 bytes of codes)

// Scale layout of the block-scaled MMA: K stage j, row tile t (128 rows),
// atom a at ((j * row_tiles + t) * kAtoms + a) * 512; in it, the scale of row
// t*128 + 32*m1 + m0 and group 4a + b of the stage at byte m0*16 + m1*4 + b.
template <int F>
__host__ __device__ __forceinline__ int64_t atom_offset(int64_t row, int64_t group, int64_t row_tiles) {
  constexpr int kPerStage = kStageK / Traits<F>::kGroup;
  const int64_t j = group / kPerStage;
  const int gi = static_cast<int>(group - j * kPerStage);
  const int mi = static_cast<int>(row & 127);
  return ((j * row_tiles + (row >> 7)) * Traits<F>::kAtoms + (gi >> 2)) * kAtom + (mi & 31) * 16 + (mi >> 5) * 4 +
         (gi & 3);
}

// ---------------------------------------------------------------- decoding

// bf16 bits of an E8M0 scale
__device__ __forceinline__ uint32_t e8m0_bf16(uint32_t s) {
  return s == 0u ? 0x0040u : (s == 255u ? 0x7FC0u : s << 7);
}
// bf16 bits of an E4M3 value (exact: 4 significant bits)
__device__ __forceinline__ uint32_t e4m3_bf16(uint32_t s) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(s)));
  return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(h & 0xFFFFu)))) >> 16;
}
template <int F>
__device__ __forceinline__ uint32_t scale_bf16x2(uint32_t s) {
  return (F == kNv ? e4m3_bf16(s) : e8m0_bf16(s)) * 0x00010001u;
}

// A packed word holds elements k..k+7.  A nibble s|ee|m moved to bf16 bits 15
// and 8:6 is the bf16 encoding of its value times 2^-126 (ee = 0 becomes a bf16
// subnormal, as in E2M1), which one product with 2^126 times the scale makes
// the value.  E2M1 times either scale has at most 6 significant bits, so the
// product is exact wherever bf16's exponent range holds it.
//
// bf16x2 of (element 2j, element 2j + 1) * 2^-126 for j = 0..3; lo / hi: the
// word's even / odd elements, one in each byte's low nibble.  The byte
// selectors 8..F replicate a byte's top bit, here 0.
__device__ __forceinline__ void e2m1x8_m126(uint32_t w, uint32_t (&o)[4]) {
  const uint32_t lo = w & 0x0F0F0F0Fu, hi = (w >> 4) & 0x0F0F0F0Fu;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t t;
    const uint32_t sel = static_cast<uint32_t>(j) | (8u << 4) | (static_cast<uint32_t>(4 + j) << 8) | (8u << 12);
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(t) : "r"(lo), "r"(hi), "r"(sel));
    o[j] = (t * 0x1040u) & 0x81C081C0u;  // nibble << 12 and << 6: no carries, the halves do not meet
  }
}
// times the scale (bf16x2 broadcast), any scale: 2^126 first, as its product
// with a scale above 2 leaves bf16's range
__device__ __forceinline__ void decode_word(uint32_t w, uint32_t s2, uint32_t (&o)[4]) {
  e2m1x8_m126(w, o);
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = fma_bf16x2(fma_bf16x2(o[j], 0x7E807E80u, 0x80008000u), s2, 0x80008000u);
}

// The products' form, one multiplication per pair: the values times
// kDecodeScale, by a multiplier that holds 2^126 * scale * kDecodeScale.
//   nvfp4: 2^-8, which brings every E4M3 scale into range; the product is
//          multiplied back with its tensor scale
//   mxfp4: 1; scales above 2 (and the NaN code) do not fit and say so, and
//          take decode_word
template <int F>
constexpr float kDecodeScale = F == kNv ? 0x1p-8f : 1.f;

// the multipliers of two groups, whose scale bytes are s's low two (mxfp4: of
// one group, its byte in s, both the same)
template <int F>
__device__ __forceinline__ void decode_mul2(uint32_t s, uint32_t (&m)[2], bool& fits) {
  if (F == kNv) {
    fits = true;
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(s)));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    // E4M3 stays below 2^9: 2^118 times it is finite in fp32, and has 4 bits, all of them in the upper half
    const uint32_t a = __float_as_uint(__fmul_rn(f.x, 0x1p118f)), b = __float_as_uint(__fmul_rn(f.y, 0x1p118f));
    m[0] = __byte_perm(a, a, 0x3232);
    m[1] = __byte_perm(b, b, 0x3232);
  } else {
    fits = s <= 128u;
    m[0] = m[1] = (s + 126u) * 0x00800080u;  // 2^(s - 127 + 126)
  }
}
__device__ __forceinline__ void decode_word1(uint32_t w, uint32_t m2, uint32_t (&o)[4]) {
  e2m1x8_m126(w, o);
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = fma_bf16x2(o[j], m2, 0x80008000u);
}

// decode_word1 in the order (0, 4), (1, 5), (2, 6), (3, 7), for products whose
// other operand is laid out the same way: nibbles j and j + 4 are the two
// halves' as they lie, so only a mask and a multiplication place them.
__device__ __forceinline__ void decode_word1_split(uint32_t w, uint32_t m2, uint32_t (&o)[4]) {
  const uint32_t v = w >> 8;
  o[0] = ((w & 0x000F000Fu) * 0x1040u) & 0x81C081C0u;
  o[1] = ((w & 0x00F000F0u) * 0x0104u) & 0x81C081C0u;
  o[2] = ((v & 0x000F000Fu) * 0x1040u) & 0x81C081C0u;
  o[3] = ((v & 0x00F000F0u) * 0x0104u) & 0x81C081C0u;
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = fma_bf16x2(o[j], m2, 0x80008000u);
}
// eight bf16 values (bf16x2 words, in order) in that order
__device__ __forceinline__ uint4 split_order(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return make_uint4(__byte_perm(a, c, 0x5410), __byte_perm(a, c, 0x7632), __byte_perm(b, d, 0x5410),
                    __byte_perm(b, d, 0x7632));
}

// ---------------------------------------------------------------- encoding

// eight fp32 values -> eight E2M1 codes (RNE, saturating), value 0 in the low nibble
__device__ __forceinline__ uint32_t to_e2m1x8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// The largest magnitude among 16 bf16 values, as bf16 bits: an integer
// maximum of the magnitudes, which orders NaN above infinity above the rest.
__device__ __forceinline__ uint32_t amax16(const uint32_t (&u)[8]) {
  uint32_t m = u[0] & 0x7FFF7FFFu;
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max_u16x2(m, u[i] & 0x7FFF7FFFu);
  return max(m & 0xFFFFu, m >> 16);
}

// How a group is scaled: value * mul (snapped, see below) -> code.
struct GroupScale {
  uint32_t byte;
  float mul;
};

__device__ __forceinline__ GroupScale mx_group(uint32_t amax_bits) {
  const int ef = static_cast<int>(amax_bits >> 7);
  // amax in [2^(ef-127), 2^(ef-126)): e = ef - 129; zeros and values below 2^-125 take 2^-127
  const uint32_t byte = ef == 255 ? 255u : static_cast<uint32_t>(max(ef - 2, 0));
  return GroupScale{byte, __uint_as_float((254u - min(byte, 253u)) << 23)};  // 2^-(byte-127)
}

// inv_g: 1 / global_scale, a power of two
__device__ __forceinline__ GroupScale nv_group(float amax, bool finite, float inv_g) {
  uint16_t p;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(p) : "f"(0.f), "f"(__fdiv_rn(amax, 6.0f)));
  const uint32_t byte = finite ? (p & 0xFFu) : 0x7Fu;
  const float s = __uint_as_float(e4m3_bf16(byte) << 16);
  return GroupScale{byte, s > 0.f ? __fmul_rn(__frcp_rn(s), inv_g) : 0.f};
}

// y / s for a bf16 y and an E4M3 s from y * (1/s): the product is within
// 2^-23 of the quotient.  y is 8 bits and a midpoint of E2M1 times s 7 bits,
// so a quotient that is no midpoint is at least 2^-8 (relative) away from
// each: rounding the product to 16 bits moves it onto a midpoint where the
// quotient is one and across none where it is not.
__device__ __forceinline__ float snap16(float q) {
  return __uint_as_float((__float_as_uint(q) + 0x80u) & 0xFFFFFF00u);
}

// 16 values (bf16x2 words, in order) -> two code words.  kDiv: an nvfp4 global
// scale that is no power of two, both divisions in fp32.
template <int F, bool kDiv>
__device__ __forceinline__ uint2 encode16(const uint32_t (&u)[8], const GroupScale& gs, float g) {
  uint32_t c[2];
  const float s = kDiv ? __uint_as_float(e4m3_bf16(gs.byte) << 16) : 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = lo_bf16(u[4 * h + i]), b = hi_bf16(u[4 * h + i]);
      if (kDiv) {
        v[2 * i] = s > 0.f ? __fdiv_rn(__fdiv_rn(a, g), s) : 0.f;
        v[2 * i + 1] = s > 0.f ? __fdiv_rn(__fdiv_rn(b, g), s) : 0.f;
      } else if (F == kNv) {
        v[2 * i] = snap16(__fmul_rn(a, gs.mul));
        v[2 * i + 1] = snap16(__fmul_rn(b, gs.mul));
      } else {
        v[2 * i] = __fmul_rn(a, gs.mul);  // a power of two: exact
        v[2 * i + 1] = __fmul_rn(b, gs.mul);
      }
    }
    c[h] = to_e2m1x8(v);
  }
  return make_uint2(c[0], c[1]);
}

}  // namespace fp4
}  // namespace ltxq
