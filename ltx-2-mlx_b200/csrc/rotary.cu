// rotary.cu -- rotary position embedding from positions and frequencies.
//
// Pair i of a head is rotated by the angle a = position * frequency[i]:
//   (u, v) -> scale * (u cos a - v sin a,  v cos a + u sin a)
// with (u, v) = (x[i], x[i + R/2]) in the half layout and (x[2i], x[2i + 1])
// in the interleaved one, i < R/2; elements past R pass through.  The inverse
// rotates by -a with the same scale, which is the gradient of the forward
// map (the map is linear and its matrix's transpose is the inverse rotation).
//
// The reference keeps cos / sin tables (model/transformer/rope.py:53-90 split,
// and its interleaved form); here the angle is formed in the kernel, so a
// call reads x, one position per token and axis, and the frequencies.  The
// product and its reduction to [-1/8, 1/8] of a turn are done in fp64, so that
// positions in the millions keep the fp32 angle's last bit; cos and sin are
// their Taylor series on that interval.
//
// Memory-bound: 2 reads/writes of x.  A thread keeps V neighbouring pairs of
// one head (two 16-byte loads) and walks tokens, so its frequencies stay in
// registers.  Where all heads share the frequencies the angles of a CTA's
// tokens are computed once into shared memory; with a row of frequencies per
// head every pair has its own angle and each thread computes its own.
#include "common.cuh"

namespace ltxq {
namespace rotary {

constexpr int kThreads = 256;
constexpr int kTableMax = 2048;  // (cos, sin) pairs of one CTA's tokens, 16 KB

struct Args {
  const void* x;
  void* out;
  int64_t xs[3], os[3];  // strides of batch, token, head (elements)
  const void* pos;
  int64_t ps[3];  // strides of batch, axis, token (elements)
  const double* freqs;
  const int32_t* axis;
  int64_t rows;  // batch * tokens
  int tokens, heads, d, half;
  int n_axes, pos_type, per_head;
  int units;      // per row: heads * (rotated units + copied units)
  int rot_units;  // per head
  int all_units;  // per head
  int rows_per_cta;
  float scale;
  int inverse;
};

__device__ __forceinline__ double load_pos(const Args& a, int64_t b, int64_t t, int axis) {
  const int64_t i = b * a.ps[0] + axis * a.ps[1] + t * a.ps[2];
  switch (a.pos_type) {
    case LTXQ_POS_I32: return static_cast<double>(__ldg(static_cast<const int32_t*>(a.pos) + i));
    case LTXQ_POS_I64: return static_cast<double>(__ldg(static_cast<const long long*>(a.pos) + i));
    case LTXQ_POS_F32: return static_cast<double>(__ldg(static_cast<const float*>(a.pos) + i));
    default: return __ldg(static_cast<const double*>(a.pos) + i);
  }
}

// cos and sin of 2 pi t.  t = q / 4 + r with an integer q and |r| <= 1/8: the
// reduction is exact in fp64, r then fits fp32 to 2^-28 of a turn.
__device__ __forceinline__ void cos_sin_turns(double t, float& c, float& s) {
  if (!(fabs(t) < 1e15)) t = t - rint(t);  // keeps 4t inside the adding trick's range; NaN and infinity give NaN
  constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
  const double m = __dadd_rn(4.0 * t, kRound);
  const int q = __double2loint(m);
  const float z = static_cast<float>(__fma_rn(__dsub_rn(m, kRound), -0.25, t)) * 6.283185307179586f;
  const float z2 = z * z;
  // |z| <= pi/4: the first terms left out are below 2e-9 (sin) and 2e-10 (cos)
  float sn = fmaf(z2, 2.7557319224e-6f, -1.9841269841e-4f);
  sn = fmaf(z2, sn, 8.3333333333e-3f);
  sn = fmaf(z2, sn, -1.6666666667e-1f);
  sn = fmaf(z * z2, sn, z);
  float cs = fmaf(z2, -2.7557319224e-7f, 2.4801587302e-5f);
  cs = fmaf(z2, cs, -1.3888888889e-3f);
  cs = fmaf(z2, cs, 4.1666666667e-2f);
  cs = fmaf(z2, cs, -0.5f);
  cs = fmaf(z2, cs, 1.0f);
  const bool swap = q & 1;
  c = swap ? sn : cs;
  s = swap ? cs : sn;
  if ((q + 1) & 2) c = -c;  // quadrants 1, 2
  if (q & 2) s = -s;        // quadrants 2, 3
}

constexpr double kInvTwoPi = 0.15915494309189535;

__device__ __forceinline__ float2 angle(const Args& a, double turns) {
  float c, s;
  cos_sin_turns(turns, c, s);
  return make_float2(c * a.scale, (a.inverse ? -s : s) * a.scale);
}

template <typename T, int V>
struct Vec {
  float v[V];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(T) * V == 16) {
      const uint4 w = *reinterpret_cast<const uint4*>(p);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2) {
          v[2 * i] = lo_bf16(u[i]);
          v[2 * i + 1] = hi_bf16(u[i]);
        } else {
          v[i] = __uint_as_float(u[i]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = sizeof(T) == 2 ? bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[i])
                                                        : reinterpret_cast<const float*>(p)[i];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (sizeof(T) * V == 16) {
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = sizeof(T) == 2 ? pack_bf16x2(v[2 * i % V], v[(2 * i + 1) % V]) : __float_as_uint(v[i]);
      *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if constexpr (sizeof(T) == 2) reinterpret_cast<uint16_t*>(p)[i] = f32_to_bf16(v[i]);
        else reinterpret_cast<float*>(p)[i] = v[i];
      }
    }
  }
};

// T: uint16_t (bf16) or float.  V pairs per unit: 16 bytes of each of the two
// vectors, or 1 where alignment or sizes leave no wider form.
template <typename T, int V, bool kHalf, bool kPerHead>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const Args a) {
  __shared__ float2 table[kPerHead ? 1 : kTableMax];
  const int64_t row0 = blockIdx.x * static_cast<int64_t>(a.rows_per_cta);
  const int n = static_cast<int>(min(static_cast<int64_t>(a.rows_per_cta), a.rows - row0));
  if (!kPerHead) {
    for (int i = threadIdx.x; i < n * a.half; i += kThreads) {
      const int r = i / a.half, k = i - r * a.half;
      const int64_t row = row0 + r;
      const int64_t b = row / a.tokens, t = row - b * a.tokens;
      const int ax = a.axis ? __ldg(a.axis + k) : 0;
      const double p = static_cast<unsigned>(ax) < static_cast<unsigned>(a.n_axes) ? load_pos(a, b, t, ax) : NAN;
      table[i] = angle(a, p * (__ldg(a.freqs + k) * kInvTwoPi));
    }
    __syncthreads();
  }
  const int u = blockIdx.y * kThreads + threadIdx.x;
  if (u >= a.units) return;
  const int h = u / a.all_units, c = u - h * a.all_units;
  const bool rot = c < a.rot_units;
  // first element of the unit's two vectors within the head
  const int e0 = !rot ? 2 * a.half + (c - a.rot_units) * 2 * V : kHalf ? c * V : c * 2 * V;
  const int e1 = rot && kHalf ? e0 + a.half : e0 + V;
  const bool second = rot || e1 < a.d;  // an odd head: the last copied unit is one element
  double f[kPerHead ? V : 1];
  int ax[kPerHead ? V : 1];
  if (kPerHead && rot) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      f[i] = __ldg(a.freqs + h * a.half + c * V + i) * kInvTwoPi;
      ax[i] = a.axis ? __ldg(a.axis + h * a.half + c * V + i) : 0;
      if (static_cast<unsigned>(ax[i]) >= static_cast<unsigned>(a.n_axes)) {
        f[i] = NAN;
        ax[i] = 0;
      }
    }
  }
  const T* x = static_cast<const T*>(a.x) + h * a.xs[2];
  T* out = static_cast<T*>(a.out) + h * a.os[2];
  for (int r = 0; r < n; ++r) {
    const int64_t row = row0 + r;
    const int64_t b = row / a.tokens, t = row - b * a.tokens;
    const T* xr = x + b * a.xs[0] + t * a.xs[1];
    T* orow = out + b * a.os[0] + t * a.os[1];
    Vec<T, V> p, q;
    p.load(xr + e0);
    if (second) q.load(xr + e1);
    if (rot) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float2 cs;
        if (kPerHead) cs = angle(a, load_pos(a, b, t, ax[kPerHead ? i : 0]) * f[kPerHead ? i : 0]);
        else cs = table[r * a.half + c * V + i];
        // interleaved: pair i is elements 2i, 2i + 1 of the unit's 2V
        float& m = kHalf ? p.v[i] : (2 * i < V ? p.v[2 * i % V] : q.v[2 * i % V]);
        float& o = kHalf ? q.v[i] : (2 * i + 1 < V ? p.v[(2 * i + 1) % V] : q.v[(2 * i + 1) % V]);
        const float mu = m, mv = o;
        m = fmaf(mu, cs.x, -(mv * cs.y));
        o = fmaf(mv, cs.x, mu * cs.y);
      }
    }
    p.store(orow + e0);
    if (second) q.store(orow + e1);
  }
}

template <typename T, int V>
static void launch(const Args& a, bool half_layout, dim3 grid, cudaStream_t s) {
  if (half_layout) {
    if (a.per_head) rotary_kernel<T, V, true, true><<<grid, kThreads, 0, s>>>(a);
    else rotary_kernel<T, V, true, false><<<grid, kThreads, 0, s>>>(a);
  } else {
    if (a.per_head) rotary_kernel<T, V, false, true><<<grid, kThreads, 0, s>>>(a);
    else rotary_kernel<T, V, false, false><<<grid, kThreads, 0, s>>>(a);
  }
}

}  // namespace rotary
}  // namespace ltxq

extern "C" ltxq_status ltxq_rotary(const ltxq_rotary_args* r, void* stream) {
  using namespace ltxq;
  using namespace ltxq::rotary;
  if (!r) return fail(LTXQ_ERR_INVALID, "rotary: NULL argument");
  if (r->batch < 0 || r->tokens < 0 || r->heads <= 0 || r->head_dim <= 0 || r->rotary_dim < 0)
    return fail(LTXQ_ERR_INVALID, "rotary: bad shape");
  if (r->rotary_dim % 2 != 0 || r->rotary_dim > r->head_dim)
    return fail(LTXQ_ERR_INVALID, "rotary: rotary_dim must be even and at most head_dim");
  if (r->layout != LTXQ_ROTARY_HALF && r->layout != LTXQ_ROTARY_INTERLEAVED)
    return fail(LTXQ_ERR_INVALID, "rotary: unknown layout");
  if (r->dtype != LTXQ_BF16 && r->dtype != LTXQ_F32) return fail(LTXQ_ERR_UNSUPPORTED, "rotary: dtype must be bf16 or f32");
  if (r->pos_dtype < LTXQ_POS_I32 || r->pos_dtype > LTXQ_POS_F64)
    return fail(LTXQ_ERR_INVALID, "rotary: unknown position type");
  if (r->n_axes < 1 || (r->n_axes > 1 && !r->axis && r->rotary_dim > 0))
    return fail(LTXQ_ERR_INVALID, "rotary: several position axes need the axis of each frequency");
  if (!(r->scale == r->scale) || r->scale > 3e38f || r->scale < -3e38f)
    return fail(LTXQ_ERR_INVALID, "rotary: scale must be finite");
  if (r->batch == 0 || r->tokens == 0) return LTXQ_OK;
  if (!r->x || !r->out || (r->rotary_dim > 0 && (!r->positions || !r->freqs)))
    return fail(LTXQ_ERR_INVALID, "rotary: NULL pointer");
  if (r->rotary_dim > 2 * kTableMax) return fail(LTXQ_ERR_UNSUPPORTED, "rotary: rotary_dim must be at most 4096");
  if (r->heads > 0x7FFFFFFF / r->head_dim || r->tokens > 0x7FFFFFFF)
    return fail(LTXQ_ERR_UNSUPPORTED, "rotary: dimension too large");
  const int es = r->dtype == LTXQ_BF16 ? 2 : 4;
  if ((reinterpret_cast<uintptr_t>(r->x) | reinterpret_cast<uintptr_t>(r->out)) % es != 0)
    return fail(LTXQ_ERR_UNSUPPORTED, "rotary: x / out not aligned to their elements");

  Args a{};
  a.x = r->x;
  a.out = r->out;
  const int64_t half = r->rotary_dim / 2;
  const int wide = 16 / es;
  // 16-byte vectors: both vectors of every unit start on 16 bytes
  bool vec = half % wide == 0 && r->head_dim % (2 * wide) == 0 &&
             ((reinterpret_cast<uintptr_t>(r->x) | reinterpret_cast<uintptr_t>(r->out)) & 15u) == 0;
  for (int i = 0; i < 3; ++i) {
    a.xs[i] = r->x_stride[i];
    a.os[i] = r->out_stride[i];
    a.ps[i] = r->pos_stride[i];
    vec = vec && a.xs[i] % wide == 0 && a.os[i] % wide == 0;
  }
  const int V = vec ? wide : 1;
  a.pos = r->positions;
  a.freqs = r->freqs;
  a.axis = r->axis;
  a.rows = r->batch * r->tokens;
  a.tokens = static_cast<int>(r->tokens);
  a.heads = static_cast<int>(r->heads);
  a.d = static_cast<int>(r->head_dim);
  a.half = static_cast<int>(half);
  a.n_axes = r->n_axes;
  a.pos_type = r->pos_dtype;
  a.per_head = r->freqs_per_head ? 1 : 0;
  a.rot_units = a.half / V;
  a.all_units = a.rot_units + (a.d - 2 * a.half + 2 * V - 1) / (2 * V);
  a.units = a.heads * a.all_units;
  a.scale = r->scale;
  a.inverse = r->inverse ? 1 : 0;
  // rows per CTA: as many as leave every SM several CTAs, within the shared table
  const int64_t gy = (a.units + kThreads - 1) / kThreads;
  int64_t per = a.rows * gy / (static_cast<int64_t>(num_sms()) * 8);
  if (!a.per_head && a.half > 0 && per > kTableMax / a.half) per = kTableMax / a.half;
  per = per < 1 ? 1 : (per > 16 ? 16 : per);
  const int64_t gx = (a.rows + per - 1) / per;
  if (gy > 65535 || gx > 0x7FFFFFFF) return fail(LTXQ_ERR_UNSUPPORTED, "rotary: dimension too large");
  a.rows_per_cta = static_cast<int>(per);
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool hl = r->layout == LTXQ_ROTARY_HALF;
  if (es == 2) {
    if (vec) launch<uint16_t, 8>(a, hl, grid, s);
    else launch<uint16_t, 1>(a, hl, grid, s);
  } else {
    if (vec) launch<float, 4>(a, hl, grid, s);
    else launch<float, 1>(a, hl, grid, s);
  }
  return launch_check("rotary launch");
}
