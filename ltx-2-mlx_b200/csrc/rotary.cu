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
// call reads x, one position per token and axis, and the frequencies.  Turns
// position * frequency / (2 pi) are formed from two fp32 parts of each (48 bits,
// the product's rounding kept by an fma) and reduced to [-1/8, 1/8] exactly: the
// error is turns * 2^-47, below the fp32 angle's last bit up to 2^20 turns (6.6
// million radians); beyond, the product is taken in fp64.  cos and sin are their
// Taylor series on the interval, or for bf16 the hardware's functions.
//
// Memory-bound where the heads share the frequencies: the angles of a CTA's
// rows are computed once into shared memory, and its threads walk (row, unit)
// items, a unit being V neighbouring pairs of one head, two vectors of 16 bytes.
// With a row of frequencies per head every pair has its own angle (37
// instructions, all told); a thread keeps one unit's frequencies in registers and
// walks rows, loading the next one's x ahead.  Issue slots are busy 64 % of the
// cycles there (1 x 9216 x 32 x 128 bf16, three axes: 35.6 us, 4.2 TB/s), and
// with 110 registers 16 warps of an SM are all there are to fill the rest while
// a quarter of their time goes to waiting for x: 512 threads have one row of 32
// bytes each under way, 16 KB an SM.
#include "common.cuh"

namespace ltxq {
namespace rotary {

constexpr int kThreads = 256;
constexpr int kTableMax = 2048;  // (cos, sin) pairs of one CTA's rows, or its (high, low) positions: 16 KB

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
  int units;      // per row: heads * (rotated units + units that pass through)
  int rot_units;  // per head
  int all_units;  // per head
  int rows_per_cta, units_per_cta;
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

// cos and sin of q / 4 + r turns, |r| <= 1/8
__device__ __forceinline__ void cos_sin_part(int q, float r, float& c, float& s) {
  const float z = r * 6.283185307179586f;
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
  // cos is negative in quadrants 1 and 2, sin in 2 and 3
  c = __uint_as_float(__float_as_uint(swap ? sn : cs) ^ ((static_cast<uint32_t>(q + 1) << 30) & 0x80000000u));
  s = __uint_as_float(__float_as_uint(swap ? cs : sn) ^ ((static_cast<uint32_t>(q) << 30) & 0x80000000u));
}

// cos and sin of t turns, any t: t = q / 4 + r, exact in fp64
__device__ __noinline__ void cos_sin_far(double t, float& c, float& s) {
  // the sum below stays in [2^52, 2^53), where its unit is 1, for |4t| < 2^51; NaN and infinity give NaN
  if (!(fabs(t) < 0x1p49)) t = t - rint(t);
  constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
  const double m = __dadd_rn(4.0 * t, kRound);
  cos_sin_part(__double2loint(m), static_cast<float>(__fma_rn(__dsub_rn(m, kRound), -0.25, t)), c, s);
}

constexpr double kInvTwoPi = 0.15915494309189535;

// an fp64 value as the sum of two fp32 ones
__device__ __forceinline__ float2 split2(double v) {
  const float hi = static_cast<float>(v);
  return make_float2(hi, static_cast<float>(v - static_cast<double>(hi)));
}

constexpr float kFarTurns = 1048576.0f;

// cos and sin of p * f turns, both as two parts, |p * f| < kFarTurns.  kShort:
// for results that are rounded to bf16, by 2^-9 to 2^-8 of a value, the hardware's
// functions, off by at most 2^-20.9 of the pair's length within a turn.  The
// series costs about twice as much per pair: 9216 x 32 x 64 fp32, half the pairs
// and the same bytes, takes 33.3 us where 9216 x 32 x 128 bf16 takes 35.
template <bool kShort>
__device__ __forceinline__ void cos_sin(float2 p, float2 f, float& c, float& s) {
  const float t = __fmul_rn(p.x, f.x);
  const float e = fmaf(p.x, f.x, -t) + fmaf(p.x, f.y, p.y * f.x);
  constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer
  if (kShort) {
    const float m = t + kRound;
    const float z = ((t - (m - kRound)) + e) * 6.283185307179586f;
    c = __cosf(z);
    s = __sinf(z);
  } else {
    const float m = fmaf(t, 4.0f, kRound);
    cos_sin_part(__float_as_int(m), fmaf(m - kRound, -0.25f, t) + e, c, s);
  }
}

// V elements as they lie in memory, and as fp32
template <typename T, int V>
struct Raw {
  static constexpr int kBytes = sizeof(T) * V;
  uint32_t w[(kBytes + 3) / 4];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kBytes == 16) {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else if constexpr (kBytes == 8) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      w[0] = u.x; w[1] = u.y;
    } else if constexpr (kBytes == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kBytes == 16) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (kBytes == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else if constexpr (kBytes == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
    else *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(w[0]);
  }
  __device__ __forceinline__ void get(float (&v)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(w[i]);
      else v[i] = i & 1 ? hi_bf16(w[i / 2]) : lo_bf16(w[i / 2]);
    }
  }
  __device__ __forceinline__ void put(const float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(v[i]);
      else if constexpr (V == 1) w[0] = f32_to_bf16(v[0]);
      else if (i % 2 == 0) w[i / 2] = pack_bf16x2(v[i], v[(i + 1) % V]);
    }
  }
};

// Where a unit's two vectors lie in its head: pairs of both halves, neighbours
// of the interleaved layout, or elements that pass through.
template <int V, bool kHalf>
struct Unit {
  int e0, e1;
  bool rot, second;
  __device__ __forceinline__ Unit(const Args& a, int c) {
    rot = c < a.rot_units;
    e0 = !rot ? 2 * a.half + (c - a.rot_units) * 2 * V : kHalf ? c * V : c * 2 * V;
    e1 = rot && kHalf ? e0 + a.half : e0 + V;
    second = rot || e1 < a.d;  // an odd head: the last unit that passes through is one element
  }
};

// rotates the V pairs of p, q; cs[i]: (cos, sin) of pair i
template <typename T, int V, bool kHalf>
__device__ __forceinline__ void rotate(Raw<T, V>& p, Raw<T, V>& q, const float2 (&cs)[V]) {
  float x[V], y[V];
  p.get(x);
  q.get(y);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    // interleaved: pair i is elements 2i, 2i + 1 of the unit's 2V
    float& m = kHalf ? x[i] : (2 * i < V ? x[2 * i % V] : y[2 * i % V]);
    float& o = kHalf ? y[i] : (2 * i + 1 < V ? x[(2 * i + 1) % V] : y[(2 * i + 1) % V]);
    const float mu = m, mv = o;
    m = fmaf(mu, cs[i].x, -(mv * cs[i].y));
    o = fmaf(mv, cs[i].x, mu * cs[i].y);
  }
  p.put(x);
  q.put(y);
}

// Heads that share the frequencies.  T: uint16_t (bf16) or float.  V pairs per
// unit: 16 bytes of each vector, or less where alignment or sizes leave no
// wider form.
template <typename T, int V, bool kHalf>
__global__ void __launch_bounds__(kThreads) rotary_shared_kernel(const Args a) {
  __shared__ float2 table[kTableMax];
  const int64_t row0 = blockIdx.x * static_cast<int64_t>(a.rows_per_cta);
  const int n = static_cast<int>(min(static_cast<int64_t>(a.rows_per_cta), a.rows - row0));
  // this CTA's share of the rows' units; an item's x is loaded one item ahead, the first one's before the table
  const int u0 = blockIdx.y * a.units_per_cta, nu = min(a.units_per_cta, a.units - u0);
  const int dr = kThreads / nu, du = kThreads - dr * nu;
  int nr = threadIdx.x / nu, ru = threadIdx.x - nr * nu;  // the item loaded next
  Raw<T, V> p, q;
  T* out = nullptr;
  int c = 0, r = nr;
  auto load = [&] {
    const int h = (u0 + ru) / a.all_units;
    c = u0 + ru - h * a.all_units;
    r = nr;
    const Unit<V, kHalf> w(a, c);
    const int64_t row = row0 + nr;
    const int64_t b = row / a.tokens, t = row - b * a.tokens;
    const T* x = static_cast<const T*>(a.x) + b * a.xs[0] + t * a.xs[1] + h * a.xs[2];
    out = static_cast<T*>(a.out) + b * a.os[0] + t * a.os[1] + h * a.os[2];
    p.load(x + w.e0);
    if (w.second) q.load(x + w.e1);
    nr += dr;
    ru += du;
    if (ru >= nu) {
      ru -= nu;
      ++nr;
    }
  };
  if (nr < n) load();
  for (int i = threadIdx.x; i < n * a.half; i += kThreads) {
    const int tr = i / a.half, k = i - tr * a.half;
    const int64_t row = row0 + tr;
    const int64_t b = row / a.tokens, t = row - b * a.tokens;
    const int ax = a.axis ? __ldg(a.axis + k) : 0;
    const double v = static_cast<unsigned>(ax) < static_cast<unsigned>(a.n_axes) ? load_pos(a, b, t, ax) : NAN;
    const double f = __ldg(a.freqs + k) * kInvTwoPi;
    const float2 ph = split2(a.inverse ? -v : v), fh = split2(f);
    float co, si;
    if (fabsf(ph.x * fh.x) < kFarTurns) cos_sin<sizeof(T) == 2>(ph, fh, co, si);
    else cos_sin_far(a.inverse ? -v * f : v * f, co, si);
    table[i] = make_float2(co * a.scale, si * a.scale);
  }
  __syncthreads();
  while (r < n) {
    Raw<T, V> m = p, o = q;
    T* const at = out;
    const int mc = c, mr = r;
    if (nr < n) load();
    else r = n;
    const Unit<V, kHalf> w(a, mc);
    if (w.rot) {
      float2 cs[V];
#pragma unroll
      for (int i = 0; i < V; ++i) cs[i] = table[mr * a.half + mc * V + i];
      rotate<T, V, kHalf>(m, o, cs);
    }
    m.store(at + w.e0);
    if (w.second) o.store(at + w.e1);
  }
}

// A row of frequencies for each head.
template <typename T, int V, bool kHalf>
__global__ void __launch_bounds__(kThreads) rotary_heads_kernel(const Args a) {
  __shared__ float2 pos[kTableMax];  // [row][axis]
  const int64_t row0 = blockIdx.x * static_cast<int64_t>(a.rows_per_cta);
  const int n = static_cast<int>(min(static_cast<int64_t>(a.rows_per_cta), a.rows - row0));
  const int threads = static_cast<int>(blockDim.x), u = blockIdx.y * threads + threadIdx.x;
  const bool live = u < a.units;
  const int h = live ? u / a.all_units : 0, c = live ? u - h * a.all_units : 0;
  const Unit<V, kHalf> w(a, c);
  const T* x = static_cast<const T*>(a.x) + h * a.xs[2];
  T* out = static_cast<T*>(a.out) + h * a.os[2];
  int64_t b = row0 / a.tokens, t = row0 - b * a.tokens;
  Raw<T, V> p, q;
  auto load = [&] {
    const T* xr = x + b * a.xs[0] + t * a.xs[1];
    p.load(xr + w.e0);
    if (w.second) q.load(xr + w.e1);
  };
  // the first row, the frequencies and the positions are read at once
  if (live) load();
  double fd[V];
  int ax[V];
  if (w.rot && live) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      fd[i] = __ldg(a.freqs + h * a.half + c * V + i);
      ax[i] = a.axis ? __ldg(a.axis + h * a.half + c * V + i) : 0;
    }
  }
  for (int i = threadIdx.x; i < n * a.n_axes; i += threads) {
    const int r = i / a.n_axes, ax1 = i - r * a.n_axes;
    const int64_t row = row0 + r;
    const int64_t b1 = row / a.tokens, t1 = row - b1 * a.tokens;
    const double p1 = load_pos(a, b1, t1, ax1);
    pos[i] = split2(a.inverse ? -p1 : p1);
  }
  __syncthreads();
  if (!live) return;
  float2 f[V];
  if (w.rot) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      f[i] = split2(fd[i] * kInvTwoPi);
      if (static_cast<unsigned>(ax[i]) >= static_cast<unsigned>(a.n_axes)) {
        f[i].x = NAN;
        ax[i] = 0;
      }
    }
  }
#pragma unroll 1
  for (int r = 0; r < n; ++r) {
    T* orow = out + b * a.os[0] + t * a.os[1];
    const int64_t b0 = b, t0 = t;
    Raw<T, V> m = p, o = q;
    if (++t == a.tokens) {
      t = 0;
      ++b;
    }
    if (r + 1 < n) load();
    if (w.rot) {
      float2 ph[V], cs[V];
      bool near = true;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        ph[i] = pos[r * a.n_axes + ax[i]];
        near = near && fabsf(ph[i].x * f[i].x) < kFarTurns;  // not for NaN: 0 times a position past fp32's range
      }
      if (near) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float c1, s1;
          cos_sin<sizeof(T) == 2>(ph[i], f[i], c1, s1);
          cs[i] = make_float2(c1 * a.scale, s1 * a.scale);
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const double v = load_pos(a, b0, t0, ax[i]) * (__ldg(a.freqs + h * a.half + c * V + i) * kInvTwoPi);
          float c1, s1;
          cos_sin_far(isnan(f[i].x) ? static_cast<double>(NAN) : a.inverse ? -v : v, c1, s1);
          cs[i] = make_float2(c1 * a.scale, s1 * a.scale);
        }
      }
      rotate<T, V, kHalf>(m, o, cs);
    }
    m.store(orow + w.e0);
    if (w.second) o.store(orow + w.e1);
  }
}

// ---------------------------------------------------------------- memory of x and out (host)

using Wide = __int128;  // strides times sizes of any call

// the axes of more than one element, by stride, smallest first (a head's elements among them)
struct Axes {
  int n = 0;
  int64_t size[4];
  Wide stride[4];
  Wide reach[5];  // largest distance of two elements along the first i axes
  Wide lo = 0, hi = 0;  // first and last element
  Axes(const ltxq_rotary_args& r, const int64_t* s) {
    const int64_t sz[4] = {r.head_dim, r.heads, r.tokens, r.batch}, st[4] = {1, s[2], s[1], s[0]};
    for (int i = 0; i < 4; ++i) {
      if (sz[i] <= 1) continue;
      const Wide last = static_cast<Wide>(sz[i] - 1) * st[i];
      (last < 0 ? lo : hi) += last;
      int at = n++;
      const Wide a = st[i] < 0 ? -static_cast<Wide>(st[i]) : st[i];
      for (; at > 0 && stride[at - 1] > a; --at) {
        size[at] = size[at - 1];
        stride[at] = stride[at - 1];
      }
      size[at] = sz[i];
      stride[at] = a;
    }
    reach[0] = 0;
    for (int i = 0; i < n; ++i) reach[i + 1] = reach[i] + static_cast<Wide>(size[i] - 1) * stride[i];
  }
  // every stride steps over all that the smaller ones reach: no element is met twice
  bool nested() const {
    for (int i = 0; i < n; ++i)
      if (stride[i] <= reach[i]) return false;
    return true;
  }
  // nested axes: whether some two elements lie `delta` apart, by the first k axes
  bool meets(Wide delta, int k) const {
    if (k == 0) return delta == 0;
    const Wide s = stride[k - 1];
    Wide i = delta / s;  // or the next one down: what is left has to be within reach of the smaller axes
    if (delta < 0 && i * s != delta) --i;
    for (int c = 0; c < 2; ++c, ++i) {
      const Wide rest = delta - i * s;
      if (i > -size[k - 1] && i < size[k - 1] && rest <= reach[k - 1] && -rest <= reach[k - 1] && meets(rest, k - 1))
        return true;
    }
    return false;
  }
};

// Threads rotate their own elements with no order among them, so out has one
// place for each, and shares one with x only as x itself.
static ltxq_status check_memory(const ltxq_rotary_args& r, int es) {
  const Axes x(r, r.x_stride), o(r, r.out_stride);
  constexpr Wide kFar = static_cast<Wide>(1) << 60;
  if (x.reach[x.n] >= kFar || o.reach[o.n] >= kFar) return fail(LTXQ_ERR_UNSUPPORTED, "rotary: strides too large");
  if (!o.nested()) return fail(LTXQ_ERR_INVALID, "rotary: out must have memory of its own for every element");
  const int64_t sizes[3] = {r.batch, r.tokens, r.heads};
  bool same = true;  // of two layouts with the same strides it can be told whether they meet
  for (int i = 0; i < 3; ++i) same = same && (sizes[i] <= 1 || r.x_stride[i] == r.out_stride[i]);
  const Wide bytes = static_cast<Wide>(reinterpret_cast<uintptr_t>(r.out)) -
                     static_cast<Wide>(reinterpret_cast<uintptr_t>(r.x));
  if (same && bytes == 0) return LTXQ_OK;
  if (bytes + o.lo * es >= (x.hi + 1) * es || bytes + (o.hi + 1) * es <= x.lo * es) return LTXQ_OK;  // apart
  if (same && bytes % es == 0 && !o.meets(bytes / es, o.n)) return LTXQ_OK;
  return fail(LTXQ_ERR_INVALID, "rotary: out must be x itself (with its strides) or share no memory with it");
}

template <typename T, int V>
static void launch(const Args& a, bool half_layout, dim3 grid, int threads, cudaStream_t s) {
  if (half_layout) {
    if (a.per_head) rotary_heads_kernel<T, V, true><<<grid, threads, 0, s>>>(a);
    else rotary_shared_kernel<T, V, true><<<grid, kThreads, 0, s>>>(a);
  } else {
    if (a.per_head) rotary_heads_kernel<T, V, false><<<grid, threads, 0, s>>>(a);
    else rotary_shared_kernel<T, V, false><<<grid, kThreads, 0, s>>>(a);
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
  const uintptr_t ps = r->pos_dtype == LTXQ_POS_I32 || r->pos_dtype == LTXQ_POS_F32 ? 4 : 8;
  if (r->rotary_dim > 0 && (reinterpret_cast<uintptr_t>(r->positions) % ps != 0 ||
                            reinterpret_cast<uintptr_t>(r->freqs) % 8 != 0 || reinterpret_cast<uintptr_t>(r->axis) % 4 != 0))
    return fail(LTXQ_ERR_UNSUPPORTED, "rotary: positions, freqs and axis must be aligned to their elements");
  if (ltxq_status st = check_memory(*r, es)) return st;

  Args a{};
  a.x = r->x;
  a.out = r->out;
  const int64_t half = r->rotary_dim / 2;
  // V: the widest vectors that start on their own size, 16 bytes, two elements or one
  auto fits = [&](int v) {
    bool ok = half % v == 0 && r->head_dim % (2 * v) == 0 &&
              ((reinterpret_cast<uintptr_t>(r->x) | reinterpret_cast<uintptr_t>(r->out)) % (v * es)) == 0;
    for (int i = 0; i < 3; ++i) ok = ok && r->x_stride[i] % v == 0 && r->out_stride[i] % v == 0;
    return ok;
  };
  const int V = fits(16 / es) ? 16 / es : fits(2) ? 2 : 1;
  for (int i = 0; i < 3; ++i) {
    a.xs[i] = r->x_stride[i];
    a.os[i] = r->out_stride[i];
    a.ps[i] = r->pos_stride[i];
  }
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
  a.per_head = r->freqs_per_head && half > 0 ? 1 : 0;  // a copy reads no positions, which may be NULL
  a.rot_units = a.half / V;
  a.all_units = a.rot_units + (a.d - 2 * a.half + 2 * V - 1) / (2 * V);
  a.units = a.heads * a.all_units;
  a.scale = r->scale;
  a.inverse = r->inverse ? 1 : 0;
  if (a.per_head && a.n_axes > kTableMax) return fail(LTXQ_ERR_UNSUPPORTED, "rotary: at most 2048 position axes");
  // Rows per CTA, within the table: shared frequencies, 1024 items of work (a few per thread, the table's cost spread
  // over every head), fewer where that would leave SMs idle.  A row of frequencies per head: as many threads as a row
  // has units, and rows so that the SMs are filled once, with 512 threads of 16-byte units or 1024 of narrower ones: a
  // CTA's start (frequencies, positions and first row, one trip to memory) is worth about ten rows.  9216 x 32 x 128
  // took 37.8 us with 16 rows a CTA, 43.6 with 8, 35.0 with the 32 that fill the SMs; 4000 x 32 x 36, whose units are
  // 4 bytes, 12.6 us with 1024 threads an SM, 19.3 with 512.
  int64_t per, gy;
  int threads = kThreads;
  const int sms = num_sms();
  if (a.per_head) {
    if (a.units < kThreads) threads = (a.units + 31) / 32 * 32;
    gy = (a.units + threads - 1) / threads;
    per = kTableMax / a.n_axes;
    a.units_per_cta = threads;
  } else {
    a.units_per_cta = a.units < 1024 ? a.units : 1024;
    gy = (a.units + a.units_per_cta - 1) / a.units_per_cta;
    per = 1024 / a.units_per_cta;
    if (a.half > 0 && per > kTableMax / a.half) per = kTableMax / a.half;
  }
  const int64_t ctas = static_cast<int64_t>(sms) * (!a.per_head ? 4 : (V * es == 16 ? 512 : 1024) / threads);
  const int64_t enough = (a.rows * gy + ctas - 1) / ctas;
  if (per > enough) per = enough;
  if (per < 1) per = 1;
  const int64_t gx = (a.rows + per - 1) / per;
  if (gy > 65535 || gx > 0x7FFFFFFF) return fail(LTXQ_ERR_UNSUPPORTED, "rotary: dimension too large");
  a.rows_per_cta = static_cast<int>(per);
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool hl = r->layout == LTXQ_ROTARY_HALF;
  if (es == 2) {
    if (V == 8) launch<uint16_t, 8>(a, hl, grid, threads, s);
    else if (V == 2) launch<uint16_t, 2>(a, hl, grid, threads, s);
    else launch<uint16_t, 1>(a, hl, grid, threads, s);
  } else {
    if (V == 4) launch<float, 4>(a, hl, grid, threads, s);
    else if (V == 2) launch<float, 2>(a, hl, grid, threads, s);
    else launch<float, 1>(a, hl, grid, threads, s);
  }
  return launch_check("rotary launch");
}
