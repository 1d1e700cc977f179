// Rotary positions of queries and keys, with or without an RMS norm of every head in front, and the gradients.
//
//   n = x * rsqrt(mean(x^2) + eps) * gamma                      (norm; otherwise n = x)
//   a_i = position * frequency_i,  c_i = scale * cos(a_i),  s_i = scale * sin(a_i),   i < r / 2
//   y_lo = n_lo c - n_hi s,  y_hi = n_hi c + n_lo s             over the r / 2 pairs (lo, hi) of a head: (i, i + r / 2)
//                                                               or (2 i, 2 i + 1); elements from r on are n itself
// Backward: dn = R^T dy, t = gamma dn, dx = rstd t - x rstd^3 mean(x t), dgamma = sum over rows of x rstd dn.
//
// HBM-bound: a row is read once and written once (backward: x and dy read, dx written); positions, frequencies and
// gammas are a few hundred bytes per token or less.  Queries and keys of a token share its angles, so one launch does
// both.  The angle is multiplied and reduced to a fraction of a turn in 64 bits and their rests: at position 10^6 a
// 32-bit product is off by up to 0.03 rad, while sin and cos of the fraction are right in fp32.  A CTA computes the sines of its tokens into shared
// memory once; a group of 4 to 32 lanes then owns a row and keeps both halves of each pair in one lane, so that the
// rotation needs no exchange and the norm one shuffle reduction.  All arithmetic is fp32, one rounding at the store.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/asc_cuda.h"
#include "host_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxHeadDim = 1024;
constexpr int kFwdCtas = 3;     // per SM: 80 registers a thread (2: 74, 3: 67, 4, which spills: 86 us at [1, 16384, 32 + 8, 128])

struct Operand {           // a [batch, sequence, head, dim] tensor: strides in elements, dim contiguous
  void* p;
  int64_t b, s, h;
};

struct RotaryArgs {
  Operand x[2], y[2];      // queries, keys: input and output (forward); x and dx (backward)
  Operand dy[2];           // backward only
  const void* gamma[2];    // null: ones
  float* partial;          // backward: [CTAs, D] partial sums of dgamma
  const void* positions;
  const double* freq;
  int64_t pos_b, pos_s;
  int32_t S, tokens;       // tokens = batch * S
  int32_t heads[2];
  int32_t D, r;
  int32_t log_lanes;       // lanes per row (vector kernels)
  int32_t slices;          // parts a token's heads are cut into, one warp each (vector kernels)
  int32_t q_ctas;          // any-size backward: CTAs [0, q_ctas) own queries, the others keys
  int32_t gamma_type;      // 0 fp16, 1 bf16, 2 fp32
  int32_t pos32;           // positions are int32 instead of int64
  int32_t norm, interleaved, conj;
  float eps, scale;
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// kBytes (16 or 8) of a row <-> fp32 registers
template <int kBytes>
struct RawOf;
template <>
struct RawOf<16> {
  using Type = uint4;
  __device__ static uint4 zero() { return make_uint4(0, 0, 0, 0); }
};
template <>
struct RawOf<8> {
  using Type = uint2;
  __device__ static uint2 zero() { return make_uint2(0, 0); }
};
__device__ __forceinline__ float2 unpack2(uint32_t w, const __half*) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float2 unpack2(uint32_t w, const __nv_bfloat16*) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __half*) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T, int kBytes>
struct Vec {
  static constexpr int E = kBytes / 2;
  using Raw = typename RawOf<kBytes>::Type;
  __device__ static Raw zero() { return RawOf<kBytes>::zero(); }
  __device__ static void unpack(const Raw& t, float* v) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&t);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float2 f = unpack2(w[i], static_cast<const T*>(nullptr));
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  }
  __device__ static Raw pack(const float* v) {
    Raw t;
    uint32_t* w = reinterpret_cast<uint32_t*>(&t);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) w[i] = pack2(v[2 * i], v[2 * i + 1], static_cast<const T*>(nullptr));
    return t;
  }
};
template <>
struct Vec<float, 16> {
  static constexpr int E = 4;
  using Raw = uint4;
  __device__ static uint4 zero() { return make_uint4(0, 0, 0, 0); }
  __device__ static void unpack(const uint4& t, float* v) {
    v[0] = __uint_as_float(t.x), v[1] = __uint_as_float(t.y), v[2] = __uint_as_float(t.z), v[3] = __uint_as_float(t.w);
  }
  __device__ static uint4 pack(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};

__device__ __forceinline__ float load_gamma(const RotaryArgs& a, int which, int i) {
  const void* g = a.gamma[which];
  if (g == nullptr) return 1.f;
  if (a.gamma_type == 0) return __half2float(static_cast<const __half*>(g)[i]);
  if (a.gamma_type == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(g)[i]);
  return static_cast<const float*>(g)[i];
}

// scale * (cos, sin) of the angle of pair `f` at position `pos`; `conj` turns back
__device__ __forceinline__ float2 turn_of(const RotaryArgs& a, double pos, int f) {
  // turns = pos * f / (2 pi) as a rounded value and what the roundings left out, so that the fraction of a turn is
  // right to 2^-50 at any position (in plain 64 bits it would be off by 2^-16 of a turn at position 2^40)
  constexpr double kInv2Pi = 0.15915494309189535, kInv2PiRest = -9.839338337591243e-18;
  const double frequency = a.freq[f];
  const double angle = pos * frequency, angle_rest = fma(pos, frequency, -angle);
  const double turns = angle * kInv2Pi;
  const double rest = fma(angle, kInv2Pi, -turns) + (angle * kInv2PiRest + angle_rest * kInv2Pi);
  float sn, cs;
  sincospif(static_cast<float>(2.0 * ((turns - rint(turns)) + rest)), &sn, &cs);
  return make_float2(cs * a.scale, (a.conj ? -sn : sn) * a.scale);
}

template <typename T>
__device__ __forceinline__ T* row_of(const Operand& o, int b, int s, int h) {
  return static_cast<T*>(o.p) + b * o.b + s * o.s + h * o.h;
}

// Which two vectors (of 16 or 8 bytes, E elements) of a row a lane owns.  Half layout: lane < r / 2 / E owns the vectors of both halves of its
// pairs; later lanes own two neighbours of the part that is not turned.  Interleaved: both halves of a pair lie in one
// vector, and a lane owns vectors `lane` and `lane + ceil(n / 2)`.
template <int E>
struct LaneVectors {
  int v0, v1;
  bool has0, has1, turns;     // turns: half layout, this lane holds pairs
  __device__ LaneVectors(const RotaryArgs& a, int lane) {
    const int n = a.D / E;
    if (a.interleaved) {
      const int half = (n + 1) / 2;
      v0 = lane, v1 = lane + half;
      has0 = lane < half, has1 = has0 && v1 < n, turns = false;
    } else {
      const int hv = a.r / 2 / E;
      turns = lane < hv;
      v0 = turns ? lane : 2 * lane;             // 2 hv + 2 (lane - hv)
      v1 = turns ? lane + hv : v0 + 1;
      has0 = v0 < n, has1 = v1 < n;
      if (turns) has0 = has1 = true;
    }
  }
};

// Coefficients of a lane's rotation, as pairs of fp32 registers (packed arithmetic halves the instructions).  Half layout,
// E pairs of elements (x_lo[e], x_hi[e]):  y_lo = lo_lo x_lo + lo_hi x_hi,  y_hi = hi_hi x_hi + hi_lo x_lo,  with the
// gammas multiplied in once per token.  Interleaved: the same for the pair (v[2 e], v[2 e + 1]).
template <int E>
struct Turn {
  float2 lo_lo[E / 2], lo_hi[E / 2], hi_hi[E / 2], hi_lo[E / 2];
};

template <int E>
__device__ __forceinline__ float& at(float2 (&v)[E], int i) {
  return (i & 1) ? v[i >> 1].y : v[i >> 1].x;
}

// index of the angle of the lane's pair e; r / 2 or more: not turned
template <int E, bool kInter>
__device__ __forceinline__ int angle_of(const RotaryArgs& a, const LaneVectors<E>& l, int e) {
  if (kInter) return (e < E / 2 ? l.v0 : l.v1) * (E / 2) + (e & (E / 2 - 1));
  return l.turns ? l.v0 * E + e : a.r / 2;
}

template <int E, bool kInter, bool kNorm>
__device__ __forceinline__ void lane_turn(const RotaryArgs& a, const LaneVectors<E>& l, const float2* table,
                                          const float* gamma, Turn<E>& t) {
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int f = angle_of<E, kInter>(a, l, e);
    const float2 cs = f < a.r / 2 ? table[f] : make_float2(1.f, 0.f);
    float g_lo = 1.f, g_hi = 1.f;
    if (kNorm) {
      // gammas of the two elements of pair e; elements past the end of the row read as 0 and are not stored
      const int lo = kInter ? (e < E / 2 ? l.v0 : l.v1) * E + 2 * (e & (E / 2 - 1)) : l.v0 * E + e;
      const int hi = kInter ? lo + 1 : l.v1 * E + e;
      g_lo = lo < a.D ? gamma[lo] : 0.f;
      g_hi = hi < a.D ? gamma[hi] : 0.f;
    }
    at(t.lo_lo, e) = g_lo * cs.x;
    at(t.hi_hi, e) = g_hi * cs.x;
    at(t.lo_hi, e) = -g_hi * cs.y;
    at(t.hi_lo, e) = g_lo * cs.y;
  }
}

// Values that are not part of a pair are only scaled: their neighbours may be infinite or NaN.
template <int E, bool kInter>
__device__ __forceinline__ void apply(const RotaryArgs& a, const LaneVectors<E>& l, const Turn<E>& t, float2 (&v)[E]) {
  if (kInter) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float2 x = v[e];
      const bool turns = angle_of<E, kInter>(a, l, e) < a.r / 2;
      const float lo = x.x * ((e & 1) ? t.lo_lo[e / 2].y : t.lo_lo[e / 2].x);
      const float hi = x.y * ((e & 1) ? t.hi_hi[e / 2].y : t.hi_hi[e / 2].x);
      v[e].x = turns ? fmaf(x.y, (e & 1) ? t.lo_hi[e / 2].y : t.lo_hi[e / 2].x, lo) : lo;
      v[e].y = turns ? fmaf(x.x, (e & 1) ? t.hi_lo[e / 2].y : t.hi_lo[e / 2].x, hi) : hi;
    }
  } else {
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
      const float2 lo = v[e], hi = v[E / 2 + e];
      v[e] = __fmul2_rn(lo, t.lo_lo[e]);
      v[E / 2 + e] = __fmul2_rn(hi, t.hi_hi[e]);
      if (l.turns) {
        v[e] = __ffma2_rn(hi, t.lo_hi[e], v[e]);
        v[E / 2 + e] = __ffma2_rn(lo, t.hi_lo[e], v[E / 2 + e]);
      }
    }
  }
}

__device__ __forceinline__ float group_sum(float v, int log_lanes) {
  for (int o = 1 << log_lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ double position_at(const RotaryArgs& a, int b, int s) {
  const int64_t i = b * a.pos_b + s * a.pos_s;
  return a.pos32 ? static_cast<double>(static_cast<const int32_t*>(a.positions)[i])
                 : static_cast<double>(static_cast<const int64_t*>(a.positions)[i]);
}

// Shared memory of the vector kernels: gammas of queries and keys as fp32 (D each, where there is a norm), then r / 2
// angles for every warp.  Loads the gammas.
__device__ __forceinline__ float2* stage(const RotaryArgs& a, float* smem) {
  int floats = 0;
  if (a.norm) {
    for (int i = threadIdx.x; i < 2 * a.D; i += kThreads) smem[i] = load_gamma(a, i >= a.D, i >= a.D ? i - a.D : i);
    floats = 2 * a.D;
  }
  __syncthreads();
  return reinterpret_cast<float2*>(smem + floats) + (threadIdx.x >> 5) * (a.r / 2);
}

// What a group of lanes does next: rows of one token, queries (w = 0) and then keys, each from head `first` in steps.
struct Place {
  int b, s, first;
};

// The vectors of one tensor's rows that a lane owns, as a pointer that walks over the heads of a token.
template <typename T, int kBytes>
struct RowWalk {
  using V = Vec<T, kBytes>;
  using Raw = typename V::Raw;
  const Raw* at;
  int64_t stride;            // in vectors
  __device__ RowWalk(const Operand& o, const Place& p, int v0, int step)
      : at(reinterpret_cast<const Raw*>(row_of<const T>(o, p.b, p.s, p.first)) + v0), stride(o.h * step / V::E) {}
  __device__ void next() { at += stride; }
  __device__ Raw* out() const { return const_cast<Raw*>(at); }
};

// --------------------------------------------------------------------------------------------------------------
// Forward, whole vectors.  A warp works on one token, or on a slice of its heads where tokens are few: it
// computes the token's angles into its own piece of shared memory (no barrier beyond the warp), then its groups of
// lanes take the queries in turn and then the keys.  The next row, also the next token's first, is loaded before the
// current one is computed.  Warps stride over the tokens.
// --------------------------------------------------------------------------------------------------------------
template <typename T, int kBytes, bool kNorm, bool kInter>
__global__ void __launch_bounds__(kThreads, kFwdCtas) rotary_fwd_kernel(const __grid_constant__ RotaryArgs a) {
  using V = Vec<T, kBytes>;
  using Raw = typename V::Raw;
  constexpr int E = V::E;
  extern __shared__ float smem[];
  float2* table = stage(a, smem);
  const int lane = threadIdx.x & ((1 << a.log_lanes) - 1), group = (threadIdx.x & 31) >> a.log_lanes;
  const int groups = 32 >> a.log_lanes;
  const int step = groups * a.slices;
  const int warps = gridDim.x * kWarps;
  const int units = a.tokens * a.slices;
  const LaneVectors<E> l(a, lane);
  const float inv_d = 1.f / a.D;
  const int w_first = a.heads[0] > 0 ? 0 : 1;

  auto place = [&](int unit) {
    const int token = unit / a.slices;
    const int b = token / a.S;
    return Place{b, token - b * a.S, (unit - token * a.slices) * groups + group};
  };
  auto load = [&](const Raw* at, bool on, Raw& lo, Raw& hi) {
    lo = hi = V::zero();
    if (on && l.has0) lo = at[0];
    if (on && l.has1) hi = at[l.v1 - l.v0];
  };
  int unit = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (unit >= units) return;
  Place p = place(unit);
  Raw lo, hi;
  load(RowWalk<T, kBytes>(a.x[w_first], p, l.v0, step).at, p.first < a.heads[w_first], lo, hi);
  double pos = a.r > 0 ? position_at(a, p.b, p.s) : 0.0;
  for (; unit < units; unit += warps) {
    __syncwarp();                                  // the previous token's angles are no longer read
    for (int f = threadIdx.x & 31; f < a.r / 2; f += 32) table[f] = turn_of(a, pos, f);
    __syncwarp();
    Place next = p;
    const bool more = unit + warps < units;
    if (more) {
      next = place(unit + warps);
      if (a.r > 0) pos = position_at(a, next.b, next.s);
    }
    Turn<E> t;
    if (!kNorm) lane_turn<E, kInter, kNorm>(a, l, table, nullptr, t);
#pragma unroll 1
    for (int w = 0; w < 2; ++w) {
      const int H = a.heads[w];
      if (H == 0) continue;
      const int iters = (H + step - 1) / step;
      if (kNorm) lane_turn<E, kInter, kNorm>(a, l, table, smem + w * a.D, t);
      RowWalk<T, kBytes> in(a.x[w], p, l.v0, step), out(a.y[w], p, l.v0, step);
      int h = p.first;
      for (int it = 0; it < iters; ++it, h += step) {
        float2 v[E];
        V::unpack(lo, reinterpret_cast<float*>(v));
        V::unpack(hi, reinterpret_cast<float*>(v + E / 2));
        if (it + 1 < iters) {
          in.next();
          load(in.at, h + step < H, lo, hi);
        } else if (w == 0 && a.heads[1] > 0) {
          load(RowWalk<T, kBytes>(a.x[1], p, l.v0, step).at, p.first < a.heads[1], lo, hi);
        } else if (more) {
          load(RowWalk<T, kBytes>(a.x[w_first], next, l.v0, step).at, next.first < a.heads[w_first], lo, hi);
        }
        if (kNorm) {
          float2 ss = make_float2(0.f, 0.f);
#pragma unroll
          for (int e = 0; e < E; ++e) ss = __ffma2_rn(v[e], v[e], ss);
          const float rstd = rsqrtf(group_sum(ss.x + ss.y, a.log_lanes) * inv_d + a.eps);
#pragma unroll
          for (int e = 0; e < E; ++e) v[e] = __fmul2_rn(v[e], make_float2(rstd, rstd));
        }
        if (h < H) {
          apply<E, kInter>(a, l, t, v);
          Raw* row = out.out();
          if (l.has0) row[0] = V::pack(reinterpret_cast<float*>(v));
          if (l.has1) row[l.v1 - l.v0] = V::pack(reinterpret_cast<float*>(v + E / 2));
        }
        out.next();
      }
    }
    p = next;
  }
}

// --------------------------------------------------------------------------------------------------------------
// Backward through norm and rotation, whole vectors: the forward's division of the work.  A lane's sums for
// dgamma stay in registers over a token's queries (then its keys) and are added to the lane's own place in shared memory
// after them, so that queries and keys share the angles without two sets of sums in registers.
// --------------------------------------------------------------------------------------------------------------
template <typename T, int kBytes, bool kInter>
__global__ void __launch_bounds__(kThreads, 2) rotary_bwd_kernel(const __grid_constant__ RotaryArgs a) {
  using V = Vec<T, kBytes>;
  using Raw = typename V::Raw;
  constexpr int E = V::E;
  extern __shared__ float smem[];
  ascdev::let_next_start();
  float2* table = stage(a, smem);
  // [queries, keys][pair][thread], behind the angles
  float2* sums = reinterpret_cast<float2*>(smem + 2 * a.D) + kWarps * (a.r / 2);
  const int lane = threadIdx.x & ((1 << a.log_lanes) - 1), group = (threadIdx.x & 31) >> a.log_lanes;
  const int groups = 32 >> a.log_lanes;
  const int H = a.heads[0] + a.heads[1];
  const int step = groups * a.slices;
  const int iters = (H + step - 1) / step;
  const int warps = gridDim.x * kWarps;
  const int units = a.tokens * a.slices;
  const LaneVectors<E> l(a, lane);
  const float inv_d = 1.f / a.D;
#pragma unroll
  for (int e = 0; e < 2 * E; ++e) sums[e * kThreads + threadIdx.x] = make_float2(0.f, 0.f);

  auto place = [&](int unit) {
    const int token = unit / a.slices;
    const int b = token / a.S;
    return Place{b, token - b * a.S, (unit - token * a.slices) * groups + group};
  };
  auto load = [&](const Place& p, int h, Raw (&x)[2], Raw (&y)[2]) {
    x[0] = x[1] = y[0] = y[1] = V::zero();
    if (h >= H) return;
    const int w = h >= a.heads[0];
    const int hw = h - (w ? a.heads[0] : 0);
    const Raw* xr = reinterpret_cast<const Raw*>(row_of<const T>(a.x[w], p.b, p.s, hw));
    const Raw* yr = reinterpret_cast<const Raw*>(row_of<const T>(a.dy[w], p.b, p.s, hw));
    if (l.has0) x[0] = xr[l.v0], y[0] = yr[l.v0];
    if (l.has1) x[1] = xr[l.v1], y[1] = yr[l.v1];
  };
  float2 g[E], dg[E];
  int which = -1;
  auto flush = [&]() {
    float2* to = sums + which * E * kThreads + threadIdx.x;
#pragma unroll
    for (int e = 0; e < E; ++e) to[e * kThreads] = __fadd2_rn(to[e * kThreads], dg[e]);
  };
  int unit = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (unit < units) {
    Place p = place(unit);
    Raw x[2], y[2];
    load(p, p.first, x, y);
    double pos = a.r > 0 ? position_at(a, p.b, p.s) : 0.0;
    for (; unit < units; unit += warps) {
      __syncwarp();
      for (int f = threadIdx.x & 31; f < a.r / 2; f += 32) table[f] = turn_of(a, pos, f);
      __syncwarp();
      Place next = p;
      const bool more = unit + warps < units;
      if (more) {
        next = place(unit + warps);
        if (a.r > 0) pos = position_at(a, next.b, next.s);
      }
      float2 c[E / 2], sn[E / 2];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int f = angle_of<E, kInter>(a, l, e);
        const float2 cs = f < a.r / 2 ? table[f] : make_float2(1.f, 0.f);
        at(c, e) = cs.x, at(sn, e) = cs.y;
      }
      for (int it = 0; it < iters; ++it) {
        const int h = p.first + it * step;
        const int w = h >= a.heads[0];
        if (w != which) {
          if (which >= 0) flush();
          which = w;
          const float* gamma = smem + w * a.D;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            at(g, e) = l.has0 ? gamma[l.v0 * E + e] : 0.f;
            at(g, E + e) = l.has1 ? gamma[l.v1 * E + e] : 0.f;
            dg[e] = make_float2(0.f, 0.f);
          }
        }
        float2 v[E], d[E];
        V::unpack(x[0], reinterpret_cast<float*>(v));
        V::unpack(x[1], reinterpret_cast<float*>(v + E / 2));
        V::unpack(y[0], reinterpret_cast<float*>(d));
        V::unpack(y[1], reinterpret_cast<float*>(d + E / 2));
        if (it + 1 < iters) load(p, h + step, x, y);
        else if (more) load(next, next.first, x, y);
        // d = R^T dy
        if (kInter) {
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float2 t = d[e];
            const float ce = (e & 1) ? c[e / 2].y : c[e / 2].x, se = (e & 1) ? sn[e / 2].y : sn[e / 2].x;
            if (angle_of<E, kInter>(a, l, e) < a.r / 2)
              d[e] = make_float2(fmaf(t.y, se, t.x * ce), fmaf(-t.x, se, t.y * ce));
          }
        } else if (l.turns) {
#pragma unroll
          for (int e = 0; e < E / 2; ++e) {
            const float2 q = d[e], r = d[E / 2 + e];
            d[e] = __ffma2_rn(r, sn[e], __fmul2_rn(q, c[e]));
            d[E / 2 + e] = __ffma2_rn(q, make_float2(-sn[e].x, -sn[e].y), __fmul2_rn(r, c[e]));
          }
        }
        float2 ss = make_float2(0.f, 0.f), xt = make_float2(0.f, 0.f);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          ss = __ffma2_rn(v[e], v[e], ss);
          xt = __ffma2_rn(__fmul2_rn(v[e], g[e]), d[e], xt);
        }
        const float total = group_sum(ss.x + ss.y, a.log_lanes), along = group_sum(xt.x + xt.y, a.log_lanes);
        const float rstd = rsqrtf(total * inv_d + a.eps);
        const float k = -rstd * rstd * rstd * along * inv_d;
        if (h < H) {
          const float2 r2 = make_float2(rstd, rstd), k2 = make_float2(k, k);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float2 rd = __fmul2_rn(r2, d[e]);
            dg[e] = __ffma2_rn(v[e], rd, dg[e]);
            d[e] = __ffma2_rn(v[e], k2, __fmul2_rn(g[e], rd));
          }
          Raw* row = reinterpret_cast<Raw*>(row_of<T>(a.y[w], p.b, p.s, h - (w ? a.heads[0] : 0)));
          if (l.has0) row[l.v0] = V::pack(reinterpret_cast<float*>(d));
          if (l.has1) row[l.v1] = V::pack(reinterpret_cast<float*>(d + E / 2));
        }
      }
      p = next;
    }
    flush();
  }
  if (a.partial == nullptr) return;
  // sums of this CTA in group order, then one row of partial sums of queries and one of keys per CTA: the same order in
  // every run
  __syncthreads();
  const int per_row = 1 << a.log_lanes;
  for (int i = threadIdx.x; i < 2 * E * per_row; i += kThreads) {
    const int e = i >> a.log_lanes, at_lane = i & (per_row - 1);       // e < E: queries
    float2 t = make_float2(0.f, 0.f);
    for (int k = 0; k < kThreads >> a.log_lanes; ++k)
      t = __fadd2_rn(t, sums[e * kThreads + (k << a.log_lanes) + at_lane]);
    const LaneVectors<E> o(a, at_lane);
    const int pair = e & (E - 1);
    const bool lo = pair < E / 2;
    if (lo ? o.has0 : o.has1) {
      float* to = a.partial + (static_cast<int64_t>(e >= E ? gridDim.x : 0) + blockIdx.x) * a.D +
                  (lo ? o.v0 : o.v1) * E + 2 * (pair & (E / 2 - 1));
      to[0] = t.x, to[1] = t.y;
    }
  }
}

// --------------------------------------------------------------------------------------------------------------
// Any head size up to 1024, any alignment: a warp owns a row and reads it twice, element by element.
// --------------------------------------------------------------------------------------------------------------
template <typename T, bool kBwd>
__global__ void __launch_bounds__(kThreads) rotary_any_kernel(const RotaryArgs a) {
  extern __shared__ float2 table[];              // r / 2 angles, then (backward) D sums for each warp
  const int half_r = a.r / 2;
  float* dg = reinterpret_cast<float*>(table + half_r) + (threadIdx.x >> 5) * a.D;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int w0 = kBwd && blockIdx.x >= a.q_ctas;
  const int cta = w0 ? blockIdx.x - a.q_ctas : blockIdx.x;
  const int ctas = !kBwd ? gridDim.x : w0 ? gridDim.x - a.q_ctas : a.q_ctas;
  const int H = kBwd ? a.heads[w0] : a.heads[0] + a.heads[1];
  const float inv_d = 1.f / a.D;
  if (kBwd)
    for (int i = lane; i < a.D; i += 32) dg[i] = 0.f;
  for (int token = cta; token < a.tokens; token += ctas) {
    __syncthreads();
    const int b = token / a.S, s = token - b * a.S;
    for (int i = threadIdx.x; i < half_r; i += kThreads) table[i] = turn_of(a, position_at(a, b, s), i);
    __syncthreads();
    for (int hh = warp; hh < H; hh += kWarps) {
      const int w = kBwd ? w0 : hh >= a.heads[0];
      const int h = !kBwd && w ? hh - a.heads[0] : hh;
      const T* x = row_of<const T>(a.x[w], b, s, h);
      const T* dy = kBwd ? row_of<const T>(a.dy[w], b, s, h) : nullptr;
      T* y = row_of<T>(a.y[w], b, s, h);
      // element p of the part that is turned pairs with element q; d = R^T dy of both
      auto pair_at = [&](int i, int& p, int& q) {
        p = a.interleaved ? 2 * i : i;
        q = a.interleaved ? 2 * i + 1 : i + half_r;
      };
      auto turned_back = [&](int i, int p, int q, float& dp, float& dq) {
        const float u = to_float(dy[p]), v = to_float(dy[q]);
        dp = u * table[i].x + v * table[i].y;
        dq = v * table[i].x - u * table[i].y;
      };
      float rstd = 1.f, k = 0.f;
      if (a.norm) {
        float ss = 0.f, xt = 0.f;
        for (int i = lane; i < a.D; i += 32) {
          const float t = to_float(x[i]);
          ss = fmaf(t, t, ss);
          if (kBwd && i >= a.r) xt = fmaf(t * load_gamma(a, w, i), to_float(dy[i]), xt);
        }
        if (kBwd) {
          for (int i = lane; i < half_r; i += 32) {
            int p, q;
            float dp, dq;
            pair_at(i, p, q);
            turned_back(i, p, q, dp, dq);
            xt = fmaf(to_float(x[p]) * load_gamma(a, w, p), dp, xt);
            xt = fmaf(to_float(x[q]) * load_gamma(a, w, q), dq, xt);
          }
          xt = group_sum(xt, 5);
        }
        rstd = 1.f / sqrtf(group_sum(ss, 5) * inv_d + a.eps);
        k = rstd * rstd * rstd * xt * inv_d;
      }
      __syncwarp();
      if (kBwd) {
        auto finish = [&](int i, float d) {
          const float t = to_float(x[i]);
          dg[i] = fmaf(t * rstd, d, dg[i]);
          return rstd * (load_gamma(a, w, i) * d) - t * k;
        };
        for (int i = lane; i < half_r; i += 32) {
          int p, q;
          float dp, dq;
          pair_at(i, p, q);
          turned_back(i, p, q, dp, dq);
          dp = finish(p, dp), dq = finish(q, dq);
          y[p] = from_float<T>(dp), y[q] = from_float<T>(dq);
        }
        for (int i = a.r + lane; i < a.D; i += 32) y[i] = from_float<T>(finish(i, to_float(dy[i])));
      } else {
        auto normed = [&](int i) {
          return a.norm ? to_float(x[i]) * rstd * load_gamma(a, w, i) : to_float(x[i]);
        };
        for (int i = lane; i < half_r; i += 32) {
          int p, q;
          pair_at(i, p, q);
          const float u = normed(p), v = normed(q);
          y[p] = from_float<T>(u * table[i].x - v * table[i].y);
          y[q] = from_float<T>(v * table[i].x + u * table[i].y);
        }
        for (int i = a.r + lane; i < a.D; i += 32) y[i] = from_float<T>(normed(i));
      }
    }
  }
  if (kBwd && a.partial != nullptr) {
    __syncthreads();
    const float* all = reinterpret_cast<const float*>(table + half_r);
    for (int i = threadIdx.x; i < a.D; i += kThreads) {
      float t = 0.f;
      for (int k = 0; k < kWarps; ++k) t += all[k * a.D + i];
      a.partial[static_cast<int64_t>(blockIdx.x) * a.D + i] = t;
    }
  }
}

// dgamma[w][c] = sum over the rows of partial sums of queries (w = 0; the first q_rows) or keys (w = 1), in a fixed
// order: 32 interleaved sums in 64 bits.  Latency-bound: a few hundred rows of D floats, so the loads of a thread are
// independent of each other (eight at a time) and a CTA takes 32 columns.
constexpr int kSumParts = 32;
__global__ void __launch_bounds__(32 * kSumParts) dgamma_kernel(const float* partial, int q_rows, int rows, int D,
                                                                float* dq_gamma, float* dk_gamma) {
  __shared__ double red[kSumParts][32];
  const int lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane, part = threadIdx.x >> 5;
  const int lo = blockIdx.y ? q_rows : 0, hi = blockIdx.y ? rows : q_rows;
  float* out = blockIdx.y ? dk_gamma : dq_gamma;
  double t = 0.0;
  ascdev::wait_for_previous();
  if (c < D)
    for (int i = lo + part; i < hi; i += 8 * kSumParts) {
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        x[k] = i + k * kSumParts < hi ? partial[static_cast<int64_t>(i + k * kSumParts) * D + c] : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) t += x[k];
    }
  red[part][lane] = t;
  __syncthreads();
  if (part == 0 && c < D && out != nullptr) {
#pragma unroll
    for (int k = 1; k < kSumParts; ++k) t += red[k][lane];
    out[c] = static_cast<float>(t);
  }
}

// ------------------------------------------------ host ---------------------------------------------------------
int64_t type_size(int32_t dtype) { return dtype == 2 ? 4 : 2; }

struct Problem {
  int64_t B, S, H[2], D, r;
  int32_t dtype;
};

// Fills an operand; a stride of a dimension of one element is never used and is read as 0.
Operand operand(const void* p, const int64_t* strides, const Problem& pr, int w) {
  return {const_cast<void*>(p), pr.B > 1 ? strides[0] : 0, pr.S > 1 ? strides[1] : 0, pr.H[w] > 1 ? strides[2] : 0};
}

// Elements of an output must not share memory: no stride of 0 over several elements.
bool writes_apart(const Operand& o, const Problem& pr, int w) {
  return (pr.B <= 1 || o.b != 0) && (pr.S <= 1 || o.s != 0) && (pr.H[w] <= 1 || o.h != 0);
}

bool is_vector_operand(const Operand& o, int64_t E, int bytes) {
  return reinterpret_cast<uintptr_t>(o.p) % bytes == 0 && o.b % E == 0 && o.s % E == 0 && o.h % E == 0;
}

// Checks shared by both directions; *done: there is nothing to compute.
int32_t check(const int64_t* dims, const int64_t* strides, const void* positions, const double* freq, int32_t dtype,
              int32_t gamma_dtype, int32_t flags, Problem& pr, bool* done) {
  *done = false;
  if (dims == nullptr || strides == nullptr) return ASC_ERR_INVALID_ARG;
  pr = {dims[0], dims[1], {dims[2], dims[3]}, dims[4], dims[5], dtype};
  if (dtype < 0 || dtype > 2 || gamma_dtype < 0 || gamma_dtype > 2 || (flags & ~15) != 0) return ASC_ERR_INVALID_ARG;
  if (pr.B < 0 || pr.S < 0 || pr.H[0] < 0 || pr.H[1] < 0 || pr.D < 0 || pr.r < 0 || pr.r > pr.D || pr.r % 2 != 0)
    return ASC_ERR_INVALID_ARG;
  if (pr.D > kMaxHeadDim || pr.H[0] > 0x100000 || pr.H[1] > 0x100000) return ASC_ERR_TOO_LARGE;
  if (pr.B == 0 || pr.S == 0 || pr.D == 0 || pr.H[0] + pr.H[1] == 0) {
    *done = true;
    return ASC_OK;
  }
  // token numbers stay below 2^30, so that rounding them up to a chunk cannot pass 32 bits
  if (pr.S > (1 << 30) || pr.B > (1 << 30) || pr.B * pr.S > (1 << 30)) return ASC_ERR_TOO_LARGE;
  if (pr.r > 0 && (positions == nullptr || freq == nullptr)) return ASC_ERR_INVALID_ARG;
  const uintptr_t pos_align = (flags & 4) ? 4 : 8;
  if (reinterpret_cast<uintptr_t>(positions) % pos_align != 0 || reinterpret_cast<uintptr_t>(freq) % 8 != 0)
    return ASC_ERR_MISALIGNED;
  return ASC_OK;
}

void fill(RotaryArgs& a, const Problem& pr, const int64_t* pos_strides, const void* positions, const double* freq,
          float eps, float scale, int32_t gamma_dtype, int32_t flags) {
  a.positions = positions;
  a.freq = freq;
  a.pos_b = pr.B > 1 ? pos_strides[0] : 0;
  a.pos_s = pr.S > 1 ? pos_strides[1] : 0;
  a.S = static_cast<int32_t>(pr.S);
  a.tokens = static_cast<int32_t>(pr.B * pr.S);
  a.heads[0] = static_cast<int32_t>(pr.H[0]);
  a.heads[1] = static_cast<int32_t>(pr.H[1]);
  a.D = static_cast<int32_t>(pr.D);
  a.r = static_cast<int32_t>(pr.r);
  a.interleaved = flags & 1;
  a.norm = (flags >> 1) & 1;
  a.pos32 = (flags >> 2) & 1;
  a.conj = (flags >> 3) & 1;
  a.gamma_type = gamma_dtype;
  a.eps = eps;
  a.scale = scale;
}

// Lanes per row of the vector kernels, as a power of two; 0 when they do not apply.
int vector_lanes(const Problem& pr, int interleaved, int bytes) {
  const int64_t E = bytes / type_size(pr.dtype);
  if (pr.D % E != 0 || (!interleaved && (pr.r / 2) % E != 0)) return 0;
  const int64_t n = pr.D / E, hv = pr.r / 2 / E;
  const int64_t units = interleaved ? (n + 1) / 2 : hv + (n - 2 * hv + 1) / 2;
  if (units > 32) return 0;
  int lanes = 4;
  while (lanes < units) lanes *= 2;
  return lanes;
}

int log2_of(int64_t v) {
  int l = 0;
  while ((int64_t{1} << (l + 1)) <= v) ++l;
  return l;
}

// Parts of a token's heads: one, unless the tokens leave warps idle; then a power of two up to `rounds` parts for each
// warp that can be resident.  A part costs the token's angles (and gammas) once more.  No part has less than one row for
// a group.
int32_t slices_for(int64_t tokens, int64_t heads, int64_t groups, int64_t warps, int64_t rounds) {
  const int64_t most = (heads + groups - 1) / groups;
  int64_t slices = 1;
  while (2 * slices <= most && tokens * slices < rounds * warps) slices *= 2;
  return static_cast<int32_t>(slices);
}

size_t vector_smem(const RotaryArgs& a) {
  return (a.norm ? 2 * a.D * sizeof(float) : 0) + static_cast<size_t>(kWarps) * (a.r / 2) * sizeof(float2);
}

// Lanes per row of the vector kernels with vectors of `bytes` for these operands, or 0.
int lanes_for(const RotaryArgs& a, const Problem& pr, int bytes, bool backward) {
  const int64_t E = bytes / type_size(pr.dtype);
  const int lanes = vector_lanes(pr, a.interleaved, bytes);
  for (int w = 0; w < 2; ++w)
    if (pr.H[w] > 0 && !(is_vector_operand(a.x[w], E, bytes) && is_vector_operand(a.y[w], E, bytes) &&
                         (!backward || is_vector_operand(a.dy[w], E, bytes))))
      return 0;
  return lanes;
}

template <typename T, int kBytes>
void launch_fwd_vectors(RotaryArgs a, int lanes, int sms, cudaStream_t st) {
  const int64_t tokens = a.tokens;
  a.log_lanes = log2_of(lanes);
  a.slices = slices_for(tokens, a.heads[0] > a.heads[1] ? a.heads[0] : a.heads[1], 32 / lanes,
                        static_cast<int64_t>(kFwdCtas) * kWarps * sms, 2);
  const int64_t units = tokens * a.slices, most = static_cast<int64_t>(kFwdCtas) * sms;
  const unsigned grid = static_cast<unsigned>(units < most * kWarps ? (units + kWarps - 1) / kWarps : most);
  const size_t smem = vector_smem(a);
  if (a.norm) {
    if (a.interleaved) rotary_fwd_kernel<T, kBytes, true, true><<<grid, kThreads, smem, st>>>(a);
    else rotary_fwd_kernel<T, kBytes, true, false><<<grid, kThreads, smem, st>>>(a);
  } else {
    if (a.interleaved) rotary_fwd_kernel<T, kBytes, false, true><<<grid, kThreads, smem, st>>>(a);
    else rotary_fwd_kernel<T, kBytes, false, false><<<grid, kThreads, smem, st>>>(a);
  }
}

// 16-byte vectors where sizes, strides and alignment allow; 8-byte ones for 16-bit types that only they divide (halves of
// 20 elements of a head of 80, say); else element by element, which reads a row twice and costs four to eight times as much.
template <typename T>
int32_t launch_fwd(RotaryArgs a, const Problem& pr, cudaStream_t st) {
  int sms = 0;
  int32_t rc = aschost::sm_count(&sms);
  if (rc != ASC_OK) return rc;
  int lanes = lanes_for(a, pr, 16, false);
  if (lanes != 0) {
    launch_fwd_vectors<T, 16>(a, lanes, sms, st);
  } else {
    if constexpr (sizeof(T) == 2) {
      lanes = lanes_for(a, pr, 8, false);
      if (lanes != 0) launch_fwd_vectors<T, 8>(a, lanes, sms, st);
    }
    if (lanes == 0) {
      const int64_t tokens = a.tokens, grid = tokens < sms * 8ll ? tokens : sms * 8ll;
      rotary_any_kernel<T, false><<<static_cast<unsigned>(grid), kThreads, a.r / 2 * sizeof(float2), st>>>(a);
    }
  }
  aschost::count_launch();
  ASC_CUDA_TRY(cudaGetLastError());
  return ASC_OK;
}

template <typename T>
int32_t launch_bwd(RotaryArgs a, const Problem& pr, float* dq_gamma, float* dk_gamma, cudaStream_t st) {
  int sms = 0;
  int32_t rc = aschost::sm_count(&sms);
  if (rc != ASC_OK) return rc;
  int bytes = 16, lanes = lanes_for(a, pr, 16, true);
  if (lanes == 0 && sizeof(T) == 2) bytes = 8, lanes = lanes_for(a, pr, 8, true);
  const size_t smem = vector_smem(a) + 2 * (bytes / sizeof(T)) * kThreads * sizeof(float2);
  if (smem > 48 * 1024) lanes = 0;      // 16-bit heads of more than 448: not worth a larger share of the L1 cache
  const int64_t slots = 2ll * sms, H = pr.H[0] + pr.H[1];
  int64_t rows[2];             // rows of partial sums of the gammas, queries' first
  if (lanes != 0) {
    a.log_lanes = log2_of(lanes);
    a.slices = slices_for(a.tokens, H, 32 / lanes, kWarps * slots, 1);
    const int64_t units = static_cast<int64_t>(a.tokens) * a.slices;
    rows[0] = rows[1] = units < slots * kWarps ? (units + kWarps - 1) / kWarps : slots;
  } else {
    // CTAs of queries and of keys in the ratio of their heads, at least one each where there are heads
    for (int w = 0; w < 2; ++w) {
      rows[w] = slots * pr.H[w] / H;
      if (rows[w] == 0 && pr.H[w] > 0) rows[w] = 1;
      if (rows[w] > a.tokens) rows[w] = a.tokens;
    }
  }
  a.q_ctas = static_cast<int32_t>(rows[0]);
  const int64_t n_rows = rows[0] + rows[1], grid = lanes != 0 ? rows[0] : n_rows;
  void* ws = nullptr;
  if (dq_gamma != nullptr || dk_gamma != nullptr) {
    if ((rc = aschost::scratch_alloc(&ws, static_cast<size_t>(n_rows) * a.D * sizeof(float), st)) != ASC_OK) return rc;
    a.partial = static_cast<float*>(ws);
  }
  if (lanes == 0) {
    const size_t any_smem = a.r / 2 * sizeof(float2) + static_cast<size_t>(kWarps) * a.D * sizeof(float);
    rotary_any_kernel<T, true><<<static_cast<unsigned>(grid), kThreads, any_smem, st>>>(a);
  } else {
    const unsigned ctas = static_cast<unsigned>(grid);
    if (bytes == 16) {
      if (a.interleaved) rotary_bwd_kernel<T, 16, true><<<ctas, kThreads, smem, st>>>(a);
      else rotary_bwd_kernel<T, 16, false><<<ctas, kThreads, smem, st>>>(a);
    } else if constexpr (sizeof(T) == 2) {
      if (a.interleaved) rotary_bwd_kernel<T, 8, true><<<ctas, kThreads, smem, st>>>(a);
      else rotary_bwd_kernel<T, 8, false><<<ctas, kThreads, smem, st>>>(a);
    }
  }
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) {
    aschost::count_launch();
    if (ws != nullptr) {
      e = aschost::launch_after(dgamma_kernel, dim3((a.D + 31) / 32, 2), dim3(32 * kSumParts), 0, st, a.partial, a.q_ctas,
                                static_cast<int>(n_rows), a.D, dq_gamma, dk_gamma);
      if (e == cudaSuccess) aschost::count_launch();
    }
  }
  if (ws != nullptr) {
    rc = aschost::scratch_free(ws, st);
    if (e == cudaSuccess && rc != ASC_OK) return rc;
  }
  ASC_CUDA_TRY(e);
  return ASC_OK;
}

}  // namespace

extern "C" int32_t asc_cuda_norm_rotary(const void* q, const void* k, void* q_out, void* k_out, const void* q_gamma,
                                        const void* k_gamma, const void* positions, const double* frequencies,
                                        const int64_t* dims, const int64_t* strides, float eps, float scale,
                                        int32_t dtype, int32_t gamma_dtype, int32_t flags, void* stream) {
  Problem pr;
  bool done;
  const int32_t rc = check(dims, strides, positions, frequencies, dtype, gamma_dtype, flags, pr, &done);
  if (rc != ASC_OK || done) return rc;
  const void* in[2] = {q, k};
  void* out[2] = {q_out, k_out};
  const void* gamma[2] = {q_gamma, k_gamma};
  RotaryArgs a{};
  fill(a, pr, strides + 12, positions, frequencies, eps, scale, gamma_dtype, flags);
  for (int w = 0; w < 2; ++w) {
    if (pr.H[w] == 0) continue;
    if (in[w] == nullptr || out[w] == nullptr) return ASC_ERR_INVALID_ARG;
    if (reinterpret_cast<uintptr_t>(in[w]) % type_size(dtype) != 0 || reinterpret_cast<uintptr_t>(out[w]) % type_size(dtype) != 0)
      return ASC_ERR_MISALIGNED;
    if (a.norm && reinterpret_cast<uintptr_t>(gamma[w]) % type_size(gamma_dtype) != 0) return ASC_ERR_MISALIGNED;
    a.x[w] = operand(in[w], strides + 3 * w, pr, w);
    a.y[w] = operand(out[w], strides + 6 + 3 * w, pr, w);
    a.gamma[w] = gamma[w];
    if (!writes_apart(a.y[w], pr, w)) return ASC_ERR_INVALID_ARG;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == 0) return launch_fwd<__half>(a, pr, st);
  if (dtype == 1) return launch_fwd<__nv_bfloat16>(a, pr, st);
  return launch_fwd<float>(a, pr, st);
}

extern "C" int32_t asc_cuda_norm_rotary_bwd(const void* dq_out, const void* dk_out, const void* q, const void* k, void* dq,
                                            void* dk, const void* q_gamma, const void* k_gamma, float* dq_gamma,
                                            float* dk_gamma, const void* positions, const double* frequencies,
                                            const int64_t* dims, const int64_t* strides, float eps, float scale,
                                            int32_t dtype, int32_t gamma_dtype, int32_t flags, void* stream) {
  Problem pr;
  bool done;
  const int32_t rc = check(dims, strides, positions, frequencies, dtype, gamma_dtype, flags, pr, &done);
  if (rc != ASC_OK) return rc;
  if ((flags & 10) != 2) return ASC_ERR_INVALID_ARG;      // norm, not turned back: see the header
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  float* dgamma[2] = {dq_gamma, dk_gamma};
  for (int w = 0; w < 2; ++w) {                           // a sum over no rows
    if (dgamma[w] == nullptr) continue;
    if (reinterpret_cast<uintptr_t>(dgamma[w]) % 4 != 0) return ASC_ERR_MISALIGNED;
    if (done && pr.D > 0) ASC_CUDA_TRY(cudaMemsetAsync(dgamma[w], 0, pr.D * sizeof(float), st));
  }
  if (done) return ASC_OK;
  const void* g_in[2] = {dq_out, dk_out};
  const void* in[2] = {q, k};
  void* out[2] = {dq, dk};
  const void* gamma[2] = {q_gamma, k_gamma};
  const uintptr_t size = type_size(dtype);
  RotaryArgs a{};
  fill(a, pr, strides + 18, positions, frequencies, eps, scale, gamma_dtype, flags);
  for (int w = 0; w < 2; ++w) {
    if (pr.H[w] == 0) continue;
    if (in[w] == nullptr || out[w] == nullptr || g_in[w] == nullptr) return ASC_ERR_INVALID_ARG;
    if (reinterpret_cast<uintptr_t>(in[w]) % size != 0 || reinterpret_cast<uintptr_t>(out[w]) % size != 0 ||
        reinterpret_cast<uintptr_t>(g_in[w]) % size != 0 ||
        reinterpret_cast<uintptr_t>(gamma[w]) % type_size(gamma_dtype) != 0)
      return ASC_ERR_MISALIGNED;
    a.dy[w] = operand(g_in[w], strides + 3 * w, pr, w);
    a.x[w] = operand(in[w], strides + 6 + 3 * w, pr, w);
    a.y[w] = operand(out[w], strides + 12 + 3 * w, pr, w);
    a.gamma[w] = gamma[w];
    if (!writes_apart(a.y[w], pr, w)) return ASC_ERR_INVALID_ARG;
  }
  if (dtype == 0) return launch_bwd<__half>(a, pr, dgamma[0], dgamma[1], st);
  if (dtype == 1) return launch_bwd<__nv_bfloat16>(a, pr, dgamma[0], dgamma[1], st);
  return launch_bwd<float>(a, pr, dgamma[0], dgamma[1], st);
}
