// Rows on their way into 8 bits: RMS norm, rotation, rounding to bf16, codes.
//
// Rows that a step rounds to bf16 (queries, canvas K and V) are normed and rotated in 64 bits: a score is a sum over one
// row's elements, and an element that a 32-bit intermediate puts on the other side of a rounding border moves every score
// of its row.  Appended rows, which end in 3 mantissa bits, take 32.  Angles are 64-bit, since a 32-bit one is off by up to 0.008 at
// position 131,072; an append looks up the first token's of each run of up to 16 and turns on from there in 32 bits (2^-20 at most).
#pragma once
#include "dg_kv8.cuh"

namespace dg {
namespace kv8 {

template <class T> struct Pair;
template <> struct Pair<float> { typedef float2 type; };
template <> struct Pair<double> { typedef double2 type; };

__device__ __forceinline__ double turns_of(const Rope& r, uint32_t d) {
  return exp2(double(d) * r.log2_step) * 0.15915494309189535;   // 1 / (2 pi)
}
__device__ __forceinline__ double2 unit_at(double position, double turns) {
  const double t = position * turns;
  double2 z;
  sincospi(2.0 * (t - rint(t)), &z.y, &z.x);
  return z;
}
__device__ __forceinline__ double2 cmul(double2 a, double2 b) {
  return make_double2(fma(a.x, b.x, -a.y * b.y), fma(a.x, b.y, a.y * b.x));
}

__device__ __forceinline__ float row_rsqrt(float x) { return rsqrtf(x); }
// one Newton step from the 32-bit root: 1e-13 relative, in a chain of four 64-bit operations
__device__ __forceinline__ double row_rsqrt(double x) {
  const double y = double(rsqrtf(float(x)));
  return fma(0.5 * y, fma(-x * y, y, 1.0), y);
}

// Warp-wide: a head's row, lane l holding elements [8 (l + 32 j), + 8).  RMS norm with weight w (null: unit; norm = false:
// none) and rotation by `tab` (null: none; laid out by angles()); the result as bf16 pairs.
template <class T, int NJ>
__device__ __forceinline__ void row_to_bf16(const uint4 (&raw)[NJ], const __nv_bfloat16* w, bool norm, float eps, const Rope& rope,
                                            const typename Pair<T>::type* tab, uint32_t lane, uint4 (&out)[NJ]) {
  T x[NJ][8];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const uint32_t u[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[j][2 * i] = T(__uint_as_float(u[i] << 16));
      x[j][2 * i + 1] = T(__uint_as_float(u[i] & 0xffff0000u));
    }
  }
  if (norm) {
    T part[4] = {T(0), T(0), T(0), T(0)};
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) part[i & 3] = fma(x[j][i], x[j][i], part[i & 3]);
    T ss = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const T inv = row_rsqrt(ss * T(1.0 / (256.0 * NJ)) + T(eps));
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const uint4 w4 = w ? *reinterpret_cast<const uint4*>(w + 8u * (lane + 32u * j)) : make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
      const uint32_t u[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[j][2 * i] = x[j][2 * i] * inv * T(__uint_as_float(u[i] << 16));
        x[j][2 * i + 1] = x[j][2 * i + 1] * inv * T(__uint_as_float(u[i] & 0xffff0000u));
      }
    }
  }
  if (tab != nullptr && NJ == 2 && rope.dist == 256u) {        // a pair lies in one lane
    const uint32_t hc = rope.half >> 3;
    if (lane < hc) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const typename Pair<T>::type cs = tab[i * hc + lane];
        const T a = x[0][i], b = x[NJ - 1][i];
        x[0][i] = fma(b, -cs.y, a * cs.x);
        x[NJ - 1][i] = fma(a, cs.y, b * cs.x);
      }
    }
  } else if (tab != nullptr && rope.half != 0) {
    // chunks of 8 elements: chunk c < half / 8 pairs with chunk c + dist / 8
    const uint32_t hc = rope.half >> 3, dc = rope.dist >> 3;
    T y[NJ][8];
    uint32_t base[NJ];
    T sign[NJ];
    bool rot[NJ];
    uint32_t src[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const uint32_t c = lane + 32u * j;
      const bool first = c < hc, second = c >= dc && c < dc + hc;
      rot[j] = first || second;
      src[j] = first ? c + dc : (second ? c - dc : c);
      base[j] = first ? c : (second ? c - dc : 0u);
      sign[j] = first ? T(-1) : T(1);
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        T other = __shfl_sync(0xffffffffu, x[0][i], int(src[j] & 31u));
        if (NJ > 1) {
          const T far = __shfl_sync(0xffffffffu, x[NJ - 1][i], int(src[j] & 31u));
          if (src[j] >= 32u) other = far;
        }
        const typename Pair<T>::type cs = tab[i * hc + base[j]];
        y[j][i] = rot[j] ? fma(other, sign[j] * cs.y, x[j][i] * cs.x) : x[j][i];
      }
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) x[j][i] = y[j][i];
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    out[j].x = pack_bf16x2(float(x[j][0]), float(x[j][1]));
    out[j].y = pack_bf16x2(float(x[j][2]), float(x[j][3]));
    out[j].z = pack_bf16x2(float(x[j][4]), float(x[j][5]));
    out[j].w = pack_bf16x2(float(x[j][6]), float(x[j][7]));
  }
}

// The same in 32 bits, by pairs: rows that are appended, whose time is their instructions.  w: the norm's weights as fp32 in
// shared memory (null: unit).  head_dim 512: pairs 256 apart only.
template <int NJ>
__device__ __forceinline__ void row_to_bf16_f32(uint4 (&row)[NJ], const float* w, bool norm, float eps, const Rope& rope, const float2* tab, uint32_t lane) {
  uint64_t x[NJ][4];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    x[j][0] = bf16x2_to_f32x2(row[j].x);
    x[j][1] = bf16x2_to_f32x2(row[j].y);
    x[j][2] = bf16x2_to_f32x2(row[j].z);
    x[j][3] = bf16x2_to_f32x2(row[j].w);
  }
  if (norm) {
    uint64_t s2 = 0ull;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) s2 = fma_f32x2(x[j][i], x[j][i], s2);
    float a, b;
    unpack_f32x2(s2, a, b);
    float ss = a + b;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = rsqrtf(ss * (1.0f / (256.0f * NJ)) + eps);
    const uint64_t inv2 = pack_f32x2(inv, inv);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[j][i] = mul_f32x2(x[j][i], inv2);
      if (w != nullptr) {
        const ulonglong2* w2 = reinterpret_cast<const ulonglong2*>(w + 8u * (lane + 32u * j));
        const ulonglong2 wa = w2[0], wb = w2[1];
        x[j][0] = mul_f32x2(x[j][0], wa.x);
        x[j][1] = mul_f32x2(x[j][1], wa.y);
        x[j][2] = mul_f32x2(x[j][2], wb.x);
        x[j][3] = mul_f32x2(x[j][3], wb.y);
      }
    }
  }
  if (tab != nullptr) {
    const uint32_t hc = rope.half >> 3, dc = rope.dist >> 3;
    if (NJ == 2) {                                             // a pair lies in one lane
      if (lane < hc) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 p = tab[(2 * i) * hc + lane], q = tab[(2 * i + 1) * hc + lane];
          const uint64_t c = pack_f32x2(p.x, q.x), sn = pack_f32x2(p.y, q.y), ng = pack_f32x2(-p.y, -q.y), a = x[0][i], b = x[NJ - 1][i];
          x[0][i] = fma_f32x2(b, ng, mul_f32x2(a, c));
          x[NJ - 1][i] = fma_f32x2(a, sn, mul_f32x2(b, c));
        }
      }
    } else {
      const bool first = lane < hc, second = lane >= dc && lane < dc + hc;
      const uint32_t src = first ? lane + dc : (second ? lane - dc : lane), at = first ? lane : (second ? lane - dc : 0u);
      const float sign = first ? -1.0f : 1.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float a, b;
        unpack_f32x2(x[0][i], a, b);
        const float o0 = __shfl_sync(0xffffffffu, a, int(src)), o1 = __shfl_sync(0xffffffffu, b, int(src));
        const float2 p = tab[(2 * i) * hc + at], q = tab[(2 * i + 1) * hc + at];
        if (first || second) x[0][i] = fma_f32x2(pack_f32x2(o0, o1), pack_f32x2(sign * p.y, sign * q.y), mul_f32x2(x[0][i], pack_f32x2(p.x, q.x)));
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    float a, b;
    unpack_f32x2(x[j][0], a, b);
    row[j].x = pack_bf16x2(a, b);
    unpack_f32x2(x[j][1], a, b);
    row[j].y = pack_bf16x2(a, b);
    unpack_f32x2(x[j][2], a, b);
    row[j].z = pack_bf16x2(a, b);
    unpack_f32x2(x[j][3], a, b);
    row[j].w = pack_bf16x2(a, b);
  }
}

// larger magnitude of each half, as bf16 bits
__device__ __forceinline__ uint32_t abs_max2(uint32_t a, uint32_t b) { return __vmaxu2(a, b & 0x7fff7fffu); }
// a bf16 pair with what is not finite replaced by zero; *bad is set where that happened
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t u, bool* bad) {
  if ((u & 0x7f80u) == 0x7f80u) { u &= 0xffff0000u; *bad = true; }
  if ((u & 0x7f800000u) == 0x7f800000u) { u &= 0xffffu; *bad = true; }
  return u;
}
// a bf16 pair times a power of two (both halves of m): exact
__device__ __forceinline__ uint32_t scale_bf16x2(uint32_t v, uint32_t m) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(m));
  return r;
}
// eight bf16 times 2^-e, given as a bf16 pair, as e4m3 codes
__device__ __forceinline__ uint2 code8_fast(const uint4& v, uint32_t m) {
  const uint32_t u[4] = {scale_bf16x2(v.x, m), scale_bf16x2(v.y, m), scale_bf16x2(v.z, m), scale_bf16x2(v.w, m)};
  uint16_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = e4m3x2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
  return make_uint2(uint32_t(h[0]) | (uint32_t(h[1]) << 16), uint32_t(h[2]) | (uint32_t(h[3]) << 16));
}
// eight bf16 times 2^-e as e4m3 codes, and the codes of what that rounding left
__device__ __forceinline__ uint2 code8(const uint4& v, float mul, uint2* rest) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
  uint16_t h[4], r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = __uint_as_float(u[i] << 16) * mul, b = __uint_as_float(u[i] & 0xffff0000u) * mul;
    h[i] = e4m3x2(a, b);
    if (rest) {
      const float2 f = f32x2_from_e4m3x2(h[i]);
      r[i] = e4m3x2(a - f.x, b - f.y);
    }
  }
  if (rest) *rest = make_uint2(uint32_t(r[0]) | (uint32_t(r[1]) << 16), uint32_t(r[2]) | (uint32_t(r[3]) << 16));
  return make_uint2(uint32_t(h[0]) | (uint32_t(h[1]) << 16), uint32_t(h[2]) | (uint32_t(h[3]) << 16));
}
// where the eight codes of chunk c (8 elements) of row r lie in a block of 128 rows
__device__ __forceinline__ uint32_t code8_off(uint32_t r, uint32_t c) {
  return (c >> 4) * SLAB + chunk_off(r, (c & 15u) >> 1) + (c & 1u) * 8u;
}

// (cos, sin) of n_tok tokens from `first` on: tab[token][8][half / 8], pair d at [d % 8][d / 8], so that the lanes of a
// warp, eight pairs each, read neighbours.  A thread's tokens follow one another: two look-ups of
// an angle, the others by rotation (64 bits: 1e-15 after a block).  Groups of half threads of THREADS; every thread of the CTA calls.
template <class T, uint32_t THREADS>
__device__ __forceinline__ void angles(const Rope& r, double first, uint32_t n_tok, typename Pair<T>::type* tab) {
  const uint32_t groups = THREADS / r.half, per = (n_tok + groups - 1u) / groups;
  const uint32_t d = threadIdx.x % r.half, t0 = threadIdx.x / r.half * per;
  if (threadIdx.x >= groups * r.half || t0 >= n_tok) return;
  const double turns = turns_of(r, d);
  double2 z = unit_at(first + double(t0), turns), one = make_double2(1.0, 0.0);
  if (per > 1u) one = unit_at(1.0, turns);
  for (uint32_t j = 0; j < per && t0 + j < n_tok; ++j) {
    typename Pair<T>::type o;
    o.x = T(z.x);
    o.y = T(z.y);
    tab[(t0 + j) * r.half + (d & 7u) * (r.half >> 3) + (d >> 3)] = o;
    z = cmul(z, one);
  }
}

__device__ __forceinline__ float max_of_halves(uint32_t two) {
  return fmaxf(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
}

}  // namespace kv8
}  // namespace dg
