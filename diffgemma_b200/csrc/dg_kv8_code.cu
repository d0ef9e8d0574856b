// Everything that enters or leaves 8 bits: the rows of a step (queries in two terms, canvas K and V in two terms), tokens
// appended to a cache, rows read back.
//
// Rows that a step rounds to bf16 (queries, canvas K and V) are normed and rotated in 64 bits: a score is a sum over one
// row's elements, and an element that a 32-bit intermediate puts on the other side of a rounding border moves every score
// of its row.  Appended rows, which end in 3 mantissa bits, take 32.  Angles are in 64 bits everywhere: at position 131,072
// a 32-bit angle is off by up to 0.008.
#include "dg_kv8.cuh"

namespace dg {
namespace kv8 {

constexpr uint32_t CT = 512;                  // threads: 16 warps
constexpr uint32_t PASS = 16;                 // tokens whose angles are in shared memory at a time, one for each warp

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
__device__ __forceinline__ double row_rsqrt(double x) { return rsqrt(x); }

// Warp-wide: a head's row, lane l holding elements [8 (l + 32 j), + 8).  RMS norm with weight w (null: unit; norm = false:
// none) and rotation by `tab` (null: none); the result as bf16 pairs.
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
    T ss = T(0);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fma(x[j][i], x[j][i], ss);
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
  if (tab != nullptr && rope.half != 0) {
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
      base[j] = 8u * (first ? c : (second ? c - dc : 0u));
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
        const typename Pair<T>::type cs = tab[base[j] + i];
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

// larger magnitude of each half, as bf16 bits
__device__ __forceinline__ uint32_t abs_max2(uint32_t a, uint32_t b) { return __vmaxu2(a, b & 0x7fff7fffu); }
// a bf16 pair with what is not finite replaced by zero; *bad is set where that happened
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t u, bool* bad) {
  if ((u & 0x7f80u) == 0x7f80u) { u &= 0xffff0000u; *bad = true; }
  if ((u & 0x7f800000u) == 0x7f800000u) { u &= 0xffffu; *bad = true; }
  return u;
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

struct PosList {
  uint64_t pos[MAX_SEQ];
};

// (cos, sin) of PASS tokens from `first` on: tab[token][half].  The angles of a thread's tokens are reached by rotation
// (64 bits: 1e-15 after a block), one table look-up of three angles for a block.
template <class T>
struct Angles {
  double2 z, one, pass;
  uint32_t d, g, per;
  bool on;
  __device__ __forceinline__ void start(const Rope& r, double first) {
    const uint32_t groups = r.half ? CT / r.half : 1u;
    per = (PASS + groups - 1u) / groups;
    d = r.half ? threadIdx.x % r.half : 0u;
    g = r.half ? threadIdx.x / r.half : 0u;
    on = r.half != 0u && g < groups && g * per < PASS;
    if (on) {
      const double t = turns_of(r, d);
      z = unit_at(first + double(g * per), t);
      one = unit_at(1.0, t);
      pass = unit_at(double(PASS), t);
    }
  }
  __device__ __forceinline__ void fill(const Rope& r, typename Pair<T>::type* tab) {
    if (!on) return;
    double2 c = z;
    for (uint32_t j = 0; j < per && g * per + j < PASS; ++j) {
      typename Pair<T>::type o;
      o.x = T(c.x);
      o.y = T(c.y);
      tab[(g * per + j) * r.half + d] = o;
      c = cmul(c, one);
    }
    z = cmul(z, pass);
  }
};

// The rows of one block of 128 tokens of one head, K or V: in registers as bf16, 8 rows a warp (row = 16 pass + warp).
// row(r) says where row r comes from.  Returns the largest magnitude of the block.
template <class T, int NJ, class Row>
__device__ __forceinline__ float block_rows(const CodeParams& p, bool is_k, double first_pos, uint32_t n_rows, Row row, uint4 (&held)[8][NJ],
                                            uint8_t* smem, float* red, bool* bad) {
  typedef typename Pair<T>::type T2;
  T2* tab = reinterpret_cast<T2*>(smem);
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const bool turn = is_k && !p.ready && p.rope.half != 0;
  const bool norm = !p.ready && (is_k || p.v_norm);
  Angles<T> ang;
  if (turn) ang.start(p.rope, first_pos);
  uint32_t top = 0;
#pragma unroll
  for (uint32_t s = 0; s < 8; ++s) {
    uint4 raw[NJ];
    const uint32_t r = s * PASS + warp;
    const bool live = r < n_rows;
    bool fresh = false;
    if (live) fresh = row(r, raw);
    if (s * PASS < n_rows && turn) {
      __syncthreads();
      ang.fill(p.rope, tab);
      __syncthreads();
    }
    if (!live) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) held[s][j] = make_uint4(0u, 0u, 0u, 0u);
      continue;
    }
    if (fresh) {
      if (turn || norm)
        row_to_bf16<T, NJ>(raw, is_k ? p.kw : nullptr, norm, p.eps, p.rope, turn ? tab + warp * p.rope.half : nullptr, lane, held[s]);
      else {
#pragma unroll
        for (int j = 0; j < NJ; ++j) held[s][j] = raw[j];
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        uint4& h = held[s][j];
        h = make_uint4(finite_or_zero(h.x, bad), finite_or_zero(h.y, bad), finite_or_zero(h.z, bad), finite_or_zero(h.w, bad));
      }
    } else {
#pragma unroll
      for (int j = 0; j < NJ; ++j) held[s][j] = raw[j];
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) top = abs_max2(abs_max2(abs_max2(abs_max2(top, held[s][j].x), held[s][j].y), held[s][j].z), held[s][j].w);
  }
  float t = fmaxf(__uint_as_float(top << 16), __uint_as_float(top & 0xffff0000u));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
  __syncthreads();
  if (lane == 0) red[warp] = t;
  __syncthreads();
  t = red[lane & 15u];
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
  return t;
}

// ------------------------------------------------------------------------------------------- rows of a step
// CTAs [0, canvas CTAs): (sequence, head, tile of 128 canvas tokens, K or V).  The others: one canvas token each, all its
// query heads (the angles are computed once for all of them), and the rows behind the last token of a row tile as zeros.
template <int NJ>
__global__ void __launch_bounds__(CT, 1) dg_kv8_rows_kernel(const __grid_constant__ QueryParams q, const __grid_constant__ CodeParams p,
                                                            const __grid_constant__ PosList pos, uint32_t canvas_ctas, uint32_t q_tokens) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float red[16];
  grid_launch_dependents();
  grid_wait();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  constexpr uint32_t D = 256u * NJ;
  if (blockIdx.x < canvas_ctas) {
    uint32_t x = blockIdx.x;
    const bool is_k = (x & 1u) == 0u;
    x >>= 1;
    const uint32_t ct = x % p.n_ctiles;
    x /= p.n_ctiles;
    const uint32_t h = x % p.Hkv, b = x / p.Hkv;
    const uint32_t t0 = ct * BLK, n_rows = p.n - t0 < BLK ? p.n - t0 : BLK;
    const __nv_bfloat16* src = (is_k ? p.k : p.v) + (size_t(b) * p.n + t0) * p.Hkv * D + size_t(h) * D;
    uint4 held[8][NJ];
    bool bad = false;
    const float top = block_rows<double, NJ>(
        p, is_k, double(pos.pos[b]) + double(t0), n_rows,
        [&](uint32_t r, uint4 (&raw)[NJ]) {
#pragma unroll
          for (int j = 0; j < NJ; ++j) raw[j] = *reinterpret_cast<const uint4*>(src + size_t(r) * p.Hkv * D + 8u * (lane + 32u * j));
          return true;
        },
        held, smem, red, &bad);
    const int e = scale_exp(top);
    const float mul = pow2i(-e);
    const size_t tile = (size_t(b) * p.Hkv + h) * p.n_ctiles + ct;
    uint8_t* dst = (is_k ? p.k_codes : p.v_codes) + tile * 2u * BLK * D;
#pragma unroll
    for (uint32_t s = 0; s < 8; ++s)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const uint32_t off = code8_off(s * PASS + warp, lane + 32u * j);
        uint2 rest;
        const uint2 c = code8(held[s][j], mul, &rest);
        *reinterpret_cast<uint2*>(dst + off) = c;
        *reinterpret_cast<uint2*>(dst + BLK * D + off) = rest;
      }
    if (threadIdx.x == 0) (is_k ? p.k_exp : p.v_exp)[tile] = e;
    if (bad) dev_status_set(p.status, DG_DEV_NOT_FINITE, KID_CODE, blockIdx.x, t0);
    return;
  }
  const uint32_t x = blockIdx.x - canvas_ctas;
  const uint32_t b = x / q_tokens, i = x % q_tokens;
  const QueryRows& o = q.rows;
  double2* tab = reinterpret_cast<double2*>(smem);
  if (!q.prenormed && i < o.C && threadIdx.x < q.rope.half)
    tab[threadIdx.x] = unit_at(double(pos.pos[b]) + double(i), turns_of(q.rope, threadIdx.x));
  __syncthreads();
  for (uint32_t h = warp; h < o.Hq; h += CT / 32u) {
    const uint32_t kvh = h / o.G, R = i * o.G + h % o.G;
    if (R >= o.MT * BLK) continue;
    uint4 v[NJ];
    const bool live = i < o.C;
    if (live) {
      const size_t at = ((size_t(b) * o.C + i) * o.Hq + h) * D + 8u * lane;
      uint4 raw[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) raw[j] = *reinterpret_cast<const uint4*>(q.q + at + 256u * j);
      if (q.prenormed) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) v[j] = raw[j];
      } else {
        row_to_bf16<double, NJ>(raw, q.qw, true, q.eps, q.rope, q.rope.half ? tab : nullptr, lane, v);
      }
      if (q.q_rot) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) *reinterpret_cast<uint4*>(q.q_rot + at + 256u * j) = v[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < NJ; ++j) v[j] = make_uint4(0u, 0u, 0u, 0u);
    }
    uint32_t top2 = 0;
#pragma unroll
    for (int j = 0; j < NJ; ++j) top2 = abs_max2(abs_max2(abs_max2(abs_max2(top2, v[j].x), v[j].y), v[j].z), v[j].w);
    uint32_t top = top2 > 0xffffu && (top2 >> 16) > (top2 & 0xffffu) ? top2 >> 16 : top2 & 0xffffu;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, top, m);
      top = other > top ? other : top;
    }
    // a row that is not finite has no scores: its codes are NaN
    const bool fin = top < 0x7f80u;
    const int e = fin ? scale_exp(__uint_as_float(top << 16)) : 0;
    const float mul = fin ? pow2i(-e) : __uint_as_float(0x7fc00000u);
    uint8_t* dst = o.codes + ((size_t(b) * o.Hkv + kvh) * o.MT + R / BLK) * 2u * BLK * D;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const uint32_t off = code8_off(R % BLK, lane + 32u * j);
      uint2 rest;
      const uint2 c = code8(v[j], mul, &rest);
      *reinterpret_cast<uint2*>(dst + off) = c;
      *reinterpret_cast<uint2*>(dst + BLK * D + off) = rest;
    }
    if (lane == 0) {
      // -log2 e * lse; rows without a sum (none, or behind the last token) draw nothing
      float nl = -INFINITY;
      if (live && q.lse != nullptr) {
        const float l = q.lse[(size_t(b) * o.C + i) * o.Hq + h];
        nl = l == -INFINITY ? -INFINITY : -1.4426950408889634f * l;
      }
      o.row[(size_t(b) * o.Hkv + kvh) * o.MT * BLK + R] = make_float2(q.scale_log2 * pow2i(e), nl);
    }
  }
}

// ------------------------------------------------------------------------------------------- append
// One CTA for each (block, head, K or V) that the new tokens touch.  The first block may hold tokens already: their values
// are read, and the block is coded as a whole at the scale that all of it needs.
template <int NJ>
__global__ void __launch_bounds__(CT, 1) dg_kv8_append_kernel(const __grid_constant__ CodeParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float red[16];
  grid_launch_dependents();
  grid_wait();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  constexpr uint32_t D = 256u * NJ;
  uint32_t x = blockIdx.x;
  const bool is_k = (x & 1u) == 0u;
  x >>= 1;
  const uint32_t h = x % p.Hkv, blk = p.n_keys / BLK + x / p.Hkv;
  const uint32_t t0 = blk * BLK, end = p.n_keys + p.n;
  const uint32_t kept = p.n_keys > t0 ? p.n_keys - t0 : 0u;
  const uint32_t n_rows = end - t0 < BLK ? end - t0 : BLK;
  uint8_t* codes = (is_k ? p.k_codes : p.v_codes) + (size_t(h) * p.blocks + blk) * BLK * D;
  int32_t* exps = (is_k ? p.k_exp : p.v_exp) + size_t(h) * p.blocks + blk;
  const float old = kept ? pow2i(*exps) : 1.0f;
  const __nv_bfloat16* src = is_k ? p.k : p.v;
  uint4 held[8][NJ];
  bool bad = false;
  const float top = block_rows<float, NJ>(
      p, is_k, double(p.pos) + double(t0) - double(p.n_keys), n_rows,
      [&](uint32_t r, uint4 (&raw)[NJ]) {
        if (r >= kept) {
          const __nv_bfloat16* s = src + (size_t(t0 + r - p.n_keys) * p.Hkv + h) * D;
#pragma unroll
          for (int j = 0; j < NJ; ++j) raw[j] = *reinterpret_cast<const uint4*>(s + 8u * (lane + 32u * j));
          return true;
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const uint2 c = *reinterpret_cast<const uint2*>(codes + code8_off(r, lane + 32u * j));
          const float2 a = f32x2_from_e4m3x2(uint16_t(c.x)), b = f32x2_from_e4m3x2(uint16_t(c.x >> 16));
          const float2 f = f32x2_from_e4m3x2(uint16_t(c.y)), g = f32x2_from_e4m3x2(uint16_t(c.y >> 16));
          raw[j] = make_uint4(pack_bf16x2(a.x * old, a.y * old), pack_bf16x2(b.x * old, b.y * old),
                              pack_bf16x2(f.x * old, f.y * old), pack_bf16x2(g.x * old, g.y * old));
        }
        return false;
      },
      held, smem, red, &bad);
  const int e = scale_exp(top);
  const float mul = pow2i(-e);
#pragma unroll
  for (uint32_t s = 0; s < 8; ++s) {
    const uint32_t r = s * PASS + warp;
    if (r >= n_rows) continue;
#pragma unroll
    for (int j = 0; j < NJ; ++j) *reinterpret_cast<uint2*>(codes + code8_off(r, lane + 32u * j)) = code8(held[s][j], mul, nullptr);
  }
  if (threadIdx.x == 0) *exps = e;
  if (bad) dev_status_set(p.status, DG_DEV_NOT_FINITE, KID_CODE, blockIdx.x, t0);
}

// ------------------------------------------------------------------------------------------- read back
// A thread takes 16 codes (one swizzled chunk) to 32 bytes of bf16; a warp's stores cover whole rows.
__global__ void __launch_bounds__(256) dg_kv8_read_kernel(const __grid_constant__ ReadParams p) {
  grid_launch_dependents();
  grid_wait();
  const uint32_t per_row = p.D / 16u;
  const uint64_t n = uint64_t(p.n) * p.Hkv * per_row;
  for (uint64_t x = uint64_t(blockIdx.x) * 256u + threadIdx.x; x < 2u * n; x += uint64_t(gridDim.x) * 256u) {
    const bool is_k = x < n;
    const uint64_t y = is_k ? x : x - n;
    const uint32_t c = uint32_t(y % per_row);
    const uint64_t row = y / per_row;
    const uint32_t h = uint32_t(row % p.Hkv), slot = p.slot0 + uint32_t(row / p.Hkv);
    const size_t blk = size_t(h) * p.blocks + slot / BLK;
    const uint8_t* src = (is_k ? p.k : p.v) + blk * BLK * p.D + (c >> 3) * SLAB + chunk_off(slot % BLK, c & 7u);
    const float mul = pow2i((is_k ? p.k_exp : p.v_exp)[blk]);
    const uint4 v = *reinterpret_cast<const uint4*>(src);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = f32x2_from_e4m3x2(uint16_t(u[i])), b = f32x2_from_e4m3x2(uint16_t(u[i] >> 16));
      o[2 * i] = pack_bf16x2(a.x * mul, a.y * mul);
      o[2 * i + 1] = pack_bf16x2(b.x * mul, b.y * mul);
    }
    uint4* dst = reinterpret_cast<uint4*>((is_k ? p.k_out : p.v_out) + row * p.D + c * 16u);
    dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

// ------------------------------------------------------------------------------------------- launches
template <class... A>
static cudaError_t launch(void (*fn)(A...), uint32_t grid, uint32_t threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fn, args...);
}

constexpr size_t ROWS_SMEM = PASS * 256u * sizeof(double2);   // angles of PASS tokens at the widest rotation

cudaError_t configure_code() {
  cudaError_t e = cudaSuccess;
  for (const void* f : {reinterpret_cast<const void*>(dg_kv8_rows_kernel<1>), reinterpret_cast<const void*>(dg_kv8_rows_kernel<2>)})
    if (e == cudaSuccess) e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, int(ROWS_SMEM));
  return e;
}

cudaError_t launch_rows(const QueryParams& q, const CodeParams& p, const uint64_t* pos, uint32_t n_seq, cudaStream_t st) {
  PosList l = {};
  for (uint32_t b = 0; b < n_seq; ++b) l.pos[b] = pos[b];
  const uint32_t canvas = n_seq * p.n_ctiles * q.rows.Hkv * 2u;
  const uint32_t tokens = (q.rows.MT * BLK + q.rows.G - 1u) / q.rows.G;
  const size_t smem = size_t(canvas ? PASS : 1u) * q.rope.half * sizeof(double2);
  return launch(q.rows.D == 256 ? dg_kv8_rows_kernel<1> : dg_kv8_rows_kernel<2>, canvas + n_seq * tokens, CT, smem, st, q, p, l, canvas, tokens);
}

cudaError_t launch_append(const CodeParams& p, cudaStream_t st) {
  const uint32_t blocks = (p.n_keys + p.n + BLK - 1u) / BLK - p.n_keys / BLK;
  const size_t smem = p.ready ? 0 : size_t(PASS) * p.rope.half * sizeof(float2);
  return launch(p.D == 256 ? dg_kv8_append_kernel<1> : dg_kv8_append_kernel<2>, blocks * p.Hkv * 2u, CT, smem, st, p);
}

cudaError_t launch_read(const ReadParams& p, cudaStream_t st) {
  const uint64_t n = 2ull * p.n * p.Hkv * (p.D / 16u);
  const uint64_t ctas = (n + 255u) / 256u;
  return launch(dg_kv8_read_kernel, uint32_t(ctas < 148u * 64u ? ctas : 148u * 64u), 256, 0, st, p);
}

}  // namespace kv8
}  // namespace dg
