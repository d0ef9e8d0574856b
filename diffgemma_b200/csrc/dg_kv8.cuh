// A prefix cache held in 8 bits: format, launch parameters and the pieces that its kernels share.
//
// Per KV head, K and V are e4m3 codes with one power-of-two scale for each block of 128 tokens:
//   value = code * 2^e,   e = min { e in [-60, 60] : largest magnitude of the block <= 448 * 2^e }
// A power of two costs e4m3 nothing (a code keeps its three mantissa bits at any scale) and makes everything but the
// rounding of a code exact: coding a block again, moving a row to a block of another scale, folding a scale into a score.
//
// Memory is what the tensor cores read: a block is D / 128 slabs of [128 tokens][128 bytes], 16-byte chunks swizzled by
// token & 7 (the 128-byte swizzle of the UMMA descriptors), K as a K-major and V as an MN-major operand.  32 KB of a block
// are one contiguous bulk copy; no tensor map is needed, so a launch over many caches carries two pointers for each.
//
// Scores and outputs as exact as the bf16 kernels': the operand that is not in the cache is split into 8-bit terms,
// q = q1 + q2 (e4m3 each, scaled by a power of two for each row; a bf16 number within 2^9.8 of its row's largest is exactly
// such a sum) and p = p1 + p2 + p3 (e5m2: 2^-11 of a weight down to 2^-18 of its row's largest).  kind::f8f6f4 runs at twice the bf16
// rate, so a product takes one pass over a bf16 cache for Q and one and a half for P, and no code is ever converted on its way to the
// tensor cores.
#pragma once
#include "dg_common.cuh"
#include "sm100_ptx.cuh"

namespace dg {
namespace kv8 {

constexpr uint32_t BLK = 128;                  // tokens of a block
constexpr uint32_t SLAB = BLK * 128;           // bytes of a slab: 128 tokens x 128 dims
constexpr uint32_t UNIT = 2 * SLAB;            // what one bulk copy brings: 128 tokens x 256 dims
constexpr int EXP_MIN = -60, EXP_MAX = 60;     // sums of scales of one row stay inside fp32
constexpr float LIFT = 12.0f;                  // weights, and partial rows, stand at 2^LIFT times their reference
constexpr uint32_t TERMS = 3;                  // e5m2 terms of a weight
constexpr uint32_t MAX_SEQ = 64;               // caches served by one launch

enum : uint32_t { KID_CODE = 16, KID_ATTN = 17, KID_WEIGHTS = 18, KID_EVICT = 19, KID_TOKEN = 20 };

// byte offset of 16-byte chunk c (of 8 per slab) of token r in a slab
__host__ __device__ __forceinline__ uint32_t chunk_off(uint32_t r, uint32_t c) { return r * 128u + ((c ^ (r & 7u)) << 4); }

__host__ __device__ __forceinline__ float pow2i(int e) {   // 2^e, e in [-126, 127]
#ifdef __CUDA_ARCH__
  return __int_as_float((e + 127) << 23);
#else
  const uint32_t u = uint32_t(e + 127) << 23;
  float f;
  __builtin_memcpy(&f, &u, 4);
  return f;
#endif
}
// scale exponent of a block whose largest magnitude is `top` (finite)
__device__ __forceinline__ int scale_exp(float top) {
  const uint32_t u = __float_as_uint(top);
  const int x = int(u >> 23) - 127;                              // top = m 2^x, m in [1, 2); 448 = 1.75 * 2^8
  const int e = x - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < EXP_MIN ? EXP_MIN : (e > EXP_MAX ? EXP_MAX : e);
}
// two fp32 -> two e4m3 codes (nearest even), lo in the low byte; out of range saturates, NaN stays NaN
__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// bytes 0 and 1 (HIGH: 2 and 3) of four e5m2 numbers as f16: e5m2 is the upper byte of an f16.  A byte permutation, where the conversion
// would wait for the unit that the exponentials need.
template <bool HIGH>
__device__ __forceinline__ uint32_t f16x2_from_e5m2(uint32_t v) { return __byte_perm(v, 0u, HIGH ? 0x3424u : 0x1404u); }
__device__ __forceinline__ uint32_t f16x2_from_e4m3x2(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}
__device__ __forceinline__ float2 f32x2_from_e4m3x2(uint16_t v) { return unpack_f16x2(f16x2_from_e4m3x2(v)); }
// Four fp32 (a in the low byte) to e5m2 with the bits of `r` added below the last kept one: a half for each of the four, which
// rounds to nearest (ties away from zero).  Two of the four take their bits mirrored.  One instruction for four numbers, where
// conversions by pairs are two each and a byte permutation.
constexpr uint32_t RS_HALF = 0x80018001u;
__device__ __forceinline__ uint32_t e5m2x4_half(float a, float b, float c, float d) {
  uint32_t r;
  asm("cvt.rs.satfinite.e5m2x4.f32 %0, {%4, %3, %2, %1}, %5;" : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d), "r"(RS_HALF));
  return r;
}
// x - h of an fp32 and an f16 number, in fp32
__device__ __forceinline__ float sub_f32_f16(float x, uint16_t h) {
  float r;
  asm("{\n\t.reg .b16 m;\n\tmov.b16 m, 0xBC00;\n\tfma.rn.f32.f16 %0, %1, m, %2;\n\t}" : "=f"(r) : "h"(h), "f"(x));
  return r;
}
// Four weights as three e5m2 terms.  Three significant bits leave 2^-3 of a weight's power of two, a number of the format or less, so
// that the next term starts four powers down: 2^-11 of a weight is left, and never less than 2^-17 (half the smallest step)
__device__ __forceinline__ void split4_e5m2(float a, float b, float c, float d, uint32_t (&t)[TERMS]) {
  float x[4] = {a, b, c, d};
#pragma unroll
  for (uint32_t i = 0; i < TERMS; ++i) {
    t[i] = e5m2x4_half(x[0], x[1], x[2], x[3]);
    if (i + 1 == TERMS) break;
    const uint32_t lo = f16x2_from_e5m2<false>(t[i]), hi = f16x2_from_e5m2<true>(t[i]);
    x[0] = sub_f32_f16(x[0], uint16_t(lo));
    x[1] = sub_f32_f16(x[1], uint16_t(lo >> 16));
    x[2] = sub_f32_f16(x[2], uint16_t(hi));
    x[3] = sub_f32_f16(x[3], uint16_t(hi >> 16));
  }
}

// ---- tensor cores: kind::f8f6f4, fp32 accumulate.  A e4m3 (0) or e5m2 (1), B e4m3; other fields as for bf16.
__host__ __device__ constexpr uint32_t idesc_f8(uint32_t m, uint32_t n, uint32_t a_e5m2, uint32_t b_mn_major) {
  return (1u << 4) | (a_e5m2 << 7) | (b_mn_major << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n"
      :
      : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t"
      "}\n"
      :
      : "r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// the same by the leader of a CTA pair, over both CTAs' operands
__device__ __forceinline__ void mma_ss_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n"
      :
      : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts_pair(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t"
      "}\n"
      :
      : "r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// all prior MMAs of this thread arrive once on the barrier at this offset of both CTAs of the pair
__device__ __forceinline__ void commit_both(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(uint16_t(3)) : "memory");
}
// contiguous copy global -> this CTA's shared memory, counted on a local barrier; both 16-byte aligned, bytes a multiple of 16
__device__ __forceinline__ void bulk_load(uint32_t smem_dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_dst),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
               : "memory");
}
// mbar_wait with its clock and the abort flag looked at every 64th poll only: a waiting warp shares its scheduler with warps that
// compute, and a poll alone is a third of the instructions.
// CLUSTER: arrivals may come from the pair's other CTA.
template <bool CLUSTER = false>
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag) {
  auto there = [&] { return CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity); };
  if (there()) return true;
  const long long t0 = clock64();
#pragma unroll 1
  for (uint32_t it = 1;; ++it) {
    if (there()) return true;
    if ((it & 63u) == 0u) {
      if (*abort_flag) return false;
      if (clock64() - t0 > DG_WAIT_LIMIT_CYCLES) {
        *abort_flag = 1u;
        return false;
      }
    }
  }
}
__device__ __forceinline__ void grid_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- launch parameters
struct Rope {
  uint32_t half, dist;       // rotated pairs (d, d + dist), d < half; both multiples of 8
  double log2_step;          // log2 of the ratio of neighbouring frequencies: -2 / head_dim * log2(theta)
};

// rows of canvas queries, coded: [seq][KV head][row tile of 128][term][slab][128 rows][128 B], and per row what its scores
// are multiplied by (scale * log2 e * 2^row exponent) and, for the key weights, -log2 e * lse (there as pairs of rows: two
// factors, then two sums)
struct QueryRows {
  uint8_t* codes;
  float2* row;
  uint32_t C, Hq, Hkv, G, D, MT;   // MT row tiles of each KV head
};

struct QueryParams {
  QueryRows rows;
  const __nv_bfloat16* q;      // [seq][C][Hq][D]
  const __nv_bfloat16* qw;     // [D] or null
  const float* lse;            // [C][Hq] or null
  __nv_bfloat16* q_rot;        // normed and rotated Q as bf16, or null
  DevStatus* status;           // rows that are not finite are reported here (key weights)
  uint32_t prenormed;          // 1: q is normed and rotated already
  float eps, scale_log2;
  Rope rope;
};

// K and V rows that enter 8 bits: the canvas (two terms, coded by itself) or tokens behind a cache's first n_keys
struct CodeParams {
  const __nv_bfloat16* k;      // [seq][n][Hkv][D]
  const __nv_bfloat16* v;
  const __nv_bfloat16* kw;     // [D] or null
  uint32_t n, Hkv, D;
  uint32_t ready;              // 1: rows are stored as they are (no norm, no rotation)
  uint32_t v_norm;
  float eps;
  Rope rope;
  DevStatus* status;
  // append: codes [Hkv][blocks][D / 128][128][128], exponents [Hkv][blocks][2] (K, V)
  uint8_t* k_codes;
  uint8_t* v_codes;
  int32_t* exps;
  uint32_t blocks, n_keys;
  uint64_t pos;
  // canvas: codes [seq][Hkv][tiles][2 terms][D / 128][128][128], exponents [seq][Hkv][tiles][2]
  uint32_t n_ctiles;
};

struct Seq {                   // one cache of an attention launch
  const uint8_t* k;
  const uint8_t* v;
  const int2* exps;
  uint32_t blocks;             // capacity in blocks: stride of a head
  uint32_t n_keys;
  uint32_t first_cta;          // CTAs of the sequences before it
  uint32_t n_splits;
};

struct AttnParams8 {
  Seq seq[MAX_SEQ];
  uint32_t n_seq, C, Hq, Hkv, G, D, MT;
  uint32_t include_canvas;
  uint32_t mode, windowed, wm1;
  const uint8_t* q_codes;
  const float2* q_row;
  const uint8_t* c_k;          // canvas codes
  const uint8_t* c_v;
  const int2* c_exps;
  uint32_t n_ctiles;
  __nv_bfloat16* out;          // [seq][C][Hq][D]
  float* lse;                  // [seq][C][Hq] or null
  float* ws_o;                 // split partials [slot][128][256], slot: sequence's first CTA + ((split * Hkv + head) * MT + row tile) * D / 256 + half
  float2* ws_ml;               // [slot][128]
  DevStatus* status;
};

// few query rows: the queries, and up to TOKEN_CANVAS canvas keys, raw
constexpr uint32_t TOKEN_ROWS = 16, TOKEN_CANVAS = 8;
struct TokenParams {
  Seq seq[MAX_SEQ];
  uint64_t pos[MAX_SEQ];
  uint32_t n_seq, C, Hq, Hkv, G, D;
  uint32_t mode, windowed, wm1, v_norm;
  const __nv_bfloat16* q;      // [seq][C][Hq][D]
  const __nv_bfloat16* k;      // [seq][C][Hkv][D], or null: the cached keys alone
  const __nv_bfloat16* v;
  const __nv_bfloat16* qw;
  const __nv_bfloat16* kw;
  __nv_bfloat16* q_rot;
  __nv_bfloat16* out;
  float* lse;
  float* ws_o;                 // split partials [CTA][D / 256][128][256]
  float2* ws_ml;
  DevStatus* status;
  float eps, scale_log2;
  Rope rope;
};

struct WeightParams {
  const uint8_t* q_codes;
  const float2* q_row;
  const uint8_t* k;
  const int2* exps;
  uint32_t blocks, n_keys;
  uint32_t C, Hkv, G, MT;
  uint32_t mode, windowed, wm1;
  uint32_t run0;               // the first run of keys that some row sees
  float* w;                    // [Hkv][ld]
  uint64_t ld;
  float decay;
  float* part;                 // [piece][Hkv][n_keys] where CTAs share runs of keys, else null
  DevStatus* status;
};

struct EvictParams {
  const float* w;              // [Hkv][ld]
  uint64_t ld;
  uint32_t n_keys, n_keep, n_recent, Hkv, D;
  int32_t* kept;               // [Hkv][n_keep]
  float* w_out;                // [Hkv][ld_out] or null
  uint64_t ld_out;
  const uint8_t* k;
  const uint8_t* v;
  const int32_t* exps;
  uint32_t blocks;
  uint8_t* to_k;
  uint8_t* to_v;
  int32_t* to_exps;
  uint32_t to_blocks;
};

struct ReadParams {
  const uint8_t* k;
  const uint8_t* v;
  const int32_t* exps;
  uint32_t blocks, Hkv, D, slot0, n;
  __nv_bfloat16* k_out;        // [n][Hkv][D]
  __nv_bfloat16* v_out;
};

__host__ __device__ __forceinline__ MaskParams seq_mask(const AttnParams8& p, uint32_t n_keys) {
  MaskParams m;
  m.kv_len = n_keys;
  m.t0 = 0;
  m.pre_hi = n_keys;
  m.can_hi = p.include_canvas ? n_keys + p.C : n_keys;
  m.mode = p.mode;
  m.windowed = p.windowed;
  m.wm1 = p.wm1;
  m.pad_ = 0;
  return m;
}
// Key tiles of canvas rows [row_first, row_last]: cached blocks [a0, a0 + nA), then nB tiles of the canvas.
struct Tiles {
  uint32_t a0, nA, nB;
};
__host__ __device__ __forceinline__ Tiles tiles_of(const MaskParams& m, uint32_t row_first, uint32_t row_last) {
  Tiles t = {0, 0, 0};
  const uint32_t lo = mask_row_lo(m, row_first);
  if (m.pre_hi > lo) {
    t.a0 = lo / BLK;
    t.nA = (m.pre_hi + BLK - 1) / BLK - t.a0;
  }
  const uint32_t hi = mask_can_hi_rows(m, row_last);
  if (hi > m.kv_len) t.nB = (hi - m.kv_len + BLK - 1) / BLK;
  return t;
}
// A canvas tile takes twice a cached one's work; split s of S has the tiles [split_cut(s), split_cut(s + 1)).
__host__ __device__ __forceinline__ uint32_t tile_cost(const Tiles& t) { return t.nA + 2 * t.nB; }
__host__ __device__ __forceinline__ uint32_t split_cut(const Tiles& t, uint32_t s, uint32_t S) {
  const uint32_t x = uint32_t(uint64_t(tile_cost(t)) * s / S);
  return x <= t.nA ? x : t.nA + (x - t.nA) / 2;
}

cudaError_t configure();
// queries of n_seq canvases and, where p.n_ctiles is not zero, their K and V
cudaError_t launch_rows(const QueryParams& q, const CodeParams& p, const uint64_t* pos, uint32_t n_seq, cudaStream_t st);
cudaError_t launch_append(const CodeParams& p, cudaStream_t st);
cudaError_t launch_read(const ReadParams& p, cudaStream_t st);
cudaError_t launch_token(const TokenParams& p, uint32_t D, uint32_t n_ctas, cudaStream_t st);
cudaError_t launch_merge(const AttnParams8& p, uint32_t most_splits, cudaStream_t st);
cudaError_t launch_attention(const AttnParams8& p, bool pair, uint32_t n_ctas, uint32_t most_splits, cudaStream_t st);
// ctas: pairs of them where pair
cudaError_t launch_weights(const WeightParams& p, uint32_t D, bool pair, uint32_t ctas, cudaStream_t st);
cudaError_t launch_evict(const EvictParams& p, cudaStream_t st);

}  // namespace kv8
}  // namespace dg
