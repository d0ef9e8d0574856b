// Attention of few query rows (at most 16 for each KV head: single tokens) over caches held in 8 bits.
//
// What bounds it is reading the cache once, 6.4 TB/s over 148 SMs: 64 KB of K and V for 128 keys of 256 dims in 2,850 cycles of
// an SM.  With 16 rows an M = 128 tile of queries would be empty for seven eighths and the two-term passes still take 2,048
// cycles, so the products are turned round, the cache as the 128-row operand and the queries as 16 columns:
//   S^T[key][row]  = K [q1 | q2]^T       D / 32 MMAs (M 128, N 32, K 32), the two halves added in fp32
//   O^T[dim][row] += V^T [p1 | p2 | p3]^T  D / 32 MMAs (M 128, N 48, K 32), V^T as it lies (MN-major), P through shared memory
// An MMA takes the 55 cycles that its 4 KB of the cache take, however few columns: 900 cycles, with the terms as columns of one
// (as passes of N 16 each: 1,750).  So P has three terms, all e5m2 (one type a product), as in the kernel of whole canvases.
// A thread of the softmax is a key and has the scores of half the rows in registers (two groups of four warps); a row's maximum is only looked for in the tiles
// where some key exceeds what the exponents refer to by more than 2^LAG (one barrier says so), sums stay in the threads until
// the end.  One CTA has all dims of a range of key tiles (head_dim 512 as well), five or six 32 KB units of K and V under way.
//
// The rows are prepared where they are used: norm and rotation of this head's queries, a warp each, while the first units
// load.  The canvas's own keys (up to 8) belong to the CTA with the last range: their scores and weighted values are fp32 sums
// over the bf16 rows, from which the accumulators start.
#include "dg_kv8_rows.cuh"

namespace dg {
namespace kv8 {

constexpr uint32_t NR = 16;                                         // query rows
constexpr uint32_t PREP_WARPS = 12, TW_LOAD = 12, TW_MMA = 13, TT = 448;
constexpr float TLAG = 3.0f;                                        // 2^(TLAG + LIFT) = 32,768 <= 57,344
constexpr uint32_t HR = NR / 2;                                     // rows of a softmax thread
// where row r stands among the columns: the even ones first, so that each group has half of however many there are
__host__ __device__ __forceinline__ uint32_t slot_of(uint32_t r) { return (r & 1u) * HR + (r >> 1); }
constexpr uint32_t NS = 2 * NR, NO = TERMS * NR;         // columns of a score and of an output accumulator
constexpr uint32_t TT_S = 0, TT_O = 2 * NS;                         // tensor memory: two S buffers, O of each 128 dims

template <uint32_t D> struct TCfg {
  static constexpr uint32_t KU = D / 256, SL = D / 128;
  static constexpr uint32_t NU = D == 256 ? 6 : 5;                  // units under way
  static constexpr uint32_t Q_SLAB = NS * 128, P_BUF = NO * 128, O_Q = NU * UNIT, O_P = O_Q + SL * Q_SLAB;
  // two buffers of P; then the bf16 rows, at head_dim 256 behind the angles in the last unit's place
  static constexpr uint32_t O_QB = D == 256 ? (NU - 1) * UNIT + TOKEN_CANVAS * 128 * 16 : O_P + 2 * P_BUF;
  static constexpr uint32_t O_KB = O_QB + NR * D * 2, O_VB = O_KB + TOKEN_CANVAS * D * 2;
  static constexpr uint32_t O_F = D == 256 ? O_P + 2 * P_BUF : O_VB + TOKEN_CANVAS * D * 2;   // see Small
  static_assert(D != 256 || O_VB + TOKEN_CANVAS * D * 2 <= NU * UNIT, "the rows fit the last unit");
  static constexpr uint32_t O_BAR = O_F + 1024 + 512;
  static constexpr uint32_t SMEM = O_BAR + 24 * 8 + 16;
  static_assert(SMEM <= 232448, "shared memory of a CTA");
  static constexpr uint32_t TM_COLS = 256;
};
struct Small {
  float c[NR];                        // (by slot) scale * log2 e * 2^exponent of the row
  float red[8][HR];                   // row maxima, row sums by warp
  float sc[NR][TOKEN_CANVAS];         // canvas scores in base 2, then weights
  float m0[NR], l0[NR];               // (by slot) reference and sum that a row starts from
  uint32_t lo[NR];                    // (by slot) first cached key that the row sees
};
static_assert(sizeof(Small) <= 1024 + 512, "small arrays");

enum { TB_FULL = 0, TB_EMPTY = 6, TB_S = 12, TB_P = 14, TB_PV = 16, TB_PREP = 18, T_BARS = 19 };

__device__ __forceinline__ float warp_max(float x) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ bool bar_any(uint32_t id, uint32_t threads, bool x) {   // a barrier that says whether any thread's x holds
  uint32_t r;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.red.or.pred q, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t"
      "}\n"
      : "=r"(r)
      : "r"(uint32_t(x)), "r"(id), "r"(threads)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void bar_threads(uint32_t id, uint32_t threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

template <uint32_t D>
__global__ void __launch_bounds__(TT, 1) dg_kv8_token_kernel(const __grid_constant__ TokenParams p) {
  typedef TCfg<D> cf;
  constexpr int NJ = int(D / 256);
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t s0 = smem_u32(smem);
  volatile uint32_t* ctl = reinterpret_cast<volatile uint32_t*>(smem + cf::O_BAR + 24 * 8);
  volatile uint32_t* abort_flag = &ctl[0];
  auto bar = [&](uint32_t i) { return s0 + cf::O_BAR + i * 8u; };
  Small& sm = *reinterpret_cast<Small*>(smem + cf::O_F);
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  grid_launch_dependents();
  if (s0 & 1023u) {
    if (tid == 0) dev_status_set(p.status, DG_DEV_SMEM_LAYOUT, KID_TOKEN, blockIdx.x, s0);
    return;
  }
  uint32_t b = 0;
  for (uint32_t step = MAX_SEQ / 2; step > 0; step >>= 1)
    if (b + step < p.n_seq && p.seq[b + step].first_cta <= blockIdx.x) b += step;
  const Seq& sq = p.seq[b];
  const uint32_t item = blockIdx.x - sq.first_cta, kvh = item % p.Hkv, split = item / p.Hkv;
  const uint32_t rows = p.C * p.G;
  MaskParams mk = {};
  mk.kv_len = mk.pre_hi = sq.n_keys;
  mk.can_hi = p.k != nullptr ? sq.n_keys + p.C : sq.n_keys;
  mk.mode = p.mode;
  mk.windowed = p.windowed;
  mk.wm1 = p.wm1;
  const Tiles ts = tiles_of(mk, 0, p.C - 1);
  const uint32_t n0 = uint32_t(uint64_t(ts.nA) * split / sq.n_splits), n1 = uint32_t(uint64_t(ts.nA) * (split + 1) / sq.n_splits);
  const uint32_t n_local = n1 - n0;
  const bool canvas = p.k != nullptr && split + 1 == sq.n_splits;

  if (tid == 0) {
    ctl[0] = 0u;
    for (uint32_t i = 0; i < T_BARS; ++i) mbar_init(bar(i), i == TB_PREP ? PREP_WARPS : (i == TB_P || i == TB_P + 1) ? 8u : 1u);
    fence_mbar_init();
  }
  if (warp == TW_MMA) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(&ctl[1])), cf::TM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl[1];
  grid_wait();

  // softmax warps: rows 2 j + half in slots HR half + j; nj of them are there
  const uint32_t half = (warp >> 2) & 1u, nj = (rows + 1u - half) / 2u, key = tid & 127u;
  float m[HR], l[HR];
#pragma unroll
  for (uint32_t j = 0; j < HR; ++j) {
    m[j] = -INFINITY;
    l[j] = 0.f;
  }
  const uint32_t t_lane = tmem + ((warp & 3u) << 21);               // 32 lanes a warp

  if (warp < PREP_WARPS) {
    // ---------------------------------------------------------------- rows
    // the angles (head_dim 256: and the bf16 rows) lie where the last unit will
    double2* tab = reinterpret_cast<double2*>(smem + (cf::NU - 1) * UNIT);
    // a warp's rows: queries, canvas K and V, then the rows of zeros; the first one's elements are requested before the angles
    const uint32_t n_live = rows + (canvas ? 2u * p.C : 0u);
    uint4 raw[NJ];
    auto request = [&](uint32_t x) {
      const bool is_q = x < rows;
      const uint32_t c = is_q ? x / p.G : (x - rows) >> 1;
      const __nv_bfloat16* src = is_q ? p.q + ((size_t(b) * p.C + c) * p.Hq + kvh * p.G + x % p.G) * D
                                      : (((x - rows) & 1u) == 0u ? p.k : p.v) + ((size_t(b) * p.C + c) * p.Hkv + kvh) * D;
#pragma unroll
      for (int j = 0; j < NJ; ++j) raw[j] = *reinterpret_cast<const uint4*>(src + 8u * (lane + 32u * j));
    };
    if (warp < n_live) request(warp);
    if (p.rope.half != 0u && tid < PREP_WARPS * 32u) angles<double, PREP_WARPS * 32>(p.rope, double(p.pos[b]), p.C, tab);
    bar_threads(2, PREP_WARPS * 32);
    bool bad = false;
    for (uint32_t y = warp; y < n_live + NR - rows; y += PREP_WARPS) {
      const bool live = y < n_live, is_q = y < rows || !live;
      const uint32_t x = live ? y : rows + (y - n_live);            // row of the tile, where it is a query
      const uint32_t c = is_q ? x / p.G : (y - rows) >> 1;          // canvas row
      const bool is_k = !is_q && ((y - rows) & 1u) == 0u;
      uint4 v[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) v[j] = make_uint4(0u, 0u, 0u, 0u);
      const size_t q_at = ((size_t(b) * p.C + c) * p.Hq + kvh * p.G + x % p.G) * D + 8u * lane;
      if (live) {
        if (y != warp) request(y);
        const bool turn = (is_q || is_k) && p.rope.half != 0u;
        row_to_bf16<double, NJ>(raw, is_q ? p.qw : is_k ? p.kw : nullptr, is_q || is_k || p.v_norm != 0u, p.eps, p.rope,
                                turn ? tab + c * p.rope.half : nullptr, lane, v);
      }
      if (!is_q) {
        uint8_t* dst = smem + (is_k ? cf::O_KB : cf::O_VB) + c * D * 2;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          v[j] = make_uint4(finite_or_zero(v[j].x, &bad), finite_or_zero(v[j].y, &bad), finite_or_zero(v[j].z, &bad), finite_or_zero(v[j].w, &bad));
          *reinterpret_cast<uint4*>(dst + (lane + 32u * j) * 16u) = v[j];
        }
        continue;
      }
      uint32_t top2 = 0;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        top2 = abs_max2(abs_max2(abs_max2(abs_max2(top2, v[j].x), v[j].y), v[j].z), v[j].w);
        *reinterpret_cast<uint4*>(smem + cf::O_QB + x * D * 2 + (lane + 32u * j) * 16u) = v[j];
        if (p.q_rot != nullptr && live && split == 0) *reinterpret_cast<uint4*>(p.q_rot + q_at + 256u * j) = v[j];
      }
      const uint32_t top = __reduce_max_sync(0xffffffffu, (top2 >> 16) > (top2 & 0xffffu) ? top2 >> 16 : top2 & 0xffffu);
      const bool fin = top < 0x7f80u;                               // a row that is not finite has no scores: its codes are NaN
      const int e = fin ? scale_exp(__uint_as_float(top << 16)) : 0;
      const float mul = fin ? pow2i(-e) : __uint_as_float(0x7fc00000u);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const uint32_t ch = lane + 32u * j;                         // chunk of 8 dims
        const uint32_t off = (ch >> 4) * cf::Q_SLAB + chunk_off(slot_of(x), (ch & 15u) >> 1) + (ch & 1u) * 8u;
        uint2 rest;
        const uint2 code = code8(v[j], mul, &rest);
        *reinterpret_cast<uint2*>(smem + cf::O_Q + off) = code;
        *reinterpret_cast<uint2*>(smem + cf::O_Q + NR * 128u + off) = rest;   // (rows 16-31 of the operand)
      }
      if (lane == 0) {
        sm.c[slot_of(x)] = p.scale_log2 * pow2i(e);
        sm.lo[slot_of(x)] = mask_row_lo(mk, live ? c : 0u);
      }
    }
    if (bad) dev_status_set(p.status, DG_DEV_NOT_FINITE, KID_TOKEN, blockIdx.x, 0u);
    fence_proxy_async_smem();
    bar_threads(2, PREP_WARPS * 32);
    if (canvas) {
      // scores of the canvas's keys, a warp for each (row, key)
      for (uint32_t x = warp; x < rows * p.C; x += PREP_WARPS) {
        const uint32_t r = x / p.C, c = x % p.C;
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const uint4 a = *reinterpret_cast<const uint4*>(smem + cf::O_QB + r * D * 2 + (lane + 32u * j) * 16u);
          const uint4 k = *reinterpret_cast<const uint4*>(smem + cf::O_KB + c * D * 2 + (lane + 32u * j) * 16u);
          const uint32_t ua[4] = {a.x, a.y, a.z, a.w}, uk[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            dot = fmaf(__uint_as_float(ua[i] << 16), __uint_as_float(uk[i] << 16), dot);
            dot = fmaf(__uint_as_float(ua[i] & 0xffff0000u), __uint_as_float(uk[i] & 0xffff0000u), dot);
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        const RowVis rv = mask_row(mk, r / p.G);
        const uint32_t t = sq.n_keys + c;
        if (lane == 0) sm.sc[r][c] = t >= rv.can_lo && t < rv.can_hi ? dot * p.scale_log2 : -INFINITY;
      }
      bar_threads(2, PREP_WARPS * 32);
      // a row's weights over the canvas, from which its sums start
      if (tid < rows) {
        float* sc = sm.sc[tid];
        float top = -INFINITY, sum = 0.f;
        for (uint32_t c = 0; c < p.C; ++c) top = fmaxf(top, sc[c]);
        for (uint32_t c = 0; c < p.C; ++c) {
          const float w = sc[c] == -INFINITY ? 0.f : fast_exp2(sc[c] - (top == -INFINITY ? 0.f : top) + LIFT);   // (NaN stays)
          sum += w;
          sc[c] = w;
        }
        sm.m0[slot_of(tid)] = top;
        sm.l0[slot_of(tid)] = sum;
      }
      bar_threads(2, PREP_WARPS * 32);
      if (warp < 8) {
#pragma unroll 1
        for (uint32_t d = 0; d < D / 128; ++d) {
          uint32_t o[8];
          float acc[HR] = {};
          for (uint32_t c = 0; c < p.C; ++c) {
            const float v = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(smem + cf::O_VB + (c * D + d * 128u + key) * 2u));
#pragma unroll
            for (uint32_t j = 0; j < HR; ++j)
              if (j < nj) acc[j] = fmaf(sm.sc[2u * j + half][c], v, acc[j]);
          }
#pragma unroll
          for (uint32_t j = 0; j < HR; ++j) o[j] = __float_as_uint(acc[j]);
          tmem_st8(t_lane + TT_O + d * NO + half * HR, o);
#pragma unroll
          for (uint32_t j = 0; j < HR; ++j) o[j] = 0u;
#pragma unroll
          for (uint32_t i = 1; i < TERMS; ++i) tmem_st8(t_lane + TT_O + d * NO + i * NR + half * HR, o);
        }
#pragma unroll
        for (uint32_t j = 0; j < HR; ++j)
          if (j < nj) {
            m[j] = sm.m0[half * HR + j];
            l[j] = key == 0 ? sm.l0[half * HR + j] : 0.f;
          }
        tmem_wait_st();
        tc_fence_before();
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(TB_PREP));
  }

  if (warp < 8) {
    // ---------------------------------------------------------------- softmax: a thread is a key
    const uint32_t bid = 3u + half;                                 // the group's barrier
    float c[HR];
#pragma unroll
    for (uint32_t j = 0; j < HR; ++j) c[j] = sm.c[half * HR + j];
    const uint32_t lo_last = mask_row_lo(mk, p.C - 1);
    const int2* ep = sq.exps + size_t(kvh) * sq.blocks + ts.a0 + n0;
    int2 ex = n_local > 0 ? *ep : make_int2(0, 0);
    for (uint32_t n = 0; n < n_local; ++n) {
      const uint32_t sb = n & 1u;
      const int ek = ex.x, ev = ex.y;
      if (n + 1 < n_local) ex = *++ep;
      // (A wait that gave up ends nothing here: a group's warps go through the same barriers to the end, and the status reports it.)
      __all_sync(0xffffffffu, bar_wait(bar(TB_S + sb), (n >> 1) & 1u, abort_flag));
      tc_fence_after();
      uint32_t s1[8], s2[8];
      tmem_ld8(t_lane + TT_S + sb * NS + half * HR, s1);
      tmem_ld8(t_lane + TT_S + sb * NS + NR + half * HR, s2);
      const float fk = pow2i(ek), fv = float(ev);
      const uint32_t t0 = (ts.a0 + n0 + n) * BLK, t = t0 + key;
      const bool edge = t0 < lo_last || t0 + BLK > sq.n_keys;
      tmem_wait_ld();
      float x[HR];                                                  // exponents in base 2, of a weight times its block's scale of V
      bool over = false;
#pragma unroll
      for (uint32_t j = 0; j < HR; ++j) {
        x[j] = fmaf(__uint_as_float(s1[j]) + __uint_as_float(s2[j]), c[j] * fk, fv);
        if (edge && (t < sm.lo[half * HR + j] || t >= sq.n_keys)) x[j] = -INFINITY;
        over = over || (x[j] > m[j] + TLAG && j < nj);
      }
      if (bar_any(bid, 128, over)) {
        // a row's reference moves: find the maxima, bring the accumulators and sums to them
#pragma unroll
        for (uint32_t j = 0; j < HR; ++j) {
          const float w = warp_max(x[j]);
          if (lane == 0) sm.red[warp][j] = w;
        }
        if (n != 0) __all_sync(0xffffffffu, bar_wait(bar(TB_PV + (sb ^ 1u)), ((n - 1u) >> 1) & 1u, abort_flag));
        tc_fence_after();
        bar_threads(bid, 128);
        float alpha[HR];
#pragma unroll
        for (uint32_t j = 0; j < HR; ++j) {
          const float* red = &sm.red[half * 4u][j];
          const float top = fmaxf(fmaxf(red[0], red[HR]), fmaxf(red[2 * HR], red[3 * HR]));
          const bool need = top > m[j] + TLAG;
          alpha[j] = need ? (m[j] == -INFINITY ? 0.f : fast_exp2(m[j] - top)) : 1.0f;
          if (need) m[j] = top;
          l[j] *= alpha[j];
        }
        if (n != 0 || canvas) {
#pragma unroll 1
          for (uint32_t i = 0; i < TERMS * (D / 128); ++i) {
            uint32_t o[8];
            tmem_ld8(t_lane + TT_O + i * NR + half * HR, o);
            tmem_wait_ld();
#pragma unroll
            for (uint32_t j = 0; j < HR; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha[j]);
            tmem_st8(t_lane + TT_O + i * NR + half * HR, o);
          }
          tmem_wait_st();
        }
        bar_threads(bid, 128);                                      // the maxima have been read
      }
      // P of the tile before last has been used
      if (n > 1) __all_sync(0xffffffffu, bar_wait(bar(TB_PV + sb), ((n - 2u) >> 1) & 1u, abort_flag));
      const float back = pow2i(-ev);
      uint8_t* pt = smem + cf::O_P + sb * cf::P_BUF + (key & 15u);
#pragma unroll
      for (uint32_t j = 0; j < HR; j += 4) {
        if (j >= nj) continue;
#pragma unroll
        for (uint32_t i = j; i < j + 4; ++i) {
          x[i] = fast_exp2(x[i] - (m[i] == -INFINITY ? 0.f : m[i]) + LIFT);
          l[i] = fmaf(x[i], back, l[i]);
        }
        uint32_t w[TERMS];
        split4_e5m2(x[j], x[j + 1], x[j + 2], x[j + 3], w);
#pragma unroll
        for (uint32_t k = 0; k < TERMS; ++k)
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i)
            if (j + i < nj) pt[chunk_off(k * NR + half * HR + j + i, key >> 4)] = uint8_t(w[k] >> (8u * i));
      }
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(TB_P + sb));
    }

    // ---------------------------------------------------------------- output: a thread is a dim
    bool have = __all_sync(0xffffffffu, !*abort_flag);
    if (have && n_local > 0) {
      have = __all_sync(0xffffffffu, bar_wait(bar(TB_PV + ((n_local - 1u) & 1u)), ((n_local - 1u) >> 1) & 1u, abort_flag));
      tc_fence_after();
    }
    const bool some = have && (n_local > 0 || canvas);
#pragma unroll
    for (uint32_t j = 0; j < HR; ++j) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], o);
      if (lane == 0) sm.red[warp][j] = l[j];
    }
    bar_threads(bid, 128);
    const bool direct = sq.n_splits == 1;
#pragma unroll
    for (uint32_t j = 0; j < HR; ++j) {
      const float* red = &sm.red[half * 4u][j];
      l[j] = (red[0] + red[HR]) + (red[2 * HR] + red[3 * HR]);
    }
#pragma unroll
    for (uint32_t d = 0; d < D / 128; ++d) {
      uint32_t o[TERMS][8];
      if (some) {
#pragma unroll
        for (uint32_t i = 0; i < TERMS; ++i) tmem_ld8(t_lane + TT_O + d * NO + i * NR + half * HR, o[i]);
        tmem_wait_ld();
      } else {
#pragma unroll
        for (uint32_t i = 0; i < TERMS; ++i)
#pragma unroll
          for (uint32_t j = 0; j < HR; ++j) o[i][j] = 0u;
      }
#pragma unroll
      for (uint32_t j = 0; j < HR; ++j) {
        if (j >= nj) continue;
        const uint32_t r = 2u * j + half;
        const float y = __uint_as_float(o[0][j]) + (__uint_as_float(o[1][j]) + __uint_as_float(o[2][j]));
        if (direct) {
          const float inv = l[j] > 0.f ? 1.0f / l[j] : (l[j] == 0.f ? 0.f : l[j]);
          p.out[((size_t(b) * p.C + r / p.G) * p.Hq + kvh * p.G + r % p.G) * D + d * 128u + key] = __float2bfloat16(y * inv);
        } else {
          p.ws_o[((size_t(blockIdx.x) * cf::KU + d / 2u) * BLK + r) * 256u + (d & 1u) * 128u + key] = y;
        }
      }
    }
#pragma unroll
    for (uint32_t j = 0; j < HR; ++j) {
      if (j >= nj || key != j) continue;
      const uint32_t r = 2u * j + half;
      if (!direct) {
        for (uint32_t z = 0; z < cf::KU; ++z) p.ws_ml[(size_t(blockIdx.x) * cf::KU + z) * BLK + r] = make_float2(m[j], l[j]);
      } else if (p.lse != nullptr) {
        p.lse[(size_t(b) * p.C + r / p.G) * p.Hq + kvh * p.G + r % p.G] = l[j] == 0.f ? -INFINITY : (m[j] - LIFT + log2f(l[j])) * 0.6931471805599453f;
      }
    }
  } else if (warp == TW_LOAD) {
    if (lane == 0) {
      uint32_t u = 0;
      bool ok = true;
      auto load = [&](const uint8_t* base, uint32_t n) {
        const uint8_t* src = base + (size_t(kvh) * sq.blocks + ts.a0 + n0 + n) * BLK * D;
        for (uint32_t i = 0; ok && i < cf::KU; ++i, ++u) {
          const uint32_t st = u % cf::NU;
          if (u >= cf::NU) ok = bar_wait(bar(TB_EMPTY + st), (u / cf::NU - 1u) & 1u, abort_flag);
          else if (st == cf::NU - 1u) ok = bar_wait(bar(TB_PREP), 0u, abort_flag);   // the angles lie there
          if (!ok) return;
          mbar_expect_tx(bar(TB_FULL + st), UNIT);
          bulk_load(s0 + st * UNIT, src + size_t(i) * UNIT, UNIT, bar(TB_FULL + st));
        }
      };
      if (n_local > 0) load(sq.k, 0);
      for (uint32_t n = 0; ok && n < n_local; ++n) {                 // the order in which they are used
        if (n + 1 < n_local) load(sq.k, n + 1);
        if (ok) load(sq.v, n);
      }
    }
  } else if (warp == TW_MMA && n_local > 0) {
    constexpr uint32_t HI = (1024u >> 4) | (1u << 14) | (2u << 29);
    auto desc = [](uint32_t lo) { return (uint64_t(HI) << 32) | uint64_t(lo); };
    constexpr uint32_t IDESC_S = idesc_f8(128, NS, 0, 0);
    constexpr uint32_t IDESC_O = idesc_f8(128, NO, 0, 0) | (1u << 15) | (1u << 10);   // A = V^T (M-major) e4m3, B = P e5m2
    const uint32_t base = ((s0 >> 4) & 0x3fffu) | (1u << 16);
    const uint32_t dq = base + (cf::O_Q >> 4), dp = base + (cf::O_P >> 4), dv = ((s0 >> 4) & 0x3fffu) | ((SLAB >> 4) << 16);
    bool ok = __all_sync(0xffffffffu, bar_wait(bar(TB_PREP), 0u, abort_flag));
    tc_fence_after();
    uint32_t u = 0;
    auto issue_s = [&](uint32_t n) -> bool {
      const uint32_t d_tmem = tmem + TT_S + (n & 1u) * NS;
      for (uint32_t i = 0; i < cf::KU; ++i, ++u) {
        const uint32_t st = u % cf::NU;
        if (!__all_sync(0xffffffffu, bar_wait(bar(TB_FULL + st), (u / cf::NU) & 1u, abort_flag))) return false;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t ka = base + st * (UNIT >> 4), qb = dq + i * 2u * (cf::Q_SLAB >> 4);
#pragma unroll
          for (uint32_t j = 0; j < 8; ++j) {                        // slab, 32 dims
            const uint32_t sl = j >> 2, kk = j & 3u;
            mma_ss(d_tmem, desc(ka + sl * (SLAB >> 4) + kk * 2u), desc(qb + sl * (cf::Q_SLAB >> 4) + kk * 2u), IDESC_S, j == 0 ? i != 0u : 1u);
          }
          umma_commit(bar(TB_EMPTY + st));
          if (i + 1 == cf::KU) umma_commit(bar(TB_S + (n & 1u)));
        }
        __syncwarp();
      }
      return true;
    };
    ok = ok && issue_s(0);
    for (uint32_t n = 0; ok && n < n_local; ++n) {
      if (n + 1 < n_local && !issue_s(n + 1)) break;
      if (!__all_sync(0xffffffffu, bar_wait(bar(TB_P + (n & 1u)), (n >> 1) & 1u, abort_flag))) break;
      for (uint32_t i = 0; ok && i < cf::KU; ++i, ++u) {
        const uint32_t st = u % cf::NU;
        ok = __all_sync(0xffffffffu, bar_wait(bar(TB_FULL + st), (u / cf::NU) & 1u, abort_flag));
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t va = dv + st * (UNIT >> 4), pb = dp + (n & 1u) * (cf::P_BUF >> 4);
#pragma unroll
          for (uint32_t j = 0; j < 8; ++j) {                        // 128 dims, 32 keys
            const uint32_t sl = j >> 2, ks = j & 3u;
            mma_ss(tmem + TT_O + (i * 2u + sl) * NO, desc(va + sl * (SLAB >> 4) + ks * 256u), desc(pb + ks * 2u), IDESC_O, ks == 0 ? (n != 0u || canvas) : 1u);
          }
          umma_commit(bar(TB_EMPTY + st));
          if (i + 1 == cf::KU) umma_commit(bar(TB_PV + (n & 1u)));
        }
        __syncwarp();
      }
    }
  }

  if (*abort_flag) {
    if (tid == 0) dev_status_set(p.status, DG_DEV_WAIT_TIMEOUT, KID_TOKEN, blockIdx.x, n_local);
    if (warp == TW_LOAD && lane == 0) {
      const long long c0 = clock64();
      while (clock64() - c0 < 2000000ll) {}   // ~1 ms: far longer than any load in flight
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == TW_MMA) tmem_dealloc(tmem, cf::TM_COLS);
}

cudaError_t configure_token() {
  cudaError_t e = cudaFuncSetAttribute(dg_kv8_token_kernel<256>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(TCfg<256>::SMEM));
  if (e == cudaSuccess) e = cudaFuncSetAttribute(dg_kv8_token_kernel<512>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(TCfg<512>::SMEM));
  return e;
}

cudaError_t launch_token(const TokenParams& p, uint32_t D, uint32_t n_ctas, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n_ctas);
  cfg.blockDim = dim3(TT);
  cfg.dynamicSmemBytes = D == 256 ? TCfg<256>::SMEM : TCfg<512>::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return D == 256 ? cudaLaunchKernelEx(&cfg, dg_kv8_token_kernel<256>, p) : cudaLaunchKernelEx(&cfg, dg_kv8_token_kernel<512>, p);
}

}  // namespace kv8
}  // namespace dg
