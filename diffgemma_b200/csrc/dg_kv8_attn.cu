// Attention of canvas rows over caches held in 8 bits (csrc/dg_kv8.cuh has the format).
//
// One CTA: 128 GQA-stacked query rows of one KV head (row R -> canvas row R / G, head R % G), one range of key tiles, 256
// value columns (a head_dim-512 layer takes two CTAs, both computing the scores).  One pass over the tiles with the running
// maximum and sum of the softmax:
//   S = (q1 + q2) K          2 x D / 32 MMAs (M 128, N 128, K 32), K as the cache holds it
//   x = s * c 2^ek + ev - m  the block's scales are powers of two: that of K multiplies, that of V shifts the exponent
//   P = 2^x = p1 + p2 + p3   e5m2 each, in tensor memory, over the columns that S occupied
//   O += (p1 + p2 + p3) V    12 MMAs (M 128, N 256, K 32)
//   l += 2^-ev sum P         in fp32, from P before it is rounded
// m follows the largest x with a lag of at most 2^LAG (O is rescaled only beyond it), so P <= 2^15 stays inside e5m2.  Three terms hold
// a weight to 2^-11 of itself down to 2^-18 of its row's largest, and to 2^-29 of that below: a strong first token without a
// value beside 10^5 weak ones spoils none of them.
// Tiles of the canvas come as two terms as well (K = k1 + k2, V = v1 + v2: the rows' bf16 values) and pass twice.
//
// Per 128 keys, 256 dims: 2,560 cycles of MMA, 64 KB from L2 / HBM, 16,384 exponentials (1,024 cycles), and 288 KB through
// shared memory (S: 4 KB of Q and 4 KB of K for each MMA of 64 cycles; PV 96 KB; the copies 64 KB), which at 128 bytes a cycle
// take 2,304.  Measured: 3,400 cycles, the rest is the way from scores to weights and the waits between (32,768 keys of 2 KV
// heads, 256 rows: 148 us).  Two terms, e4m3 + e5m2, are 512 cycles of MMA less (123 us), but hold a weight at 2^-16 of its row's
// largest to 2^-3 of itself only; a third term in the tiles that have such weights would be in nearly all of them.
// head_dim 512: 3,584 cycles of MMA and 448 KB (3,584 cycles) a tile.  There two row tiles make a pair of CTAs
// (cta_group::2, M = 256): each brings half of K's tokens and half of V's dims, so that copies and B operands halve (288 KB).
// 256 rows over 2 KV heads, two terms, us alone / in pairs: 2,000 keys 47.6 / 46.7, 8,000 98.5 / 93.3, 32,000 313.6 / 285.9 (three
// terms in pairs: 324); a canvas of 64, 32,000 keys 91.1 / 88.9.  head_dim 256 gains nothing (122 / 128: its tiles are too short to hide
// the other CTA's word).
#include "dg_kv8.cuh"

namespace dg {
namespace kv8 {

constexpr uint32_t T_S = 0, T_O = 256;          // tensor memory: two S buffers of 128 columns, O
constexpr float LAG = 3.0f;                     // 2^(LAG + LIFT) = 32,768 <= 57,344
constexpr uint32_t SM_WARPS = 16, W_K = 16, W_V = 17, W_MMA = 18, W_PASS = 19;   // W_PASS: CTA pairs only
// B_P_FULL of a tile counts its softmax warps and the bytes of its first V unit; B_V2_FULL those of a canvas tile's second
enum { B_Q = 0, B_O = 1, B_K_FULL = 2, B_K_EMPTY = 6, B_V2_FULL = 10, B_V_EMPTY = 11, B_S_FULL = 13, B_P_FULL = 15, B_V_OWN = 17, N_BARS = 19 };

template <uint32_t D, bool PAIR> struct Cfg {
  static constexpr uint32_t THREADS = (PAIR ? W_PASS + 1 : W_PASS) * 32;
  static constexpr uint32_t KU = D / 256;                       // K units of a tile (32 KB each)
  static constexpr uint32_t NK = PAIR ? 4 : D == 256 ? 3 : 2, NV = PAIR || D == 256 ? 2 : 1;   // stages
  static_assert(!PAIR || D == 512, "pairs: see launch_attention");
  static constexpr uint32_t HAVE = PAIR ? UNIT / 2 : UNIT;      // bytes of a unit in this CTA
  static constexpr uint32_t Q_BYTES = 2 * BLK * D;
  static constexpr uint32_t O_K = Q_BYTES, O_V = O_K + NK * HAVE, O_X = O_V + NV * HAVE;
  static constexpr uint32_t X_BYTES = 4 * BLK * 4;              // row maxima of a row's four threads
  static constexpr uint32_t O_BAR = O_X + X_BYTES, SMEM = O_BAR + N_BARS * 8 + 16;
  static_assert(SMEM <= 232448, "shared memory of a CTA");
};

__device__ __forceinline__ void bar_sync_id(uint32_t id, uint32_t threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
// 32 weights of a row from their scores: a word of codes of each term for every four; sums into ls
__device__ __forceinline__ void weights32(const uint32_t (&s)[32], uint64_t c2, uint64_t sh2, uint64_t (&ls)[2], uint32_t (&p)[TERMS][8]) {
#pragma unroll
  for (uint32_t e = 0; e < 32; e += 4) {
    float w[4];
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
      unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(s[e + 2 * j]), __uint_as_float(s[e + 2 * j + 1])), c2, sh2), w[2 * j], w[2 * j + 1]);
      w[2 * j] = fast_exp2(w[2 * j]);
      w[2 * j + 1] = fast_exp2(w[2 * j + 1]);
      ls[j] = add_f32x2(ls[j], pack_f32x2(w[2 * j], w[2 * j + 1]));
    }
    uint32_t t[TERMS];
    split4_e5m2(w[0], w[1], w[2], w[3], t);
#pragma unroll
    for (uint32_t i = 0; i < TERMS; ++i) p[i][e >> 2] = t[i];
  }
}
__device__ __forceinline__ float max32(const uint32_t (&s)[32]) {
  float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (uint32_t e = 0; e < 32; e += 2) mx[(e >> 1) & 3u] = max3_f32(mx[(e >> 1) & 3u], __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
  return max3_f32(max3_f32(mx[0], mx[1], mx[2]), mx[3], -INFINITY);
}
// scores of keys [k0, k0 + 32) that the row does not see become -inf
__device__ __forceinline__ void hide32(uint32_t (&s)[32], uint32_t lo, uint32_t hi, uint32_t k0) {
  if (k0 >= lo && k0 + 32u <= hi) return;
  const uint32_t seen = mask_run16(lo, hi, k0) | (mask_run16(lo, hi, k0 + 16u) << 16);
#pragma unroll
  for (uint32_t e = 0; e < 32; ++e)
    if (!((seen >> e) & 1u)) s[e] = 0xff800000u;
}

template <uint32_t D, bool PAIR>
__global__ void __launch_bounds__(Cfg<D, PAIR>::THREADS, 1) dg_kv8_attn_kernel(const __grid_constant__ AttnParams8 p) {
  typedef Cfg<D, PAIR> cf;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t s0 = smem_u32(smem);
  volatile uint32_t* ctl = reinterpret_cast<volatile uint32_t*>(smem + cf::O_BAR + N_BARS * 8);   // {abort, tmem}
  volatile uint32_t* abort_flag = &ctl[0];
  const uint32_t bars = s0 + cf::O_BAR;
  auto bar = [&](uint32_t i) { return bars + i * 8u; };
  float* xch = reinterpret_cast<float*>(smem + cf::O_X);
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;

  grid_launch_dependents();
  if (s0 & 1023u) {   // the swizzled operands need the window itself aligned
    if (tid == 0) dev_status_set(p.status, DG_DEV_SMEM_LAYOUT, KID_ATTN, blockIdx.x, s0);
    return;
  }
  // which sequence, row tile, head, split and value half this CTA has
  uint32_t b = 0;
  for (uint32_t step = MAX_SEQ / 2; step > 0; step >>= 1)
    if (b + step < p.n_seq && p.seq[b + step].first_cta <= blockIdx.x) b += step;
  const Seq& sq = p.seq[b];
  uint32_t item = blockIdx.x - sq.first_cta;
  const uint32_t rank = PAIR ? item & 1u : 0u;                 // in the pair; the leader is 0
  if (PAIR) item >>= 1;
  const uint32_t z = item % cf::KU;
  item /= cf::KU;
  const uint32_t row_tiles = PAIR ? p.MT / 2u : p.MT;
  const uint32_t mt0 = PAIR ? item % row_tiles * 2u : item % row_tiles, mt = mt0 + rank;
  item /= row_tiles;
  const uint32_t kvh = item % p.Hkv, split = item / p.Hkv;
  const uint32_t slot = sq.first_cta + ((split * p.Hkv + kvh) * p.MT + mt) * cf::KU + z;
  const MaskParams mk = seq_mask(p, sq.n_keys);
  const uint32_t rows_per_head = p.C * p.G;
  const uint32_t R_end = (mt0 + (PAIR ? 2u : 1u)) * BLK, R_last = R_end < rows_per_head ? R_end - 1 : rows_per_head - 1;
  const Tiles ts = tiles_of(mk, mt0 * BLK / p.G, R_last / p.G);   // a pair's two row tiles pass over the same keys
  const uint32_t n0 = split_cut(ts, split, sq.n_splits), n1 = split_cut(ts, split + 1, sq.n_splits);
  const uint32_t n_local = n1 - n0;
  const uint32_t n_cached = ts.nA > n0 ? (ts.nA - n0 < n_local ? ts.nA - n0 : n_local) : 0u;   // cached tiles come first
  // Units are numbered through the CTA's tiles, one of a cached tile, two of a canvas tile; unit u goes through stage u % stages.
  // Waits until the last unit of tile n has been used, for a warp that has seen the one of tile n - 2 (K) or n - 2 (V) used: a
  // canvas tile's first unit is waited for as well, so that no phase is skipped and its parity mistaken.
  auto wait_unit = [&](uint32_t barrier, uint32_t stages, uint32_t n) -> bool {
    const uint32_t u = n < n_cached ? n : 2u * n + 1u - n_cached;
    bool ok = true;
    if (n >= n_cached) ok = bar_wait(bar(barrier + (u - 1u) % stages), ((u - 1u) / stages) & 1u, abort_flag);
    return __all_sync(0xffffffffu, ok && bar_wait(bar(barrier + u % stages), (u / stages) & 1u, abort_flag));
  };

  if (tid == 0) {
    ctl[0] = 0u;
    // the leader's barriers count the other CTA's share as well: its softmax warps, and a word that its operands are there
    const uint32_t both = PAIR && rank == 0u ? 2u : 1u;
    for (uint32_t i = 0; i < N_BARS; ++i) {
      uint32_t count = 1u;
      if (i == B_Q || i == B_V2_FULL || (i >= B_K_FULL && i < B_K_EMPTY)) count = both;
      if (i == B_P_FULL || i == B_P_FULL + 1) count = rank != 0u ? SM_WARPS : both * (SM_WARPS + 1u);
      mbar_init(bar(i), count);
    }
    fence_mbar_init();
  }
  if (warp == W_MMA) {
    if (PAIR) {
      tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(&ctl[1])), 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(const_cast<uint32_t*>(&ctl[1])), 512);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if (PAIR) cluster_sync_all(); else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl[1];
  grid_wait();

  const uint32_t head_tile = (b * p.Hkv + kvh) * p.n_ctiles;   // first canvas tile of this head
  float m_used = -INFINITY, l_run = 0.f;
  const uint32_t quarter = warp & 3u, part = warp >> 2;        // softmax: rows 32 quarter + lane, score columns 32 part ..
  const uint32_t r = quarter * 32u + lane;

  if (warp < SM_WARPS) {
    // What counts here is the time from a tile's scores to its weights: at most the 2,560 cycles of MMAs that are issued in
    // between.  So all sixteen warps work on one tile, four threads a row (two groups of eight on alternate tiles: 1,640 cycles
    // to the first half of P, 2,650 to the second).
    const uint32_t R = mt * BLK + r;
    const bool valid = R < rows_per_head;
    const RowVis rv = mask_row(mk, valid ? R / p.G : 0u);
    const float c_row = valid ? p.q_row[(size_t(b) * p.Hkv + kvh) * p.MT * BLK + R].x : 0.f;
    const bool warp_on = mt * BLK + quarter * 32u < rows_per_head;   // any row of this warp
    const uint32_t t_lane = tmem + ((quarter * 32u) << 16);
    // what changes from tile to tile: the scales (requested a tile ahead), the first key, and at the first canvas tile the range
    // of keys that the row sees
    const int2* ep = sq.exps + size_t(kvh) * sq.blocks + ts.a0 + n0;
    const int2* ec = p.c_exps + head_tile + (n0 > ts.nA ? n0 - ts.nA : 0u);
    uint32_t lo = rv.lo, hi = mk.pre_hi, k0 = (ts.a0 + n0) * BLK + part * 32u, stage = 0, phase = 0;
    // this warp's rows of P are there: for the MMA warp, and for the warps that wait for its reads
    auto p_ready = [&](uint32_t sb) {
      if (lane != 0) return;
      mbar_arrive(bar(B_P_FULL + sb));
      if (PAIR && rank != 0u) mbar_arrive_remote(dsmem_addr(bar(B_P_FULL + sb), 0u));
    };
    int2 ex = make_int2(0, 0);
    if (n_local > 0) ex = n_cached > 0 ? *ep : *ec;
    if (n_cached == 0) ep = ec;
    for (uint32_t n = 0; n < n_local; ++n) {
      const uint32_t sb = n & 1u;
      if (n == n_cached) {
        lo = rv.can_lo;
        hi = rv.can_hi;
        k0 = mk.kv_len + (n0 > ts.nA ? n0 - ts.nA : 0u) * BLK + part * 32u;
      }
      const int ek = ex.x, ev = ex.y;
      ep = n + 1 == n_cached ? ec : ep + 1;
      if (n + 1 < n_local) ex = *ep;
      // head_dim 256, a cached tile: the scores are there when its K unit has been used.  That unit's stage is used again by tile
      // n + 2 at the earliest, whose scores wait for this warp's weights of tile n: the phase cannot pass unseen.  Two canvas tiles in a
      // row are four units over three stages, so canvas tiles have barriers of their own, by turns: a second commit for each of them.
      bool there;
      if (D == 256 && n < n_cached) {
        there = bar_wait(bar(B_K_EMPTY) + stage * 8u, phase, abort_flag);
        if (++stage == cf::NK) { stage = 0; phase ^= 1u; }
      } else {
        const uint32_t x = D == 256 ? n - n_cached : n;
        there = bar_wait(bar(B_S_FULL + (x & 1u)), (x >> 1) & 1u, abort_flag);
      }
      // (A wait that gave up ends nothing here: the warps of a row go through the same barriers to the end, and the status reports it.)
      __all_sync(0xffffffffu, there);
      if (!warp_on) {
        // rows behind the last one: their P stays whatever it is, no row of the output reads it
        p_ready(sb);
        continue;
      }
      tc_fence_after();
      uint32_t s[32];
      tmem_ld32(t_lane + T_S + sb * 128u + part * 32u, s);
      // the maxima of the tile before have been read by all: their warps have arrived
      if (n != 0) __all_sync(0xffffffffu, bar_wait(bar(B_P_FULL + (sb ^ 1u)), ((n - 1u) >> 1) & 1u, abort_flag));
      tmem_wait_ld();
      hide32(s, lo, hi, k0);
      k0 += BLK;
      float top = max32(s);
      xch[part * BLK + r] = top;
      const float c = c_row * pow2i(ek);
      // after this barrier all four threads of a row have their scores in registers: P may overwrite them
      bar_sync_id(1u + quarter, 128u);
      top = fmaxf(fmaxf(xch[r], xch[BLK + r]), fmaxf(xch[2 * BLK + r], xch[3 * BLK + r]));
      const float m_new = top * c + float(ev);
      const bool need = n == 0 || m_new > m_used + LAG;
      if (n != 0 && __any_sync(0xffffffffu, need)) {
        // the outputs of the tile before: its last V unit has been used
        wait_unit(B_V_EMPTY, cf::NV, n - 1u);
        tc_fence_after();
        const float alpha = need ? (m_used == -INFINITY ? 0.f : fast_exp2(m_used - m_new)) : 1.0f;
#pragma unroll 1
        for (uint32_t cc = 0; cc < 2; ++cc) {
          uint32_t o[32];
          tmem_ld32(t_lane + T_O + part * 64u + cc * 32u, o);
          tmem_wait_ld();
#pragma unroll
          for (uint32_t e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          tmem_st32(t_lane + T_O + part * 64u + cc * 32u, o);
        }
        l_run *= alpha;
      }
      if (need) m_used = m_new;
      const float shift = (m_used == -INFINITY ? 0.f : -m_used) + float(ev) + LIFT;
      const uint64_t c2 = pack_f32x2(c, c), sh2 = pack_f32x2(shift, shift);
      uint64_t ls[2] = {0ull, 0ull};
      uint32_t pt[TERMS][8];
      weights32(s, c2, sh2, ls, pt);
      // the 32 keys of a thread are the K of one MMA: columns 8 part .. of p1, the other terms 32 columns on each
#pragma unroll
      for (uint32_t i = 0; i < TERMS; ++i) tmem_st8(t_lane + T_S + sb * 128u + i * 32u + part * 8u, pt[i]);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      p_ready(sb);
      float a, d;
      unpack_f32x2(add_f32x2(ls[0], ls[1]), a, d);
      l_run = fmaf(a + d, pow2i(-ev), l_run);
    }
  } else if (warp == W_K) {
    if (lane == 0 && n_local > 0) {
      mbar_expect_tx(bar(B_Q), cf::Q_BYTES);
      const uint8_t* q = p.q_codes + ((size_t(b) * p.Hkv + kvh) * p.MT + mt) * cf::Q_BYTES;
      for (uint32_t o = 0; o < cf::Q_BYTES; o += UNIT) bulk_load(s0 + o, q + o, UNIT, bar(B_Q));
      uint32_t u = 0;
      bool ok = true;
      for (uint32_t t = n0; ok && t < n1; ++t) {
        const bool cached = t < ts.nA;
        const uint8_t* src = cached ? sq.k + (size_t(kvh) * sq.blocks + ts.a0 + t) * BLK * D
                                    : p.c_k + size_t(head_tile + t - ts.nA) * 2u * BLK * D;
        const uint32_t units = cached ? cf::KU : 2 * cf::KU;
        for (uint32_t i = 0; i < units; ++i, ++u) {
          const uint32_t st = u % cf::NK;
          if (u >= cf::NK && !bar_wait(bar(B_K_EMPTY + st), (u / cf::NK - 1u) & 1u, abort_flag)) { ok = false; break; }
          mbar_expect_tx(bar(B_K_FULL + st), cf::HAVE);
          const uint32_t dst = s0 + cf::O_K + st * cf::HAVE;
          if (PAIR) {   // 64 of the 128 tokens
            for (uint32_t sl = 0; sl < 2; ++sl)
              bulk_load(dst + sl * (SLAB / 2u), src + size_t(i) * UNIT + sl * SLAB + rank * (SLAB / 2u), SLAB / 2u, bar(B_K_FULL + st));
          } else {
            bulk_load(dst, src + size_t(i) * UNIT, UNIT, bar(B_K_FULL + st));
          }
        }
      }
    }
  } else if (warp == W_V) {
    if (lane == 0) {
      uint32_t u = 0;
      bool ok = true;
      for (uint32_t t = n0; ok && t < n1; ++t) {
        const bool cached = t < ts.nA;
        const uint8_t* src = (cached ? sq.v + (size_t(kvh) * sq.blocks + ts.a0 + t) * BLK * D
                                     : p.c_v + size_t(head_tile + t - ts.nA) * 2u * BLK * D) + size_t(z) * UNIT + rank * SLAB;   // (a pair's CTAs: 128 of the 256 dims each)
        for (uint32_t i = 0; i < (cached ? 1u : 2u); ++i, ++u) {
          const uint32_t st = u % cf::NV;
          if (u >= cf::NV && !bar_wait(bar(B_V_EMPTY + st), (u / cf::NV - 1u) & 1u, abort_flag)) { ok = false; break; }
          const uint32_t full = bar(i == 0 ? (rank == 0u ? B_P_FULL : B_V_OWN) + ((t - n0) & 1u) : B_V2_FULL);
          mbar_expect_tx(full, cf::HAVE);
          bulk_load(s0 + cf::O_V + st * cf::HAVE, src + size_t(i) * BLK * D, cf::HAVE, full);
        }
      }
    }
  } else if (PAIR && rank != 0u) {
    // Tells the leader what has come here: Q and K one warp, V the other (an arrival at cluster scope takes some 700 cycles; one
    // warp for both was late for the next tile).  The bytes came through the async proxy and are read through it.
    auto pass_on = [&](uint32_t own, uint32_t parity, uint32_t lead) -> bool {
      if (!bar_wait(bar(own), parity, abort_flag)) return false;
      mbar_arrive_cluster(dsmem_addr(bar(lead), 0u));
      return true;
    };
    if (lane == 0 && n_local > 0) {
      if (warp == W_MMA) {
        const uint32_t units = (n_cached + 2u * (n_local - n_cached)) * cf::KU;
        bool ok = pass_on(B_Q, 0u, B_Q);
        for (uint32_t u = 0; ok && u < units; ++u) ok = pass_on(B_K_FULL + u % cf::NK, (u / cf::NK) & 1u, B_K_FULL + u % cf::NK);
      } else {
        bool ok = true;
        for (uint32_t n = 0; ok && n < n_local; ++n) {
          ok = pass_on(B_V_OWN + (n & 1u), (n >> 1) & 1u, B_P_FULL + (n & 1u));
          if (ok && n >= n_cached) ok = pass_on(B_V2_FULL, (n - n_cached) & 1u, B_V2_FULL);
        }
      }
    }
  } else if (warp == W_MMA && n_local > 0) {
    // The whole warp runs the loop, one elected lane issues.  A wait costs this warp some 150 cycles in which it issues nothing;
    // one before each group of 1,024 cycles of MMAs and one commit behind it keep the tensor pipe full (2,054 cycles for 24
    // MMAs of a 256-wide tile, 8 of them PV; two waits and two commits: 2,360), so V's bytes are counted where P's arrivals are and a cached K
    // unit's release is the signal that scores are there.  Descriptors advance by adds on their low word (every operand lives
    // below 256 KB: the address field cannot carry).
    constexpr uint32_t HI = (1024u >> 4) | (1u << 14) | (2u << 29);           // 8-row groups 1024 apart, version 1, 128-byte swizzle
    auto desc = [](uint32_t lo) { return (uint64_t(HI) << 32) | uint64_t(lo); };
    constexpr uint32_t M = PAIR ? 256 : 128;
    constexpr uint32_t IDESC = idesc_f8(M, 128, 0, 0), IDESC_P = idesc_f8(M, 256, 1, 1);
    auto commit = [&](uint32_t b) { if (PAIR) commit_both(bar(b)); else umma_commit(bar(b)); };
    const uint32_t dq = ((s0 >> 4) & 0x3fffu) | (1u << 16), dk = (((s0 + cf::O_K) >> 4) & 0x3fffu) | (1u << 16);
    const uint32_t dv = (((s0 + cf::O_V) >> 4) & 0x3fffu) | ((SLAB >> 4) << 16);   // MN-major: 128-column chunks SLAB apart
    bool ok = __all_sync(0xffffffffu, bar_wait<PAIR>(bar(B_Q), 0u, abort_flag));
    uint32_t uk = 0, uv = 0;
    auto issue_qk = [&](uint32_t n) -> bool {
      const uint32_t units = n < n_cached ? cf::KU : 2 * cf::KU;
      const uint32_t d_tmem = tmem + T_S + (n & 1u) * 128u;
      for (uint32_t i = 0; i < units; ++i, ++uk) {
        const uint32_t st = uk % cf::NK;
        if (!__all_sync(0xffffffffu, bar_wait<PAIR>(bar(B_K_FULL + st), (uk / cf::NK) & 1u, abort_flag))) return false;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t qa = dq + (((i % cf::KU) * UNIT) >> 4), kb = dk + st * (cf::HAVE >> 4);
#pragma unroll
          for (uint32_t j = 0; j < 16; ++j) {   // term, slab, 32 dims
            const uint32_t slab = (j >> 2) & 1u, kk = (j & 3u) * 2u;
            const uint64_t a = desc(qa + (j >> 3) * ((BLK * D) >> 4) + slab * (SLAB >> 4) + kk), k = desc(kb + slab * (cf::HAVE >> 5) + kk);
            if (PAIR) mma_ss_pair(d_tmem, a, k, IDESC, j == 0 ? i != 0u : 1u); else mma_ss(d_tmem, a, k, IDESC, j == 0 ? i != 0u : 1u);
          }
          commit(B_K_EMPTY + st);
          if (i + 1 == units && (D != 256 || n >= n_cached)) commit(B_S_FULL + ((D == 256 ? n - n_cached : n) & 1u));
        }
        __syncwarp();
      }
      return true;
    };
    ok = ok && issue_qk(0);
    for (uint32_t n = 0; ok && n < n_local; ++n) {
      // (S of tile n + 1 goes where P of tile n - 1 was read by MMAs issued before)
      if (n + 1 < n_local && !issue_qk(n + 1)) break;
      const uint32_t units = n < n_cached ? 1u : 2u;
      // V rows of a canvas tile behind its last whole step of 32 keys were never written
      const uint32_t keys = n < n_cached ? BLK : p.C - (n0 + n - ts.nA) * BLK;
      const uint32_t pt = tmem + T_S + (n & 1u) * 128u;
      for (uint32_t i = 0; i < units; ++i, ++uv) {
        ok = __all_sync(0xffffffffu, i == 0 ? bar_wait<PAIR>(bar(B_P_FULL + (n & 1u)), (n >> 1) & 1u, abort_flag)
                                            : bar_wait<PAIR>(bar(B_V2_FULL), (n - n_cached) & 1u, abort_flag));
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t st = uv % cf::NV, vb = dv + st * (cf::HAVE >> 4);
#pragma unroll
          for (uint32_t ks = 0; ks < 4; ++ks) {
            if (ks != 0 && ks * 32u >= keys) break;
            const uint64_t v = desc(vb + ks * (4096u >> 4));
            const uint32_t add = ks == 0 ? (n | i) != 0u : 1u;
#pragma unroll
            for (uint32_t t = 0; t < TERMS; ++t) {
              const uint32_t a = pt + t * 32u + ks * 8u, on = t == 0 ? add : 1u;
              if (PAIR) mma_ts_pair(tmem + T_O, a, v, IDESC_P, on); else mma_ts(tmem + T_O, a, v, IDESC_P, on);
            }
          }
          commit(B_V_EMPTY + st);
          if (n + 1 == n_local && i + 1 == units) commit(B_O);
        }
        __syncwarp();
      }
    }
  }

  // ------------------------------------------------------------------ output (softmax warps)
  if (warp < SM_WARPS) {
    bool have = __all_sync(0xffffffffu, n_local > 0 && !*abort_flag);
    if (have) {
      have = __all_sync(0xffffffffu, bar_wait(bar(B_O), 0u, abort_flag));
      tc_fence_after();
    }
    // the row's sum is its four threads' sums
    bar_sync_id(1u + quarter, 128u);
    xch[part * BLK + r] = l_run;
    bar_sync_id(1u + quarter, 128u);
    const float l = (xch[r] + xch[BLK + r]) + (xch[2 * BLK + r] + xch[3 * BLK + r]);
    const bool direct = sq.n_splits == 1;
    const float mul = direct ? (l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l)) : 1.0f;   // a sum that is NaN stays one
    const uint32_t t_lane = tmem + ((quarter * 32u) << 16);
    // 32 x 32 pieces through a padded tile of dead shared memory: every store instruction writes whole lines
    float* tile = reinterpret_cast<float*>(smem) + warp * (32 * 36);
    size_t row_k[8];
    bool valid_k[8];
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) {
      const uint32_t rk = quarter * 32u + k * 4u + (lane >> 3), Rk = mt * BLK + rk;
      valid_k[k] = Rk < rows_per_head;
      const uint32_t Rc = valid_k[k] ? Rk : 0u;
      row_k[k] = direct ? ((size_t(b) * p.C + Rc / p.G) * p.Hq + kvh * p.G + Rc % p.G) * D + z * 256u
                        : (size_t(slot) * BLK + rk) * 256u;
    }
#pragma unroll 1
    for (uint32_t cc = 0; cc < 2; ++cc) {
      const uint32_t col = part * 64u + cc * 32u;
      uint32_t o[32];
      if (have) {
        tmem_ld32(t_lane + T_O + col, o);
        tmem_wait_ld();
      } else {
#pragma unroll
        for (uint32_t e = 0; e < 32; ++e) o[e] = 0u;
      }
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e)
        *reinterpret_cast<float4*>(tile + lane * 36u + e * 4u) =
            make_float4(__uint_as_float(o[e * 4]) * mul, __uint_as_float(o[e * 4 + 1]) * mul, __uint_as_float(o[e * 4 + 2]) * mul,
                        __uint_as_float(o[e * 4 + 3]) * mul);
      __syncwarp();
#pragma unroll
      for (uint32_t k = 0; k < 8; ++k) {
        const float4 v = *reinterpret_cast<const float4*>(tile + (k * 4u + (lane >> 3)) * 36u + (lane & 7u) * 4u);
        if (!valid_k[k]) continue;
        const size_t at = row_k[k] + col + (lane & 7u) * 4u;
        if (direct)
          *reinterpret_cast<uint2*>(p.out + at) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
        else
          *reinterpret_cast<float4*>(p.ws_o + at) = v;
      }
      __syncwarp();
    }
    const uint32_t R = mt * BLK + r;
    if (part == 0 && R < rows_per_head) {
      if (!direct)
        p.ws_ml[size_t(slot) * BLK + r] = make_float2(m_used, l);
      else if (p.lse != nullptr && z == 0)
        p.lse[(size_t(b) * p.C + R / p.G) * p.Hq + kvh * p.G + R % p.G] =
            l == 0.f ? -INFINITY : (m_used - LIFT + log2f(l)) * 0.6931471805599453f;
    }
  }

  if (*abort_flag) {
    if (tid == 0) dev_status_set(p.status, DG_DEV_WAIT_TIMEOUT, KID_ATTN, blockIdx.x, n_local);
    if (warp == W_K && lane == 0) {
      const long long c0 = clock64();
      while (clock64() - c0 < 2000000ll) {}   // ~1 ms: far longer than any load in flight
    }
  }
  tc_fence_before();
  if (PAIR) {
    cluster_sync_all();   // the leader's products read this CTA's memory, and its barriers take arrivals from here
    if (warp == W_MMA) tmem_dealloc_pair(tmem, 512);
  } else {
    __syncthreads();
    if (warp == W_MMA) tmem_dealloc(tmem, 512);
  }
}

// Splits of a row joined: a row's 256 columns by WARPS warps, each a run of the splits in order, then the warps in order.  A
// warp's sums stand at the largest reference of its own splits until the warps meet: one round trip to memory.  One warp a row
// where the splits are few (and the rows many).  A split without keys has m = -inf and l = 0.
template <uint32_t WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? 256 : WARPS * 32) dg_kv8_merge_kernel(const __grid_constant__ AttnParams8 p) {
  __shared__ float part[WARPS][256];
  __shared__ float2 ml_w[WARPS];
  grid_launch_dependents();
  grid_wait();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, w = warp % WARPS, b = blockIdx.y, KU = p.D / 256u;
  const Seq& sq = p.seq[b];
  const uint32_t x = WARPS == 1 ? blockIdx.x * 8u + warp : blockIdx.x;
  if (sq.n_splits == 1 || x >= p.C * p.Hq * KU) return;      // (whole CTAs where warps work together)
  const uint32_t z = x % KU, row = x / KU, i = row / p.Hq, h = row % p.Hq, kvh = h / p.G;
  const uint32_t R = i * p.G + h % p.G, mt = R / BLK, r = R % BLK, S = sq.n_splits;
  const uint32_t stride = p.Hkv * p.MT * KU, first = sq.first_cta + (kvh * p.MT + mt) * KU + z;
  float m = -INFINITY, l = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const uint32_t s1 = (w + 1) * S / WARPS;
  for (uint32_t s = w * S / WARPS; s < s1; s += 4) {
    float2 ml[4];
    float4 o[4][2];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      const size_t at = size_t(first + (s + k < s1 ? s + k : s) * stride) * BLK + r;
      const float4* src = reinterpret_cast<const float4*>(p.ws_o + at * 256u + lane * 8u);
      ml[k] = s + k < s1 ? p.ws_ml[at] : make_float2(-INFINITY, 0.f);
      o[k][0] = src[0];
      o[k][1] = src[1];
    }
    const float top = fmaxf(fmaxf(m, ml[0].x), fmaxf(ml[1].x, fmaxf(ml[2].x, ml[3].x)));
    const float keep = m == -INFINITY ? 0.f : fast_exp2(m - top);
    l *= keep;
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) acc[e] *= keep;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      if (ml[k].x == -INFINITY && ml[k].y == 0.f) continue;
      const float f = ml[k].x == -INFINITY ? ml[k].y : fast_exp2(ml[k].x - top);   // no reference but a sum: not a number
      l = fmaf(f, ml[k].y, l);
      acc[0] = fmaf(f, o[k][0].x, acc[0]); acc[1] = fmaf(f, o[k][0].y, acc[1]); acc[2] = fmaf(f, o[k][0].z, acc[2]); acc[3] = fmaf(f, o[k][0].w, acc[3]);
      acc[4] = fmaf(f, o[k][1].x, acc[4]); acc[5] = fmaf(f, o[k][1].y, acc[5]); acc[6] = fmaf(f, o[k][1].z, acc[6]); acc[7] = fmaf(f, o[k][1].w, acc[7]);
    }
    m = top;
  }
  const size_t orow = (size_t(b) * p.C + i) * p.Hq + h;
  if (WARPS > 1) {
    *reinterpret_cast<float4*>(&part[warp][lane * 8u]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    *reinterpret_cast<float4*>(&part[warp][lane * 8u + 4u]) = make_float4(acc[4], acc[5], acc[6], acc[7]);
    if (lane == 0) ml_w[warp] = make_float2(m, l);
    __syncthreads();
    if (threadIdx.x >= 256u) return;
    float top = -INFINITY;
#pragma unroll
    for (uint32_t k = 0; k < WARPS; ++k) top = fmaxf(top, ml_w[k].x);
    float sum = 0.f, y = 0.f;
#pragma unroll
    for (uint32_t k = 0; k < WARPS; ++k) {
      if (ml_w[k].x == -INFINITY && ml_w[k].y == 0.f) continue;
      const float f = ml_w[k].x == -INFINITY ? ml_w[k].y : fast_exp2(ml_w[k].x - top);
      sum = fmaf(f, ml_w[k].y, sum);
      y = fmaf(f, part[k][threadIdx.x], y);
    }
    m = top;
    l = sum;
    const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
    p.out[orow * p.D + z * 256u + threadIdx.x] = __float2bfloat16(y * inv);
  } else {
    const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
    *reinterpret_cast<uint4*>(p.out + orow * p.D + z * 256u + lane * 8u) =
        make_uint4(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv),
                   pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv));
  }
  if (p.lse != nullptr && z == 0 && w == 0 && lane == 0) p.lse[orow] = l == 0.f ? -INFINITY : (m - LIFT + log2f(l)) * 0.6931471805599453f;
}

template <uint32_t D, bool PAIR>
static cudaError_t configure_one() {
  return cudaFuncSetAttribute(dg_kv8_attn_kernel<D, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(Cfg<D, PAIR>::SMEM));
}
cudaError_t configure_attn() {
  cudaError_t e = configure_one<256, false>();
  if (e == cudaSuccess) e = configure_one<512, false>();
  if (e == cudaSuccess) e = configure_one<512, true>();
  return e;
}

cudaError_t launch_merge(const AttnParams8& p, uint32_t most_splits, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const uint32_t rows = p.C * p.Hq * (p.D / 256u);
  if (most_splits > 4) {
    cfg.gridDim = dim3(rows, p.n_seq);
    if (most_splits > 16) {
      cfg.blockDim = dim3(512);
      return cudaLaunchKernelEx(&cfg, dg_kv8_merge_kernel<16>, p);
    }
    return cudaLaunchKernelEx(&cfg, dg_kv8_merge_kernel<8>, p);
  }
  cfg.gridDim = dim3((rows + 7u) / 8u, p.n_seq);
  return cudaLaunchKernelEx(&cfg, dg_kv8_merge_kernel<1>, p);
}

template <uint32_t D, bool PAIR>
static cudaError_t launch_one(const AttnParams8& p, uint32_t n_ctas, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n_ctas);
  cfg.blockDim = dim3(Cfg<D, PAIR>::THREADS);
  cfg.dynamicSmemBytes = Cfg<D, PAIR>::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, dg_kv8_attn_kernel<D, PAIR>, p);
}
cudaError_t launch_attention(const AttnParams8& p, bool pair, uint32_t n_ctas, uint32_t most_splits, cudaStream_t st) {
  const cudaError_t e = p.D == 256 ? launch_one<256, false>(p, n_ctas, st) : pair ? launch_one<512, true>(p, n_ctas, st) : launch_one<512, false>(p, n_ctas, st);
  return e != cudaSuccess || most_splits == 1 ? e : launch_merge(p, most_splits, st);
}

}  // namespace kv8
}  // namespace dg
