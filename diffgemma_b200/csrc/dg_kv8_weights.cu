// What each cached key drew of the softmax of a step's rows:  w[t] = decay * w[t] + sum over rows of e^(s - lse).
//
// The scores are computed transposed, S^T = K Q^T: the keys are the 128 lanes of the accumulator and the rows its columns,
// so that a key's sum is an addition in one thread's register for every row and nothing crosses lanes.  A CTA keeps 64 KB
// of keys in shared memory (256 keys of 256 dims, or 128 of 512) and streams all query rows past them in 64 KB stages (two
// terms, as in the attention kernel); rows come out of L2, keys out of HBM once.
// The work is a line of units, (head, run of keys, stage of rows): a CTA a run, or the line cut evenly and the runs at the cuts
// shared.  Every key's sum is one thread's, or of a few CTAs whose sums a second launch adds in order: no atomics.
//
// What bounds it: 256 keys, 128 rows and 256 dims are 2,048 cycles of MMA, and 320 KB through shared memory (the operands of 32
// MMAs, 8 KB each, and the stage's copy: 2,560 cycles at 128 bytes a cycle); 2,600 to 2,800 measured (32,768 keys of 2 heads,
// 2,048 rows: 60 us; with part of the exponentials on the FMA units as long).
// head_dim 512 alone has room for stages of 64 rows only, and an MMA of 64 columns takes 48 cycles, one of 128 takes 64.  From
// 512 rows on two CTAs make a pair there (cta_group::2): 128 keys each, 128 rows a stage, of which each brings 64.  us alone / in
// pairs, 2 KV heads, 2,048 rows: 2,000 keys 24.3 / 25.4, 8,191 39.1 / 33.2, 32,768 124.9 / 103.2; 512 rows: 49.1 / 48.2; 128
// rows: 25.7 / 30.5.  head_dim 256 in pairs: 60.2 / 64.6.
#include "dg_kv8.cuh"

namespace dg {
namespace kv8 {

constexpr uint32_t W_EPI = 16, WW_LOAD = 16, WW_MMA = 17, W_THREADS = 18 * 32;
// WB_Q_FULL of a stage counts its bytes and the sixteen warps that have read the scores of the stage before last: one wait for
// the MMA warp.  WB_S_FULL says that the scores are there and the stage is free.
// WB_C_EMPTY of each of the four places of row constants counts the warps that are done with them: they hold on to them longer than to
// the scores, by any number of steps where a window's edge makes them look at every row.
enum { WB_K = 0, WB_Q_FULL = 1, WB_S_FULL = 3, WB_C_EMPTY = 5, W_BARS = 9 };

template <uint32_t D, bool PAIR> struct WCfg {
  static_assert(!PAIR || D == 512, "pairs: see above");
  static constexpr uint32_t KT = 512 / D, NR = D == 256 || PAIR ? 128 : 64;   // key tiles of a CTA, rows of a stage
  static constexpr uint32_t RUN = PAIR ? 2 * KT : KT, HR = PAIR ? NR / 2 : NR;   // key tiles of a run, rows of a stage in this CTA
  static constexpr uint32_t K_BYTES = KT * BLK * D, STAGE = 2 * HR * D;
  static constexpr uint32_t O_Q = K_BYTES, O_C = O_Q + 2 * STAGE, O_R = O_C + 4 * NR * 8, O_BAR = O_R + 4 * BLK * 4;
  static constexpr uint32_t SMEM = O_BAR + W_BARS * 8 + 8;
  static constexpr uint32_t COLS = KT * NR / 4;                          // score columns of an epilogue thread
  static constexpr uint32_t TM_COLS = 2 * KT * NR;
};
template <uint32_t D, bool PAIR>
__global__ void __launch_bounds__(W_THREADS, 1) dg_kv8_weights_kernel(const __grid_constant__ WeightParams p) {
  typedef WCfg<D, PAIR> cf;
  const uint32_t rank = PAIR ? blockIdx.x & 1u : 0u, cta = PAIR ? blockIdx.x >> 1 : blockIdx.x, ctas = PAIR ? gridDim.x >> 1 : gridDim.x;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t s0 = smem_u32(smem);
  volatile uint32_t* ctl = reinterpret_cast<volatile uint32_t*>(smem + cf::O_BAR + W_BARS * 8);
  volatile uint32_t* abort_flag = &ctl[0];
  auto bar = [&](uint32_t i) { return s0 + cf::O_BAR + i * 8u; };
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  grid_launch_dependents();
  if (s0 & 1023u) {
    if (tid == 0) dev_status_set(p.status, DG_DEV_SMEM_LAYOUT, KID_WEIGHTS, blockIdx.x, s0);
    return;
  }
  if (tid == 0) {
    ctl[0] = 0u;
    // the leader of a pair counts the other CTA's share as well; there Q_FULL counts bytes alone
    const uint32_t both = PAIR && rank == 0u ? 2u : 1u;
    mbar_init(bar(WB_K), both);
    for (uint32_t i = 0; i < 2; ++i) {
      mbar_init(bar(WB_Q_FULL + i), rank != 0u ? 1u : both * (W_EPI + 1u));
      mbar_init(bar(WB_S_FULL + i), 1u);
    }
    for (uint32_t i = 0; i < 4; ++i) mbar_init(bar(WB_C_EMPTY + i), W_EPI);
    fence_mbar_init();
  }
  if (warp == WW_MMA) {
    if (PAIR) {
      tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(&ctl[1])), cf::TM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(const_cast<uint32_t*>(&ctl[1])), cf::TM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if (PAIR) cluster_sync_all(); else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl[1];
  grid_wait();

  const uint32_t rows = p.C * p.G, n_blocks = (p.n_keys + BLK - 1) / BLK, runs = (n_blocks + cf::RUN - 1) / cf::RUN - p.run0;
  const uint32_t steps = (rows + cf::NR - 1) / cf::NR;
  MaskParams mk = {};
  mk.kv_len = mk.pre_hi = mk.can_hi = p.n_keys;
  mk.mode = p.mode;
  mk.windowed = p.windowed;
  mk.wm1 = p.wm1;
  const uint64_t units = uint64_t(p.Hkv) * runs * steps;
  const uint64_t u0 = units * cta / ctas, u1 = units * (cta + 1u) / ctas;
  float* red = reinterpret_cast<float*>(smem + cf::O_R);
  // a CTA's (a pair's) pieces: f(first stage, last + 1, KV head, run, first block, blocks, piece) for each run of keys that its stretch touches
  auto each_piece = [&](auto f) {
    uint32_t piece = 0;
    for (uint64_t u = u0; u < u1; ++piece) {
      const uint32_t run = uint32_t(u / steps), st0 = uint32_t(u % steps);
      const uint64_t end = u1 < uint64_t(run + 1) * steps ? u1 : uint64_t(run + 1) * steps;
      const uint32_t first = (p.run0 + run % runs) * cf::RUN + rank * cf::KT, left = first < n_blocks ? n_blocks - first : 0u;
      if (!f(st0, st0 + uint32_t(end - u), run, first, left < cf::KT ? left : cf::KT, piece)) break;
      u = end;
    }
  };

  if (warp < W_EPI) {
    const uint32_t quarter = warp & 3u, g = warp >> 2;
    const uint32_t kt = g * cf::COLS / cf::NR, col0 = g * cf::COLS % cf::NR;
    const uint32_t key = quarter * 32u + lane;
    constexpr uint32_t W = cf::COLS < 32 ? cf::COLS : 32, CH = cf::COLS / W;
    uint32_t n = 0;
    // this warp has read the scores: for the stage after next
    auto scores_read = [&](uint32_t sb) {
      if (lane != 0) return;
      if (PAIR && rank != 0u) mbar_arrive_remote(dsmem_addr(bar(WB_Q_FULL + sb), 0u)); else mbar_arrive(bar(WB_Q_FULL + sb));
    };
    scores_read(0);
    scores_read(1);
    // keys ahead of every row's window
    if (p.decay != 1.0f) {
      const uint32_t behind = p.run0 * cf::RUN * BLK;
      for (uint64_t x = uint64_t(blockIdx.x) * (W_EPI * 32) + tid; x < uint64_t(behind) * p.Hkv; x += uint64_t(gridDim.x) * (W_EPI * 32)) {
        float* w = p.w + x / behind * p.ld + x % behind;
        *w = p.decay != 0.f ? p.decay * *w : 0.f;
      }
    }
    each_piece([&](uint32_t st0, uint32_t st1, uint32_t run, uint32_t first, uint32_t have, uint32_t) -> bool {
      const uint32_t kvh = run / runs;
      const uint32_t t = (first + kt) * BLK + key;
      const float kscale = kt < have ? pow2i(p.exps[size_t(kvh) * p.blocks + first + kt].x) : 0.f;
      // keys that some row does not see: a look at each row's window
      const bool edge = (first + kt) * BLK < mask_row_lo(mk, p.C - 1);
      uint64_t acc = 0ull;
      const uint64_t ks2 = pack_f32x2(kscale, kscale);
      bool ok = true;
      for (uint32_t st = st0; st < st1; ++st, ++n) {
        const uint32_t sb = n & 1u;
        // (a wait that gave up ends nothing here: all warps go through the same barriers, and nothing is stored)
        if (!__all_sync(0xffffffffu, bar_wait(bar(WB_S_FULL + sb), (n >> 1) & 1u, abort_flag))) ok = false;
        tc_fence_after();
        const ulonglong2* cst = reinterpret_cast<const ulonglong2*>(smem + cf::O_C + (n & 3u) * cf::NR * 8u) + col0 / 2u;
        const uint32_t src = tmem + ((quarter * 32u) << 16) + sb * (cf::KT * cf::NR) + kt * cf::NR + col0;
        uint32_t s[CH][W];
#pragma unroll
        for (uint32_t c = 0; c < CH; ++c) {
          if constexpr (W == 32) tmem_ld32(src + c * W, s[c]); else tmem_ld16(src + c * W, s[c]);
        }
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        scores_read(sb);
        auto weight = [&](uint32_t c, uint32_t e) -> uint64_t {
          const ulonglong2 k = cst[(c * W + e) >> 1];      // factors and -lse of two rows, one broadcast
          float x0, x1;
          unpack_f32x2(fma_f32x2(mul_f32x2(pack_f32x2(__uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1])), ks2), k.x, k.y), x0, x1);
          return pack_f32x2(fast_exp2(x0), fast_exp2(x1));
        };
        if (!edge) {
#pragma unroll
          for (uint32_t c = 0; c < CH; ++c)
#pragma unroll
            for (uint32_t e = 0; e < W; e += 2) acc = add_f32x2(acc, weight(c, e));
        } else {
#pragma unroll 1
          for (uint32_t c = 0; c < CH; ++c)
#pragma unroll
            for (uint32_t e = 0; e < W; e += 2) {
              const uint32_t R = st * cf::NR + col0 + c * W + e;
              float x0, x1;
              unpack_f32x2(c == 0 ? weight(0, e) : weight(CH - 1, e), x0, x1);
              x0 = t >= mask_row_lo(mk, R / p.G) ? x0 : 0.f;
              x1 = t >= mask_row_lo(mk, (R + 1) / p.G) ? x1 : 0.f;
              acc = add_f32x2(acc, pack_f32x2(x0, x1));
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(WB_C_EMPTY + (n & 3u)));
      }
      float a, b;
      unpack_f32x2(acc, a, b);
      red[g * BLK + key] = a + b;
      asm volatile("bar.sync 1, %0;" ::"n"(W_EPI * 32) : "memory");
      // the threads that share a key: the column groups of its tile
      constexpr uint32_t PER = 4 / cf::KT;
      if (g % PER == 0 && t < p.n_keys && kt < have && ok && !*abort_flag) {
        float sum = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) sum += red[(g + i) * BLK + key];
        if (st0 != 0 || st1 != steps) {
          // a piece of the run's stages: its place is the CTA's distance from the first that has one of them
          const uint64_t at = uint64_t(run) * steps;
          const uint32_t owner = uint32_t((at * ctas + ctas) / units);   // CTA with the run's first stage, or the one after
          const uint32_t lead = units * owner / ctas > at ? owner - 1u : owner;
          p.part[(size_t(cta - lead) * p.Hkv + kvh) * p.n_keys + t] = sum;
        } else {
          float* w = p.w + size_t(kvh) * p.ld + t;
          *w = p.decay != 0.f ? fmaf(p.decay, *w, sum) : sum;
        }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(W_EPI * 32) : "memory");
      return true;
    });
  } else if (warp == WW_LOAD) {
    if (lane == 0) {
      uint32_t n = 0;
      each_piece([&](uint32_t st0, uint32_t st1, uint32_t run, uint32_t first, uint32_t have, uint32_t) -> bool {
        const uint32_t kvh = run / runs;
        // the keys' place is free when the last products with them are done
        if (n != 0 && !bar_wait(bar(WB_S_FULL + ((n - 1u) & 1u)), ((n - 1u) >> 1) & 1u, abort_flag)) return false;
        mbar_expect_tx(bar(WB_K), have * BLK * D);
        const uint8_t* k = p.k + (size_t(kvh) * p.blocks + first) * BLK * D;
        for (uint32_t o = 0; o < have * BLK * D; o += UNIT) bulk_load(s0 + o, k + o, UNIT, bar(WB_K));
        for (uint32_t st = st0; st < st1; ++st, ++n) {
          const uint32_t sb = n & 1u, full = bar(WB_Q_FULL + sb);
          if (n > 1 && !bar_wait(bar(WB_S_FULL + sb), ((n - 2) >> 1) & 1u, abort_flag)) return false;
          if (n > 3 && !bar_wait(bar(WB_C_EMPTY + (n & 3u)), ((n >> 2) - 1u) & 1u, abort_flag)) return false;
          mbar_expect_tx(full, cf::STAGE + cf::NR * 8u);
          const uint32_t dst = s0 + cf::O_Q + sb * cf::STAGE;
          const uint32_t R0 = st * cf::NR, mt = R0 / BLK;
          const uint8_t* q = p.q_codes + (size_t(kvh) * p.MT + mt) * 2u * BLK * D;
          if (cf::HR == BLK) {
            for (uint32_t o = 0; o < cf::STAGE; o += UNIT) bulk_load(dst + o, q + o, UNIT, full);
          } else {
            for (uint32_t sl = 0; sl < 2 * D / 128; ++sl)
              bulk_load(dst + sl * cf::HR * 128u, q + sl * SLAB + (R0 % BLK + rank * cf::HR) * 128u, cf::HR * 128u, full);
          }
          bulk_load(s0 + cf::O_C + (n & 3u) * cf::NR * 8u, p.q_row + size_t(kvh) * p.MT * BLK + R0, cf::NR * 8u, full);
        }
        return true;
      });
    }
  } else if (PAIR && rank != 0u) {
    // tells the leader what has come here
    uint32_t n = 0;
    auto pass_on = [&](uint32_t b, uint32_t parity) -> bool {
      if (!bar_wait(bar(b), parity, abort_flag)) return false;
      mbar_arrive_cluster(dsmem_addr(bar(b), 0u));
      return true;
    };
    if (lane == 0)
      each_piece([&](uint32_t st0, uint32_t st1, uint32_t, uint32_t, uint32_t, uint32_t piece) -> bool {
        if (!pass_on(WB_K, piece & 1u)) return false;
        for (uint32_t st = st0; st < st1; ++st, ++n)
          if (!pass_on(WB_Q_FULL + (n & 1u), (n >> 1) & 1u)) return false;
        return true;
      });
  } else {
    constexpr uint32_t IDESC = idesc_f8(PAIR ? 256 : 128, cf::NR, 0, 0);
    constexpr uint32_t HI = (1024u >> 4) | (1u << 14) | (2u << 29);
    auto desc = [](uint32_t lo) { return (uint64_t(HI) << 32) | uint64_t(lo); };
    const uint32_t dk = ((s0 >> 4) & 0x3fffu) | (1u << 16), dq = (((s0 + cf::O_Q) >> 4) & 0x3fffu) | (1u << 16);
    uint32_t n = 0;
    each_piece([&](uint32_t st0, uint32_t st1, uint32_t, uint32_t, uint32_t, uint32_t piece) -> bool {
      if (!__all_sync(0xffffffffu, bar_wait<PAIR>(bar(WB_K), piece & 1u, abort_flag))) return false;
      for (uint32_t st = st0; st < st1; ++st, ++n) {
        const uint32_t sb = n & 1u;
        if (!__all_sync(0xffffffffu, bar_wait<PAIR>(bar(WB_Q_FULL + sb), (n >> 1) & 1u, abort_flag))) return false;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (uint32_t kt = 0; kt < cf::KT; ++kt) {
            const uint32_t d_tmem = tmem + sb * (cf::KT * cf::NR) + kt * cf::NR;
#pragma unroll
            for (uint32_t j = 0; j < 8 * D / 128; ++j) {   // term and slab of the rows, 32 dims
              const uint32_t ts = j >> 2, kk = j & 3u;
              const uint64_t a = desc(dk + ((kt * BLK * D + (ts % (D / 128)) * SLAB) >> 4) + kk * 2u);
              const uint64_t q = desc(dq + sb * (cf::STAGE >> 4) + ((ts * cf::HR * 128u) >> 4) + kk * 2u);
              if (PAIR) mma_ss_pair(d_tmem, a, q, IDESC, j != 0 ? 1u : 0u); else mma_ss(d_tmem, a, q, IDESC, j != 0 ? 1u : 0u);
            }
          }
          if (PAIR) commit_both(bar(WB_S_FULL + sb)); else umma_commit(bar(WB_S_FULL + sb));
        }
        __syncwarp();
      }
      return true;
    });
  }

  if (*abort_flag) {
    if (tid == 0) dev_status_set(p.status, DG_DEV_WAIT_TIMEOUT, KID_WEIGHTS, blockIdx.x, uint32_t(u1 - u0));
    if (warp == WW_LOAD && lane == 0) {
      const long long c0 = clock64();
      while (clock64() - c0 < 2000000ll) {}
    }
  }
  tc_fence_before();
  if (PAIR) {
    cluster_sync_all();   // the leader's products read this CTA's memory, and its barriers take arrivals from here
    if (warp == WW_MMA) tmem_dealloc_pair(tmem, cf::TM_COLS);
  } else {
    __syncthreads();
    if (warp == WW_MMA) tmem_dealloc(tmem, cf::TM_COLS);
  }
}

// The pieces of runs that several CTAs share, in order.
__global__ void __launch_bounds__(256) dg_kv8_weights_sum_kernel(const __grid_constant__ WeightParams p, uint32_t ctas, uint32_t run_keys, uint32_t steps) {
  grid_launch_dependents();
  grid_wait();
  const uint32_t t = blockIdx.x * 256u + threadIdx.x, kvh = blockIdx.y;
  if (t >= p.n_keys || t < p.run0 * run_keys) return;
  const uint32_t runs = (p.n_keys + run_keys - 1) / run_keys - p.run0;
  const uint64_t units = uint64_t(p.Hkv) * runs * steps, a = (uint64_t(kvh) * runs + t / run_keys - p.run0) * steps, z = a + steps;
  // CTA i has units [units * i / ctas, units * (i + 1) / ctas)
  uint32_t i = uint32_t((a * ctas + ctas) / units);
  if (units * i / ctas > a) --i;
  if (units * (i + 1) / ctas >= z) return;         // one CTA has them all
  float sum = 0.f;
  for (uint32_t k = 0; i < ctas && units * i / ctas < z; ++i, ++k) sum += p.part[(size_t(k) * p.Hkv + kvh) * p.n_keys + t];
  float* w = p.w + size_t(kvh) * p.ld + t;
  *w = p.decay != 0.f ? fmaf(p.decay, *w, sum) : sum;
}

template <uint32_t D, bool PAIR>
static cudaError_t configure_one() {
  return cudaFuncSetAttribute(dg_kv8_weights_kernel<D, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(WCfg<D, PAIR>::SMEM));
}
cudaError_t configure_weights() {
  cudaError_t e = configure_one<256, false>();
  if (e == cudaSuccess) e = configure_one<512, false>();
  if (e == cudaSuccess) e = configure_one<512, true>();
  return e;
}

template <uint32_t D, bool PAIR>
static cudaError_t launch_one(const WeightParams& p, uint32_t ctas, cudaStream_t st) {
  typedef WCfg<D, PAIR> cf;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(PAIR ? 2 * ctas : ctas);
  cfg.blockDim = dim3(W_THREADS);
  cfg.dynamicSmemBytes = cf::SMEM;
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, dg_kv8_weights_kernel<D, PAIR>, p);
  if (e != cudaSuccess || p.part == nullptr) return e;
  cfg.gridDim = dim3((p.n_keys + 255u) / 256u, p.Hkv);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, dg_kv8_weights_sum_kernel, p, ctas, cf::RUN * BLK, (p.C * p.G + cf::NR - 1) / cf::NR);
}
cudaError_t launch_weights(const WeightParams& p, uint32_t D, bool pair, uint32_t ctas, cudaStream_t st) {
  if (D == 256) return launch_one<256, false>(p, ctas, st);
  return pair ? launch_one<512, true>(p, ctas, st) : launch_one<512, false>(p, ctas, st);
}

}  // namespace kv8
}  // namespace dg
