// What each cached key drew of the softmax of a step's rows:  w[t] = decay * w[t] + sum over rows of e^(s - lse).
//
// The scores are computed transposed, S^T = K Q^T: the keys are the 128 lanes of the accumulator and the rows its columns,
// so that a key's sum is an addition in one thread's register for every row and nothing crosses lanes.  A CTA keeps 64 KB
// of keys in shared memory (256 keys of 256 dims, or 128 of 512) and streams all query rows past them in 64 KB stages (two
// terms, as in the attention kernel); rows come out of L2, keys out of HBM once.  Per 128 keys, 128 rows and 256 dims:
// 1,024 cycles of MMA, 16,384 exponentials (1,024 cycles), 32 bytes a cycle of rows.
// Every key belongs to one thread of one CTA, or of a fixed number of CTAs whose sums are added in order: no atomics.
#include "dg_kv8.cuh"

namespace dg {
namespace kv8 {

template <uint32_t D> struct WCfg {
  static constexpr uint32_t KT = 512 / D, NR = D == 256 ? 128 : 64;      // key tiles of a CTA, rows of a stage
  static constexpr uint32_t K_BYTES = KT * BLK * D, STAGE = 2 * NR * D;  // 64 KB each
  static constexpr uint32_t O_Q = K_BYTES, O_C = O_Q + 2 * STAGE, O_R = O_C + 4 * NR * 8, O_BAR = O_R + 4 * BLK * 4;
  static constexpr uint32_t SMEM = O_BAR + 9 * 8 + 8;
  static constexpr uint32_t COLS = KT * NR / 4;                          // score columns of an epilogue thread
  static constexpr uint32_t TM_COLS = 2 * KT * NR;
};
constexpr uint32_t W_EPI = 16, WW_LOAD = 16, WW_MMA = 17, W_THREADS = 18 * 32;
enum { WB_K = 0, WB_Q_FULL = 1, WB_Q_EMPTY = 3, WB_S_FULL = 5, WB_S_EMPTY = 7 };

template <uint32_t D>
__global__ void __launch_bounds__(W_THREADS, 1) dg_kv8_weights_kernel(const __grid_constant__ WeightParams p) {
  typedef WCfg<D> cf;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t s0 = smem_u32(smem);
  volatile uint32_t* ctl = reinterpret_cast<volatile uint32_t*>(smem + cf::O_BAR + 9 * 8);
  volatile uint32_t* abort_flag = &ctl[0];
  auto bar = [&](uint32_t i) { return s0 + cf::O_BAR + i * 8u; };
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  const uint32_t kvh = blockIdx.y, rs = blockIdx.z;
  grid_launch_dependents();
  if (s0 & 1023u) {
    if (tid == 0) dev_status_set(p.status, DG_DEV_SMEM_LAYOUT, KID_WEIGHTS, blockIdx.x, s0);
    return;
  }
  if (tid == 0) {
    ctl[0] = 0u;
    for (uint32_t i = 0; i < 9; ++i) mbar_init(bar(i), i >= WB_S_EMPTY ? W_EPI : 1u);
    fence_mbar_init();
  }
  if (warp == WW_MMA) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(&ctl[1])), cf::TM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl[1];
  grid_wait();

  const uint32_t rows = p.C * p.G, n_blocks = (p.n_keys + BLK - 1) / BLK;
  const uint32_t first = blockIdx.x * cf::KT, have = n_blocks - first < cf::KT ? n_blocks - first : cf::KT;
  MaskParams mk = {};
  mk.kv_len = mk.pre_hi = mk.can_hi = p.n_keys;
  mk.mode = p.mode;
  mk.windowed = p.windowed;
  mk.wm1 = p.wm1;
  const uint32_t all_steps = (rows + cf::NR - 1) / cf::NR;
  const uint32_t st0 = uint32_t(uint64_t(all_steps) * rs / p.row_splits);
  uint32_t st1 = uint32_t(uint64_t(all_steps) * (rs + 1) / p.row_splits);
  if ((first + have) * BLK <= mask_row_lo(mk, 0)) st1 = st0;   // nobody sees these keys
  const uint32_t n_steps = st1 - st0;
  const size_t q_head = size_t(kvh) * p.MT;
  float* red = reinterpret_cast<float*>(smem + cf::O_R);

  if (warp < W_EPI) {
    const uint32_t quarter = warp & 3u, g = warp >> 2;
    const uint32_t kt = g * cf::COLS / cf::NR, col0 = g * cf::COLS % cf::NR;
    const uint32_t key = quarter * 32u + lane, t = (first + kt) * BLK + key;
    const bool live = t < p.n_keys;
    const float kscale = kt < have ? pow2i(p.exps[size_t(kvh) * p.blocks + first + kt].x) : 0.f;
    // keys that some row does not see: a look at each row's window
    const bool edge = (first + kt) * BLK < mask_row_lo(mk, p.C - 1);
    float acc[2] = {0.f, 0.f};
    for (uint32_t n = 0; n < n_steps; ++n) {
      const uint32_t sb = n & 1u;
      if (!__all_sync(0xffffffffu, bar_wait(bar(WB_S_FULL + sb), (n >> 1) & 1u, abort_flag))) break;
      tc_fence_after();
      const float4* cst = reinterpret_cast<const float4*>(smem + cf::O_C + ((n & 3u) * cf::NR + col0) * 8u);
      const uint32_t src = tmem + ((quarter * 32u) << 16) + sb * (cf::KT * cf::NR) + kt * cf::NR + col0;
      constexpr uint32_t W = cf::COLS < 32 ? cf::COLS : 32;
#pragma unroll 1
      for (uint32_t c = 0; c < cf::COLS; c += W) {
        uint32_t s[W];
        if constexpr (W == 32) tmem_ld32(src + c, s); else tmem_ld16(src + c, s);
        tmem_wait_ld();
        if (c + W >= cf::COLS) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(WB_S_EMPTY + sb));
        }
        if (!edge) {
#pragma unroll
          for (uint32_t e = 0; e < W; e += 2) {
            const float4 k = cst[(c + e) >> 1];   // (factor, -lse) of two rows, one broadcast
            acc[0] += fast_exp2(fmaf(__uint_as_float(s[e]) * kscale, k.x, k.y));
            acc[1] += fast_exp2(fmaf(__uint_as_float(s[e + 1]) * kscale, k.z, k.w));
          }
        } else {
#pragma unroll
          for (uint32_t e = 0; e < W; e += 2) {
            const float4 k = cst[(c + e) >> 1];
            const uint32_t R = (st0 + n) * cf::NR + col0 + c + e;
            if (t >= mask_row_lo(mk, R / p.G)) acc[0] += fast_exp2(fmaf(__uint_as_float(s[e]) * kscale, k.x, k.y));
            if (t >= mask_row_lo(mk, (R + 1) / p.G)) acc[1] += fast_exp2(fmaf(__uint_as_float(s[e + 1]) * kscale, k.z, k.w));
          }
        }
      }
    }
    red[g * BLK + key] = acc[0] + acc[1];
    asm volatile("bar.sync 1, %0;" ::"n"(W_EPI * 32) : "memory");
    // the threads that share a key: the column groups of its tile
    constexpr uint32_t PER = 4 / cf::KT;
    if (g % PER == 0 && live && kt < have && !*abort_flag) {
      float sum = 0.f;
#pragma unroll
      for (uint32_t i = 0; i < PER; ++i) sum += red[(g + i) * BLK + key];
      if (p.row_splits > 1) {
        p.part[(size_t(rs) * p.Hkv + kvh) * p.n_keys + t] = sum;
      } else {
        float* w = p.w + size_t(kvh) * p.ld + t;
        *w = p.decay != 0.f ? fmaf(p.decay, *w, sum) : sum;
      }
    }
  } else if (warp == WW_LOAD) {
    if (lane == 0 && n_steps > 0) {
      mbar_expect_tx(bar(WB_K), have * BLK * D);
      const uint8_t* k = p.k + (size_t(kvh) * p.blocks + first) * BLK * D;
      for (uint32_t o = 0; o < have * BLK * D; o += UNIT) bulk_load(s0 + o, k + o, UNIT, bar(WB_K));
      for (uint32_t n = 0; n < n_steps; ++n) {
        const uint32_t sb = n & 1u, full = bar(WB_Q_FULL + sb), step = st0 + n;
        if (n > 1 && !bar_wait(bar(WB_Q_EMPTY + sb), ((n - 2) >> 1) & 1u, abort_flag)) break;
        // the constants' slot was last read for step n - 4, which S^T of step n - 2 waited for
        mbar_expect_tx(full, cf::STAGE + cf::NR * 8u);
        const uint32_t dst = s0 + cf::O_Q + sb * cf::STAGE;
        const uint32_t R0 = step * cf::NR, mt = R0 / BLK;
        const uint8_t* q = p.q_codes + (q_head + mt) * 2u * BLK * D;
        if (cf::NR == BLK) {
          for (uint32_t o = 0; o < cf::STAGE; o += UNIT) bulk_load(dst + o, q + o, UNIT, full);
        } else {
          for (uint32_t sl = 0; sl < 2 * D / 128; ++sl)
            bulk_load(dst + sl * cf::NR * 128u, q + sl * SLAB + (R0 % BLK) * 128u, cf::NR * 128u, full);
        }
        bulk_load(s0 + cf::O_C + (n & 3u) * cf::NR * 8u, p.q_row + q_head * BLK + R0, cf::NR * 8u, full);
      }
    }
  } else if (n_steps > 0) {
    constexpr uint32_t IDESC = idesc_f8(128, cf::NR, 0, 0);
    const uint64_t dk = umma_smem_desc(s0, 16, 1024), dq = umma_smem_desc(s0 + cf::O_Q, 16, 1024);
    bool ok = __all_sync(0xffffffffu, bar_wait(bar(WB_K), 0u, abort_flag));
    for (uint32_t n = 0; ok && n < n_steps; ++n) {
      const uint32_t sb = n & 1u;
      if (n > 1 && !__all_sync(0xffffffffu, bar_wait(bar(WB_S_EMPTY + sb), ((n - 2) >> 1) & 1u, abort_flag))) break;
      if (!__all_sync(0xffffffffu, bar_wait(bar(WB_Q_FULL + sb), (n >> 1) & 1u, abort_flag))) break;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll 1
        for (uint32_t kt = 0; kt < cf::KT; ++kt) {
          const uint32_t d_tmem = tmem + sb * (cf::KT * cf::NR) + kt * cf::NR;
#pragma unroll 1
          for (uint32_t ts = 0; ts < 2 * D / 128; ++ts) {   // term and slab of the rows
            const uint64_t qb = dq + uint64_t((sb * cf::STAGE + ts * cf::NR * 128u) >> 4);
            const uint64_t ka = dk + uint64_t((kt * BLK * D + (ts % (D / 128)) * SLAB) >> 4);
#pragma unroll
            for (uint32_t kk = 0; kk < 4; ++kk) mma_ss(d_tmem, ka + kk * 2u, qb + kk * 2u, IDESC, (ts | kk) != 0u);
          }
        }
        umma_commit(bar(WB_Q_EMPTY + sb));
        umma_commit(bar(WB_S_FULL + sb));
      }
      __syncwarp();
    }
  }

  if (*abort_flag) {
    if (tid == 0) dev_status_set(p.status, DG_DEV_WAIT_TIMEOUT, KID_WEIGHTS, blockIdx.x, n_steps);
    if (warp == WW_LOAD && lane == 0) {
      const long long c0 = clock64();
      while (clock64() - c0 < 2000000ll) {}
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == WW_MMA) tmem_dealloc(tmem, cf::TM_COLS);
}

__global__ void __launch_bounds__(256) dg_kv8_weights_sum_kernel(const __grid_constant__ WeightParams p) {
  grid_launch_dependents();
  grid_wait();
  const uint32_t t = blockIdx.x * 256u + threadIdx.x, kvh = blockIdx.y;
  if (t >= p.n_keys) return;
  float sum = 0.f;
  for (uint32_t s = 0; s < p.row_splits; ++s) sum += p.part[(size_t(s) * p.Hkv + kvh) * p.n_keys + t];
  float* w = p.w + size_t(kvh) * p.ld + t;
  *w = p.decay != 0.f ? fmaf(p.decay, *w, sum) : sum;
}

cudaError_t configure_weights() {
  cudaError_t e = cudaFuncSetAttribute(dg_kv8_weights_kernel<256>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(WCfg<256>::SMEM));
  if (e == cudaSuccess) e = cudaFuncSetAttribute(dg_kv8_weights_kernel<512>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(WCfg<512>::SMEM));
  return e;
}

cudaError_t launch_weights(const WeightParams& p, uint32_t D, cudaStream_t st) {
  const uint32_t kt = 512 / D, blocks = (p.n_keys + BLK - 1) / BLK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((blocks + kt - 1) / kt, p.Hkv, p.row_splits);
  cfg.blockDim = dim3(W_THREADS);
  cfg.dynamicSmemBytes = D == 256 ? WCfg<256>::SMEM : WCfg<512>::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = D == 256 ? cudaLaunchKernelEx(&cfg, dg_kv8_weights_kernel<256>, p) : cudaLaunchKernelEx(&cfg, dg_kv8_weights_kernel<512>, p);
  if (e != cudaSuccess || p.row_splits == 1) return e;
  cfg.gridDim = dim3((p.n_keys + 255u) / 256u, p.Hkv);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, dg_kv8_weights_sum_kernel, p);
}

}  // namespace kv8
}  // namespace dg
