// Eviction: the n_recent last tokens of a cache and, of those before them, the n_keep - n_recent with the largest weights
// (equal ones: lowest index), in order, into another cache.
//
// Selection, a cluster of up to eight CTAs for each head: the cut is found exactly by a radix over 32-bit order keys (digits of
// 11, 11 and 10 bits).  A thread holds its run of up to 16 tokens in registers (131,072 tokens a head; longer rows are read
// again for each digit).  A CTA counts its part; of the digit's bins each CTA adds up an eighth over the cluster and stores the
// sums to all (distributed shared memory carries every count once), then each finds the cut for itself, and each thread places
// its run by the counts ahead of it.  Moving, a CTA for each block of the new cache: 128 gathered rows of codes, whose values
// get the scale of their new block; the codes stay as they are where the scale does.
#include "dg_kv8.cuh"

namespace dg {
namespace kv8 {

constexpr uint32_t SEL_T = 1024, BINS = 2048, RUN = 16;

// larger key = larger weight; NaN below everything
__device__ __forceinline__ uint32_t weight_key(float w) { return w != w ? 0u : score_order_key(w); }

__device__ __forceinline__ uint32_t ld_dsmem(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_dsmem(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// exclusive sum over the block of two counts
__device__ __forceinline__ uint2 block_scan2(uint2 v, uint2* warp_sum, uint2* total) {
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  uint2 x = v;
#pragma unroll
  for (uint32_t o = 1; o < 32; o <<= 1) {
    const uint32_t a = __shfl_up_sync(0xffffffffu, x.x, o), b = __shfl_up_sync(0xffffffffu, x.y, o);
    if (lane >= o) { x.x += a; x.y += b; }
  }
  __syncthreads();
  if (lane == 31) warp_sum[warp] = x;
  __syncthreads();
  uint2 w = warp_sum[lane];
  uint2 y = w;
#pragma unroll
  for (uint32_t o = 1; o < 32; o <<= 1) {
    const uint32_t a = __shfl_up_sync(0xffffffffu, y.x, o), b = __shfl_up_sync(0xffffffffu, y.y, o);
    if (lane >= o) { y.x += a; y.y += b; }
  }
  *total = make_uint2(__shfl_sync(0xffffffffu, y.x, 31), __shfl_sync(0xffffffffu, y.y, 31));
  const uint32_t bx = __shfl_sync(0xffffffffu, y.x - w.x, warp), by = __shfl_sync(0xffffffffu, y.y - w.y, warp);
  return make_uint2(bx + x.x - v.x, by + x.y - v.y);
}

template <bool IN_REGS>
__global__ void __launch_bounds__(SEL_T, 1) dg_kv8_select_kernel(const __grid_constant__ EvictParams p, uint32_t ctas) {
  __shared__ uint32_t hist[BINS];            // this CTA's counts of a digit
  __shared__ uint32_t sums[BINS];            // the cluster's
  __shared__ uint2 warp_sum[32];
  __shared__ uint32_t found[2];
  __shared__ uint32_t totals[2];             // kept and tied tokens of this CTA
  grid_launch_dependents();
  grid_wait();
  const uint32_t tid = threadIdx.x, rank = blockIdx.x % ctas, h = blockIdx.x / ctas;
  const float* w = p.w + size_t(h) * p.ld;
  const uint32_t n = p.n_keys - p.n_recent, take = p.n_keep - p.n_recent;
  const uint32_t seg = (n + ctas - 1) / ctas, per = (seg + SEL_T - 1) / SEL_T;
  // this thread's run of tokens
  const uint32_t end_c = (rank + 1) * seg < n ? (rank + 1) * seg : n;
  uint32_t t0 = rank * seg + tid * per, t1 = t0 + per;
  if (t0 > end_c) t0 = end_c;
  if (t1 > end_c) t1 = end_c;
  float run[IN_REGS ? RUN : 1];
  if (IN_REGS) {
#pragma unroll
    for (uint32_t i = 0; i < RUN; ++i) run[i] = t0 + i < t1 ? __ldg(w + t0 + i) : 0.f;
  }
  // f(token, weight) for the tokens of the run, in order
  auto each = [&](auto f) {
    if (IN_REGS) {
#pragma unroll
      for (uint32_t i = 0; i < RUN; ++i)
        if (t0 + i < t1) f(t0 + i, run[i]);
    } else {
      for (uint32_t t = t0; t < t1; ++t) f(t, __ldg(w + t));
    }
  };
  auto sync_all = [&] {
    if (ctas > 1) cluster_sync_all(); else __syncthreads();
  };

  uint32_t prefix = 0, left = take;          // the digits found so far; tokens to take among those that share them
  if (take > 0) {
#pragma unroll 1
    for (uint32_t pass = 0; pass < 3; ++pass) {
      const uint32_t shift = pass == 0 ? 21u : pass == 1 ? 10u : 0u, bits = pass == 2 ? 10u : 11u, bins = 1u << bits;
      hist[tid] = 0u;
      hist[tid + SEL_T] = 0u;
      __syncthreads();
      each([&](uint32_t, float x) {
        const uint32_t key = weight_key(x);
        if (pass == 0 || (key >> (shift + bits)) == prefix) atomicAdd(hist + ((key >> shift) & (bins - 1u)), 1u);
      });
      sync_all();
      if (ctas > 1) {
        for (uint32_t i = tid; i < bins / ctas; i += SEL_T) {
          const uint32_t bin = rank * (bins / ctas) + i;
          uint32_t s = 0;
          for (uint32_t r = 0; r < ctas; ++r) s += ld_dsmem(dsmem_addr(smem_u32(hist + bin), r));
          for (uint32_t r = 0; r < ctas; ++r) st_dsmem(dsmem_addr(smem_u32(sums + bin), r), s);
        }
        cluster_sync_all();
      }
      // largest digit first: thread i has the bins bins - 1 - 2i and bins - 2 - 2i
      const uint32_t* src = ctas > 1 ? sums : hist;
      const uint32_t c0 = 2u * tid < bins ? src[bins - 1u - 2u * tid] : 0u, c1 = 2u * tid < bins ? src[bins - 2u - 2u * tid] : 0u;
      uint2 total;
      const uint32_t before = block_scan2(make_uint2(c0 + c1, 0u), warp_sum, &total).x;
      if (before < left && left <= before + c0 + c1) {
        const bool in_first = left <= before + c0;
        found[0] = bins - 1u - 2u * tid - (in_first ? 0u : 1u);
        found[1] = left - before - (in_first ? 0u : c0);
      }
      __syncthreads();
      prefix = (prefix << bits) | found[0];
      left = found[1];
    }
  }
  // kept: above the cut, and the first `left` of those at it
  uint32_t gt = 0, eq = 0;
  if (take > 0)
    each([&](uint32_t, float x) {
      const uint32_t key = weight_key(x);
      gt += key > prefix ? 1u : 0u;
      eq += key == prefix ? 1u : 0u;
    });
  uint2 total;
  uint2 at = block_scan2(make_uint2(gt, eq), warp_sum, &total);
  if (ctas > 1) {
    if (tid == 0) {
      totals[0] = total.x;
      totals[1] = total.y;
    }
    cluster_sync_all();
    for (uint32_t r = 0; r < rank; ++r) {
      at.x += ld_dsmem(dsmem_addr(smem_u32(&totals[0]), r));
      at.y += ld_dsmem(dsmem_addr(smem_u32(&totals[1]), r));
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  }
  int32_t* kept = p.kept + size_t(h) * p.n_keep;
  float* w_out = p.w_out ? p.w_out + size_t(h) * p.ld_out : nullptr;
  if (take > 0)
    each([&](uint32_t t, float x) {
      const uint32_t key = weight_key(x);
      const bool tie = key == prefix;
      if (key > prefix || (tie && at.y < left)) {
        const uint32_t o = at.x + (at.y < left ? at.y : left);
        kept[o] = int32_t(t);
        if (w_out) w_out[o] = x;
      }
      at.x += key > prefix ? 1u : 0u;
      at.y += tie ? 1u : 0u;
    });
  for (uint32_t i = rank * SEL_T + tid; i < p.n_recent; i += ctas * SEL_T) {
    kept[take + i] = int32_t(n + i);
    if (w_out) w_out[take + i] = w[n + i];
  }
  if (ctas > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // no CTA leaves while its counts may be read
}

template <uint32_t D>
__global__ void __launch_bounds__(512) dg_kv8_move_kernel(const __grid_constant__ EvictParams p) {
  constexpr uint32_t CH = D / 16, PER = BLK * CH / 512;     // 16-byte chunks of a row, of a thread
  __shared__ float red[16];
  __shared__ int32_t exps[BLK];
  grid_launch_dependents();
  grid_wait();
  const bool is_k = blockIdx.z == 0;
  const uint32_t h = blockIdx.y, blk = blockIdx.x, tid = threadIdx.x;
  const uint32_t rows = p.n_keep - blk * BLK < BLK ? p.n_keep - blk * BLK : BLK;
  const int32_t* kept = p.kept + size_t(h) * p.n_keep + blk * BLK;
  const uint8_t* src = (is_k ? p.k : p.v) + size_t(h) * p.blocks * BLK * D;
  const int32_t* from = p.exps + size_t(h) * p.blocks * 2 + (is_k ? 0 : 1);
  uint4 v[PER];
  float top = 0.f;
#pragma unroll
  for (uint32_t i = 0; i < PER; ++i) {
    const uint32_t x = i * 512u + tid, r = x / CH, c = x % CH;
    v[i] = make_uint4(0u, 0u, 0u, 0u);
    if (r < rows) {
      const uint32_t slot = uint32_t(kept[r]);
      v[i] = *reinterpret_cast<const uint4*>(src + size_t(slot / BLK) * BLK * D + (c >> 3) * SLAB + chunk_off(slot % BLK, c & 7u));
      const int e = from[slot / BLK * 2];
      if (c == 0) exps[r] = e;
      uint32_t m = __vmaxu4(__vmaxu4(v[i].x & 0x7f7f7f7fu, v[i].y & 0x7f7f7f7fu), __vmaxu4(v[i].z & 0x7f7f7f7fu, v[i].w & 0x7f7f7f7fu));
      m = __vmaxu4(m, m >> 16);
      m = __vmaxu4(m, m >> 8) & 0xffu;
      top = fmaxf(top, f32x2_from_e4m3x2(uint16_t(m)).x * pow2i(e));
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((tid & 31u) == 0) red[tid >> 5] = top;
  __syncthreads();
  top = red[tid & 15u];
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const int e = scale_exp(top);
  uint8_t* dst = (is_k ? p.to_k : p.to_v) + (size_t(h) * p.to_blocks + blk) * BLK * D;
#pragma unroll
  for (uint32_t i = 0; i < PER; ++i) {
    const uint32_t x = i * 512u + tid, r = x / CH, c = x % CH;
    if (r >= rows) continue;
    const int de = exps[r] - e;
    if (de != 0) {
      const float mul = pow2i(de);
      uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 a = f32x2_from_e4m3x2(uint16_t(u[j])), b = f32x2_from_e4m3x2(uint16_t(u[j] >> 16));
        u[j] = uint32_t(e4m3x2(a.x * mul, a.y * mul)) | (uint32_t(e4m3x2(b.x * mul, b.y * mul)) << 16);
      }
      v[i] = make_uint4(u[0], u[1], u[2], u[3]);
    }
    *reinterpret_cast<uint4*>(dst + (c >> 3) * SLAB + chunk_off(r, c & 7u)) = v[i];
  }
  if (tid == 0) p.to_exps[(size_t(h) * p.to_blocks + blk) * 2 + (is_k ? 0 : 1)] = e;
}

cudaError_t launch_evict(const EvictParams& p, cudaStream_t st) {
  // CTAs of a head: one up to 4,096 tokens (four each thread), eight from 16,385
  uint32_t ctas = 1;
  while (ctas < 8 && (p.n_keys - p.n_recent) > ctas * 4u * SEL_T) ctas *= 2;
  const bool in_regs = p.n_keys - p.n_recent <= ctas * SEL_T * RUN;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas * p.Hkv);
  cfg.blockDim = dim3(SEL_T);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = in_regs ? cudaLaunchKernelEx(&cfg, dg_kv8_select_kernel<true>, p, ctas) : cudaLaunchKernelEx(&cfg, dg_kv8_select_kernel<false>, p, ctas);
  if (e != cudaSuccess) return e;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3((p.n_keep + BLK - 1) / BLK, p.Hkv, 2);
  cfg.blockDim = dim3(512);
  return p.D == 256 ? cudaLaunchKernelEx(&cfg, dg_kv8_move_kernel<256>, p) : cudaLaunchKernelEx(&cfg, dg_kv8_move_kernel<512>, p);
}

}  // namespace kv8
}  // namespace dg
