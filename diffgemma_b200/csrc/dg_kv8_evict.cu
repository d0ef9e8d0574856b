// Eviction: the n_recent last tokens of a cache and, of those before them, the n_keep - n_recent with the largest weights
// (equal ones: lowest index), in order, into another cache.
//
// Selection, a cluster of up to sixteen CTAs for each head: the cut is found exactly by a radix over 32-bit order keys, eight
// bits a pass.  A lane holds every 32nd token of its warp's stretch in registers, up to 16 of them (262,144 tokens a head; longer
// rows are read again for each pass), so that loads are whole lines and a token's place comes from ballots.  In a pass a CTA
// counts its tokens by digit, every CTA reads the counts of all (distributed shared memory, one barrier a pass) and finds the
// digit for itself; the counts of the CTAs ahead that lie above the cut add up to its first place in the output, so that no
// exchange follows the last pass.  What bounds it is those barriers and the CTAs that hold the row: 131,072 tokens of 2 heads
// take 16.7 us (24.1 with 8 CTAs, runs of tokens by thread and digits of 11 bits; counts of a digit aggregated by match or in
// copies by lane were slower than plain shared-memory adds, which the unit merges: 2,000 cycles a pass against 5,000 and 9,000).
// Moving, a CTA for each block of the new cache: 128 gathered rows of codes, whose values get the scale of their new block; the
// codes stay as they are where the scale does.
#include "dg_kv8.cuh"

namespace dg {
namespace kv8 {

constexpr uint32_t SEL_T = 1024, BINS = 256, RUN = 16, MAX_CTAS = 16;

// larger key = larger weight; NaN below everything
__device__ __forceinline__ uint32_t weight_key(float w) { return w != w ? 0u : score_order_key(w); }

__device__ __forceinline__ uint32_t ld_dsmem(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
// sum over the lanes before this one, and over all
__device__ __forceinline__ uint32_t warp_scan(uint32_t v, uint32_t* total) {
  const uint32_t lane = threadIdx.x & 31u;
  uint32_t x = v;
#pragma unroll
  for (uint32_t o = 1; o < 32; o <<= 1) {
    const uint32_t a = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += a;
  }
  *total = __shfl_sync(0xffffffffu, x, 31);
  return x - v;
}

template <bool IN_REGS>
__global__ void __launch_bounds__(SEL_T, 1) dg_kv8_select_kernel(const __grid_constant__ EvictParams p, uint32_t ctas) {
  __shared__ uint32_t hist[4][BINS];         // this CTA's counts of a digit
  __shared__ __align__(16) uint32_t part[4][BINS];         // the cluster's, by pairs of CTAs
  __shared__ uint32_t warp_gt[32], warp_eq[32];
  __shared__ uint32_t found[2];
  __shared__ uint32_t ahead_gt, ahead_eq;    // tokens above the cut and at it in the CTAs ahead
  grid_launch_dependents();
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, rank = blockIdx.x % ctas, h = blockIdx.x / ctas;
  hist[tid / BINS][tid % BINS] = 0u;
  if (tid == 0) ahead_gt = ahead_eq = 0u;
  grid_wait();
  const float* w = p.w + size_t(h) * p.ld;
  const uint32_t n = p.n_keys - p.n_recent, take = p.n_keep - p.n_recent;
  // a CTA has `per` times 1,024 tokens, a warp `per` times 32 of them, a lane every 32nd
  const uint32_t per = ((n + ctas - 1) / ctas + SEL_T - 1) / SEL_T;
  const uint32_t t0 = (rank * SEL_T + warp * 32u) * per + lane;
  float run[IN_REGS ? RUN : 1];
  if (IN_REGS) {
#pragma unroll
    for (uint32_t i = 0; i < RUN; ++i) run[i] = i < per && t0 + i * 32u < n ? __ldg(w + t0 + i * 32u) : 0.f;
  }
  // f(token, weight, is there one) for the warp's tokens, in order, by all lanes at once
  auto each = [&](auto f) {
    if (IN_REGS) {
#pragma unroll
      for (uint32_t i = 0; i < RUN; ++i)
        if (i < per) f(t0 + i * 32u, run[i], t0 + i * 32u < n);
    } else {
#pragma unroll 1
      for (uint32_t i = 0; i < per; ++i) {
        const uint32_t t = t0 + i * 32u;
        f(t, t < n ? __ldg(w + t) : 0.f, t < n);
      }
    }
  };
  __syncthreads();

  uint32_t cut = 0, left = take;             // the digits found so far; tokens to take among those that share them
  if (take > 0) {
#pragma unroll 1
    for (uint32_t pass = 0; pass < 4; ++pass) {
      const uint32_t shift = 24u - 8u * pass, high = pass == 0 ? 0u : 0xffffffffu << (shift + 8u);
      each([&](uint32_t, float x, bool is) {
        const uint32_t key = weight_key(x);
        if (is && ((key ^ cut) & high) == 0u) atomicAdd(&hist[pass][(key >> shift) & (BINS - 1u)], 1u);
      });
      if (ctas > 1) cluster_sync_all(); else __syncthreads();
      const uint32_t bin = tid % BINS, r = tid / BINS;
      uint32_t s = 0, ahead = 0;
#pragma unroll
      for (uint32_t i = 0; i < MAX_CTAS; i += 4)
        if (r + i < ctas) {
          const uint32_t c = ld_dsmem(dsmem_addr(smem_u32(&hist[pass][bin]), r + i));
          s += c;
          ahead += r + i < rank ? c : 0u;
        }
      part[r][bin] = s;
      __syncthreads();
      if (warp == 0) {
        // largest digit first: lane i has the bins 255 - 8i down to 248 - 8i
        uint32_t c[8] = {}, all = 0, total;
#pragma unroll
        for (uint32_t r2 = 0; r2 < 4; ++r2)
#pragma unroll
          for (uint32_t q = 0; q < 2; ++q) {
            const uint4 v = *reinterpret_cast<const uint4*>(&part[r2][BINS - 8u - 8u * lane + 4u * q]);
            c[4 * q] += v.x; c[4 * q + 1] += v.y; c[4 * q + 2] += v.z; c[4 * q + 3] += v.w;
          }
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) all += c[i];
        uint32_t before = warp_scan(all, &total);
        if (before < left && left <= before + all) {
#pragma unroll
          for (uint32_t i = 8; i-- > 0;) {
            if (before < left && left <= before + c[i]) {
              found[0] = BINS - 8u - 8u * lane + i;
              found[1] = left - before;
            }
            before += c[i];
          }
        }
      }
      __syncthreads();
      cut |= found[0] << shift;
      left = found[1];
      if (ctas > 1) {
        const uint32_t above = __reduce_add_sync(0xffffffffu, bin > found[0] ? ahead : 0u);
        if (lane == 0 && above != 0u) atomicAdd(&ahead_gt, above);
        if (pass == 3 && bin == found[0] && ahead != 0u) atomicAdd(&ahead_eq, ahead);
      }
    }
  }
  if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  // kept: above the cut, and the first `left` of those at it
  uint32_t gt = 0, eq = 0;
  if (take > 0)
    each([&](uint32_t, float x, bool is) {
        const uint32_t key = weight_key(x);
      gt += __popc(__ballot_sync(0xffffffffu, is && key > cut));
      eq += __popc(__ballot_sync(0xffffffffu, is && key == cut));
    });
  if (lane == 0) {
    warp_gt[warp] = gt;
    warp_eq[warp] = eq;
  }
  __syncthreads();
  uint32_t total;
  const uint32_t base_gt = warp_scan(warp_gt[lane], &total), base_eq = warp_scan(warp_eq[lane], &total);
  uint32_t at_gt = ahead_gt + __shfl_sync(0xffffffffu, base_gt, warp), at_eq = ahead_eq + __shfl_sync(0xffffffffu, base_eq, warp);
  int32_t* kept = p.kept + size_t(h) * p.n_keep;
  float* w_out = p.w_out ? p.w_out + size_t(h) * p.ld_out : nullptr;
  if (take > 0)
    each([&](uint32_t t, float x, bool is) {
      const uint32_t key = weight_key(x);
      const uint32_t g = __ballot_sync(0xffffffffu, is && key > cut), q = __ballot_sync(0xffffffffu, is && key == cut);
      if ((g | q) == 0u) return;
      const uint32_t ahead = (1u << lane) - 1u;
      const uint32_t ties = at_eq + __popc(q & ahead);      // those at the cut ahead of this token
      if (is && key >= cut && (key > cut || ties < left)) {
        const uint32_t o = at_gt + __popc(g & ahead) + (ties < left ? ties : left);
        kept[o] = int32_t(t);
        if (w_out) w_out[o] = x;
      }
      at_gt += __popc(g);
      at_eq += __popc(q);
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

cudaError_t configure_evict() {
  cudaError_t e = cudaFuncSetAttribute(dg_kv8_select_kernel<true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(dg_kv8_select_kernel<false>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  return e;
}

cudaError_t launch_evict(const EvictParams& p, cudaStream_t st) {
  // CTAs of a head: one up to 4,096 tokens (four each thread), sixteen from 32,769
  uint32_t ctas = 1;
  while (ctas < MAX_CTAS && (p.n_keys - p.n_recent) > ctas * 4u * SEL_T) ctas *= 2;
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
