// Everything that enters or leaves 8 bits: the rows of a step (queries in two terms, canvas K and V in two terms), tokens
// appended to a cache, rows read back.
//
#include "dg_kv8_rows.cuh"

namespace dg {
namespace kv8 {

constexpr uint32_t CT = 512;                  // threads: 16 warps
constexpr uint32_t PASS = 16;                 // tokens whose angles are in shared memory at a time, one for each warp

struct PosList {
  uint64_t pos[MAX_SEQ];
};

// ------------------------------------------------------------------------------------------- rows of a step
// A warp takes one row.  Canvas K and V: the rows of one (head, tile, K or V) share a scale; they lie in `slots` neighbouring
// warps (up to 16 canvas tokens) or in the CTAs of a cluster, 16 tokens each, whose maxima meet over distributed shared memory.
// Queries: a CTA for each canvas token, all heads (the angles are computed once for all of them).
// A step's rows of 256 tokens: 14 us (8 KV heads of 256 dims), 13.5 (2 of 512), most of it one chain - launch, loads, angles,
// norm, rotation, the cluster's maxima, stores; two or three tokens a CTA, which make one wave of two, take as long.
struct RowsPlan {
  uint32_t slots, cluster;             // warps of a scale group in a CTA; CTAs of one (16 slots)
  uint32_t canvas_ctas, per_seq;       // CTAs of canvas rows; of them, of a sequence
  uint32_t heads;                      // KV heads that a CTA of 16 slots takes one after the other
  uint32_t q_tokens, q_ctas;           // query CTAs of a sequence, of all
};
// heads that a CTA of 16 slots holds in registers
__host__ __device__ constexpr uint32_t row_heads(int nj) { return nj == 1 ? 4u : 2u; }

// One row of canvas K or V: normed, rotated, rounded, what is not finite as zero.  Returns its largest magnitude.
template <int NJ>
__device__ __forceinline__ float canvas_row(const CodeParams& p, bool is_k, const uint4 (&raw)[NJ], const double2* tab, uint32_t lane, uint4 (&v)[NJ],
                                            bool* bad) {
  if (is_k || p.v_norm)
    row_to_bf16<double, NJ>(raw, is_k ? p.kw : nullptr, true, p.eps, p.rope, is_k && p.rope.half != 0u ? tab : nullptr, lane, v);
  else {
#pragma unroll
    for (int j = 0; j < NJ; ++j) v[j] = raw[j];
  }
  uint32_t top2 = 0;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    v[j] = make_uint4(finite_or_zero(v[j].x, bad), finite_or_zero(v[j].y, bad), finite_or_zero(v[j].z, bad), finite_or_zero(v[j].w, bad));
    top2 = abs_max2(abs_max2(abs_max2(abs_max2(top2, v[j].x), v[j].y), v[j].z), v[j].w);
  }
  float top = max_of_halves(top2);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  return top;
}
// Stores row r of a canvas tile of `valid` tokens as two terms, and zeros behind V's last row up to a whole step of 32 keys
// (their weights are zero, and zero times NaN is not); rows r, r + stride, ...
template <int NJ>
__device__ __forceinline__ void store_canvas_row(const CodeParams& p, bool is_k, size_t tile, uint32_t r, uint32_t stride, uint32_t valid, float top,
                                                 uint32_t lane, const uint4 (&v)[NJ]) {
  constexpr uint32_t D = 256u * NJ;
  const int e = scale_exp(top);
  const float mul = pow2i(-e);
  uint8_t* dst = (is_k ? p.k_codes : p.v_codes) + tile * 2u * BLK * D;
  const uint32_t end = is_k ? valid : (valid + 31u) / 32u * 32u;
  for (uint32_t x = r; x < end; x += stride) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const uint32_t off = code8_off(x, lane + 32u * j);
      uint2 c = make_uint2(0u, 0u), rest = c;
      if (x < valid) c = code8(v[j], mul, &rest);
      *reinterpret_cast<uint2*>(dst + off) = c;
      *reinterpret_cast<uint2*>(dst + BLK * D + off) = rest;
    }
  }
  if (lane == 0 && r == 0) p.exps[tile * 2 + (is_k ? 0 : 1)] = e;
}

template <int NJ>
__global__ void __launch_bounds__(CT, NJ == 1 ? 2 : 1) dg_kv8_rows_kernel(const __grid_constant__ QueryParams q, const __grid_constant__ CodeParams p,
                                                                         const __grid_constant__ PosList pos, const __grid_constant__ RowsPlan plan) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr uint32_t ROW_HEADS = row_heads(NJ);
  __shared__ float red[ROW_HEADS][16];
  grid_launch_dependents();
  grid_wait();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  constexpr uint32_t D = 256u * NJ;
  double2* tab = reinterpret_cast<double2*>(smem);
  if (blockIdx.x < plan.canvas_ctas && plan.slots < 16u) {
    // few tokens: the warps are (head, K or V, token)
    const uint32_t b = blockIdx.x / plan.per_seq, g = blockIdx.x % plan.per_seq * (16u / plan.slots) + warp / plan.slots;
    const uint32_t t = warp % plan.slots, h = g >> 1;
    const bool on = h < p.Hkv, is_k = (g & 1u) == 0u, live = on && t < p.n;
    const __nv_bfloat16* src = (is_k ? p.k : p.v) + ((size_t(b) * p.n + t) * p.Hkv + h) * D + 8u * lane;
    uint4 raw[NJ], v[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) raw[j] = live ? *reinterpret_cast<const uint4*>(src + 256u * j) : make_uint4(0u, 0u, 0u, 0u);
    if (p.rope.half != 0u) angles<double, CT>(p.rope, double(pos.pos[b]), p.n, tab);
    __syncthreads();
    bool bad = false;
    const float mine = live ? canvas_row<NJ>(p, is_k, raw, tab + t * p.rope.half, lane, v, &bad) : 0.f;
    if (lane == 0) red[0][warp] = mine;
    __syncthreads();
    float top = 0.f;
    for (uint32_t i = 0; i < plan.slots; ++i) top = fmaxf(top, red[0][warp / plan.slots * plan.slots + i]);
    if (on) store_canvas_row<NJ>(p, is_k, size_t(b) * p.Hkv + h, t, plan.slots, p.n, top, lane, v);
    if (bad) dev_status_set(p.status, DG_DEV_NOT_FINITE, KID_CODE, blockIdx.x, t);
    return;
  }
  if (blockIdx.x < plan.canvas_ctas) {
    // a cluster: (sequence, run of heads, tile, K or V); a CTA 16 tokens, a warp one of them in every head of the run
    const uint32_t rank = blockIdx.x % plan.cluster;
    uint32_t x = blockIdx.x / plan.cluster;
    const uint32_t b = x / plan.per_seq;
    x %= plan.per_seq;
    const bool is_k = (x & 1u) == 0u;
    const uint32_t ct = (x >> 1) % p.n_ctiles, h0 = (x >> 1) / p.n_ctiles * plan.heads;
    const uint32_t r = rank * 16u + warp, t = ct * BLK + r;
    const bool live = t < p.n;
    const __nv_bfloat16* src = (is_k ? p.k : p.v) + ((size_t(b) * p.n + t) * p.Hkv + h0) * D + 8u * lane;
    uint4 v[ROW_HEADS][NJ];
#pragma unroll
    for (uint32_t i = 0; i < ROW_HEADS; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        v[i][j] = live && i < plan.heads && h0 + i < p.Hkv ? *reinterpret_cast<const uint4*>(src + size_t(i) * D + 256u * j) : make_uint4(0u, 0u, 0u, 0u);
    if (is_k && p.rope.half != 0u) {
      const uint32_t first = ct * BLK + rank * 16u;
      if (first < p.n) angles<double, CT>(p.rope, double(pos.pos[b]) + double(first), p.n - first < 16u ? p.n - first : 16u, tab);
      __syncthreads();
    }
    bool bad = false;
#pragma unroll
    for (uint32_t i = 0; i < ROW_HEADS; ++i) {
      if (i >= plan.heads) continue;
      float mine = 0.f;
      if (live) {
        uint4 y[NJ];
        mine = canvas_row<NJ>(p, is_k, v[i], tab + warp * p.rope.half, lane, y, &bad);
#pragma unroll
        for (int j = 0; j < NJ; ++j) v[i][j] = y[j];
      }
      if (lane == 0) red[i][warp] = mine;
    }
    float top[ROW_HEADS] = {};
    if (plan.cluster > 1u) {
      cluster_sync_all();
#pragma unroll
      for (uint32_t i = 0; i < ROW_HEADS; ++i) {
        if (i >= plan.heads) continue;
        const uint32_t at = smem_u32(&red[i][lane & 15u]);
        for (uint32_t c = lane >> 4; c < plan.cluster; c += 2u) {
          float y;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(y) : "r"(dsmem_addr(at, c)) : "memory");
          top[i] = fmaxf(top[i], y);
        }
      }
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    } else {
      __syncthreads();
#pragma unroll
      for (uint32_t i = 0; i < ROW_HEADS; ++i) top[i] = red[i][lane & 15u];
    }
    const uint32_t valid = p.n - ct * BLK < BLK ? p.n - ct * BLK : BLK;
#pragma unroll
    for (uint32_t i = 0; i < ROW_HEADS; ++i) {
      if (i >= plan.heads || h0 + i >= p.Hkv) continue;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
      store_canvas_row<NJ>(p, is_k, (size_t(b) * p.Hkv + h0 + i) * p.n_ctiles + ct, r, 16u * plan.cluster, valid, top[i], lane, v[i]);
    }
    if (bad) dev_status_set(p.status, DG_DEV_NOT_FINITE, KID_CODE, blockIdx.x, t);
    if (plan.cluster > 1u) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // nobody leaves while its maxima may be read
    return;
  }
  if (blockIdx.x >= plan.canvas_ctas + plan.q_ctas) return;      // the grid is a whole number of clusters
  const uint32_t x = blockIdx.x - plan.canvas_ctas;
  const uint32_t b = x / plan.q_tokens, i = x % plan.q_tokens;
  const QueryRows& o = q.rows;
  const bool live = i < o.C;
  if (live && q.rope.half != 0u) {
    angles<double, CT>(q.rope, double(pos.pos[b]) + double(i), 1u, tab);
    __syncthreads();
  }
  for (uint32_t h = warp; h < o.Hq; h += CT / 32u) {
    const uint32_t kvh = h / o.G, R = i * o.G + h % o.G;
    if (R >= o.MT * BLK) continue;
    uint4 v[NJ];
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
    // key weights: the row's -log2 e * lse, -inf for a row that draws nothing
    float nl = -INFINITY;
    if (live && q.lse != nullptr) nl = -1.4426950408889634f * q.lse[(size_t(b) * o.C + i) * o.Hq + h];
    uint32_t top2 = 0;
#pragma unroll
    for (int j = 0; j < NJ; ++j) top2 = abs_max2(abs_max2(abs_max2(abs_max2(top2, v[j].x), v[j].y), v[j].z), v[j].w);
    uint32_t top = (top2 >> 16) > (top2 & 0xffffu) ? top2 >> 16 : top2 & 0xffffu;
    top = __reduce_max_sync(0xffffffffu, top);
    // a row that is not finite has no scores: its codes are NaN
    bool fin = top < 0x7f80u;
    if (q.lse != nullptr) {
      // no share of any key has a row without a sum (none, -lse = inf; or behind the last token), and one that is not finite or
      // whose sum is not, which is reported: its NaN would be every key's, and a running mean's from then on
      if (live && (!fin || !(nl < INFINITY && nl > -INFINITY))) {
        if (lane == 0 && (!fin || nl != INFINITY)) dev_status_set(q.status, DG_DEV_NOT_FINITE, KID_CODE, blockIdx.x, i);
        nl = -INFINITY;
      }
      if (nl == -INFINITY) {
        top = 0u;
        fin = true;
#pragma unroll
        for (int j = 0; j < NJ; ++j) v[j] = make_uint4(0u, 0u, 0u, 0u);
      }
    }
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
      const size_t at = (size_t(b) * o.Hkv + kvh) * o.MT * BLK + R;
      if (q.lse != nullptr) {   // two rows' factors, then their -lse: as pairs
        float* pair = reinterpret_cast<float*>(o.row) + (at & ~size_t(1)) * 2u + (at & 1u);
        pair[0] = q.scale_log2 * pow2i(e);
        pair[2] = nl;
      } else {
        o.row[at] = make_float2(q.scale_log2 * pow2i(e), nl);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------- append
// One CTA (head_dim 512: a cluster of two, 64 tokens each) for each (block, head, K or V) that the new tokens touch; the rows
// are in registers from load to store, 16-byte chunks of 8 / NJ rows a warp, two CTAs an SM: one loads while the other works.
// The first block may hold tokens already: their values are read, and the block is coded as a whole at the scale that all
// of it needs.  The angles of 32 tokens at a time: a thread's pair turns from pass to pass in 64 bits, within one in 32.
constexpr uint32_t APASS = 32;

template <int NJ>
__global__ void __launch_bounds__(CT, 2) dg_kv8_append_kernel(const __grid_constant__ CodeParams p) {
  constexpr uint32_t D = 256u * NJ, RW = 8u / NJ, TOK = 16u * RW;     // rows of a warp, tokens of a CTA
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float red[16];
  __shared__ __align__(16) float weight[D];
  float2* tab = reinterpret_cast<float2*>(smem);
  grid_launch_dependents();
  grid_wait();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  uint32_t x = blockIdx.x / NJ;
  const uint32_t rank = blockIdx.x % NJ;
  const bool is_k = (x & 1u) == 0u;
  x >>= 1;
  const uint32_t h = x % p.Hkv, blk = p.n_keys / BLK + x / p.Hkv;
  const uint32_t t0 = blk * BLK, end = p.n_keys + p.n;
  const uint32_t kept = p.n_keys > t0 ? p.n_keys - t0 : 0u;
  const uint32_t n_rows = end - t0 < BLK ? end - t0 : BLK;
  uint8_t* codes = (is_k ? p.k_codes : p.v_codes) + (size_t(h) * p.blocks + blk) * BLK * D;
  int32_t* exps = p.exps + (size_t(h) * p.blocks + blk) * 2 + (is_k ? 0 : 1);
  const __nv_bfloat16* src = is_k ? p.k : p.v;
  // row s of this warp
  auto row = [&](uint32_t s) { return rank * TOK + (s >> 1) * APASS + warp * 2u + (s & 1u); };
  uint4 held[RW][NJ];
#pragma unroll
  for (uint32_t s = 0; s < RW; ++s) {
    const uint32_t r = row(s);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      held[s][j] = make_uint4(0u, 0u, 0u, 0u);
      if (r < n_rows && r >= kept)
        held[s][j] = __ldcs(reinterpret_cast<const uint4*>(src + (size_t(t0 + r - p.n_keys) * p.Hkv + h) * D + 8u * (lane + 32u * j)));
    }
  }
  if (kept != 0u) {
    const float old = pow2i(*exps);
#pragma unroll
    for (uint32_t s = 0; s < RW; ++s) {
      const uint32_t r = row(s);
      if (r >= kept) continue;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const uint2 c = *reinterpret_cast<const uint2*>(codes + code8_off(r, lane + 32u * j));
        const float2 a = f32x2_from_e4m3x2(uint16_t(c.x)), b = f32x2_from_e4m3x2(uint16_t(c.x >> 16));
        const float2 f = f32x2_from_e4m3x2(uint16_t(c.y)), g = f32x2_from_e4m3x2(uint16_t(c.y >> 16));
        held[s][j] = make_uint4(pack_bf16x2(a.x * old, a.y * old), pack_bf16x2(b.x * old, b.y * old),
                                pack_bf16x2(f.x * old, f.y * old), pack_bf16x2(g.x * old, g.y * old));
      }
    }
  }
  const bool turn = is_k && !p.ready && p.rope.half != 0u, norm = !p.ready && (is_k || p.v_norm), weighed = norm && is_k && p.kw != nullptr;
  if (weighed) {
    if (threadIdx.x < D) weight[threadIdx.x] = __bfloat162float(p.kw[threadIdx.x]);
    if (!turn) __syncthreads();
  }
  // a thread's pair and its run of the pass's tokens
  const uint32_t groups = turn ? CT / p.rope.half : 1u, per = (APASS + groups - 1u) / groups;
  const uint32_t dim = turn ? threadIdx.x % p.rope.half : 0u, tok = turn ? threadIdx.x / p.rope.half * per : APASS;
  double2 z = {}, hop = {};
  float2 one = {};
  if (turn && threadIdx.x < groups * p.rope.half && tok < APASS) {
    const double turns = turns_of(p.rope, dim);
    z = unit_at(double(p.pos) + double(t0 + rank * TOK + tok) - double(p.n_keys), turns);
    hop = unit_at(double(APASS), turns);
    const double2 o = unit_at(1.0, turns);
    one = make_float2(float(o.x), float(o.y));
  }
  bool bad = false;
  uint32_t top = 0;
#pragma unroll
  for (uint32_t s = 0; s < RW; ++s) {
    const uint32_t r = row(s);
    if (turn && (s & 1u) == 0u) {
      if (s != 0u) __syncthreads();
      if (threadIdx.x < groups * p.rope.half) {
        float2 c = make_float2(float(z.x), float(z.y));
        for (uint32_t i = tok; i < tok + per && i < APASS; ++i) {
          tab[i * p.rope.half + (dim & 7u) * (p.rope.half >> 3) + (dim >> 3)] = c;
          c = make_float2(fmaf(c.x, one.x, -c.y * one.y), fmaf(c.x, one.y, c.y * one.x));
        }
        z = cmul(z, hop);
      }
      __syncthreads();
    }
    if (r < n_rows && r >= kept) {
      const float2* cs = turn ? tab + (r % APASS) * p.rope.half : nullptr;
      if (NJ == 2 && turn && p.rope.dist != 256u) {
        uint4 y[NJ];
        row_to_bf16<float, NJ>(held[s], p.kw, true, p.eps, p.rope, cs, lane, y);
#pragma unroll
        for (int j = 0; j < NJ; ++j) held[s][j] = y[j];
      } else if (turn || norm) {
        row_to_bf16_f32<NJ>(held[s], weighed ? weight : nullptr, norm, p.eps, p.rope, cs, lane);
      }
    }
    uint32_t big = 0;
#pragma unroll
    for (int j = 0; j < NJ; ++j) big = abs_max2(abs_max2(abs_max2(abs_max2(big, held[s][j].x), held[s][j].y), held[s][j].z), held[s][j].w);
    if ((big & 0x7f80u) == 0x7f80u || big >= 0x7f800000u) {    // something is not finite
      big = 0;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        uint4& y = held[s][j];
        y = make_uint4(finite_or_zero(y.x, &bad), finite_or_zero(y.y, &bad), finite_or_zero(y.z, &bad), finite_or_zero(y.w, &bad));
        big = abs_max2(abs_max2(abs_max2(abs_max2(big, y.x), y.y), y.z), y.w);
      }
    }
    top = abs_max2(top, big);
  }
  float t = max_of_halves(top);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
  if (lane == 0) red[warp] = t;
  if (NJ == 1) {
    __syncthreads();
    t = red[lane & 15u];
  } else {
    cluster_sync_all();
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(t) : "r"(dsmem_addr(smem_u32(&red[lane & 15u]), lane >> 4)) : "memory");
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
  const int e = scale_exp(t);
  const uint32_t mul = (__float_as_uint(pow2i(-e)) >> 16) * 0x10001u;
#pragma unroll
  for (uint32_t s = 0; s < RW; ++s) {
    const uint32_t r = row(s);
    if (r >= n_rows) continue;
#pragma unroll
    for (int j = 0; j < NJ; ++j) *reinterpret_cast<uint2*>(codes + code8_off(r, lane + 32u * j)) = code8_fast(held[s][j], mul);
  }
  if (bad) dev_status_set(p.status, DG_DEV_NOT_FINITE, KID_CODE, blockIdx.x, t0);
  if (NJ > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // nobody leaves while its maximum may be read
  if (threadIdx.x == 0 && rank == 0) *exps = e;                                     // (the other CTA has read the old scale)
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
    const float mul = pow2i(p.exps[blk * 2 + (is_k ? 0 : 1)]);
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

constexpr size_t ROWS_SMEM = PASS * 256u * sizeof(double2);   // angles of PASS (append: APASS, in fp32) tokens at the widest rotation

cudaError_t configure_code() {
  cudaError_t e = cudaSuccess;
  for (const void* f : {reinterpret_cast<const void*>(dg_kv8_rows_kernel<1>), reinterpret_cast<const void*>(dg_kv8_rows_kernel<2>),
                        reinterpret_cast<const void*>(dg_kv8_append_kernel<1>), reinterpret_cast<const void*>(dg_kv8_append_kernel<2>)})
    if (e == cudaSuccess) e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, int(ROWS_SMEM));
  return e;
}

cudaError_t launch_rows(const QueryParams& q, const CodeParams& p, const uint64_t* pos, uint32_t n_seq, cudaStream_t st) {
  PosList l = {};
  for (uint32_t b = 0; b < n_seq; ++b) l.pos[b] = pos[b];
  RowsPlan plan = {16, 1, 0, 1, 1, q.rows.C, 0};
  if (p.n_ctiles != 0u) {
    if (p.n <= 8u) {
      plan.slots = 1;
      while (plan.slots < p.n) plan.slots *= 2u;
      plan.per_seq = (q.rows.Hkv * 2u + 16u / plan.slots - 1u) / (16u / plan.slots);
      plan.canvas_ctas = n_seq * plan.per_seq;
    } else {
      const uint32_t tokens = p.n < BLK ? p.n : BLK;
      while (plan.cluster * 16u < tokens) plan.cluster *= 2u;
      const uint32_t most = row_heads(int(q.rows.D / 256u));
      plan.heads = q.rows.Hkv < most ? q.rows.Hkv : most;
      plan.per_seq = (q.rows.Hkv + plan.heads - 1u) / plan.heads * p.n_ctiles * 2u;
      plan.canvas_ctas = n_seq * plan.per_seq * plan.cluster;
    }
  }
  // the key weights sum over whole row tiles: rows behind the last token are zeros there
  if (q.lse != nullptr) plan.q_tokens = (q.rows.MT * BLK + q.rows.G - 1u) / q.rows.G;
  plan.q_ctas = n_seq * plan.q_tokens;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((plan.canvas_ctas + plan.q_ctas + plan.cluster - 1u) / plan.cluster * plan.cluster);
  cfg.blockDim = dim3(CT);
  cfg.dynamicSmemBytes = size_t(p.n_ctiles ? plan.slots : 1u) * q.rope.half * sizeof(double2);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = plan.cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return q.rows.D == 256 ? cudaLaunchKernelEx(&cfg, dg_kv8_rows_kernel<1>, q, p, l, plan) : cudaLaunchKernelEx(&cfg, dg_kv8_rows_kernel<2>, q, p, l, plan);
}

cudaError_t launch_append(const CodeParams& p, cudaStream_t st) {
  const uint32_t blocks = (p.n_keys + p.n + BLK - 1u) / BLK - p.n_keys / BLK, nj = p.D / 256u;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks * p.Hkv * 2u * nj);
  cfg.blockDim = dim3(CT);
  cfg.dynamicSmemBytes = p.ready ? 0 : size_t(APASS) * p.rope.half * sizeof(float2);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = nj;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return nj == 1 ? cudaLaunchKernelEx(&cfg, dg_kv8_append_kernel<1>, p) : cudaLaunchKernelEx(&cfg, dg_kv8_append_kernel<2>, p);
}

cudaError_t launch_read(const ReadParams& p, cudaStream_t st) {
  const uint64_t n = 2ull * p.n * p.Hkv * (p.D / 16u);
  const uint64_t ctas = (n + 255u) / 256u;
  return launch(dg_kv8_read_kernel, uint32_t(ctas < 148u * 64u ? ctas : 148u * 64u), 256, 0, st, p);
}

}  // namespace kv8
}  // namespace dg
