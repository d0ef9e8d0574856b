// C ABI of the caches held in 8 bits: objects, argument checks, split planning, launches (kernels: csrc/dg_kv8_*.cu).
#include <cmath>
#include <initializer_list>
#include <new>

#include "dg_host.h"
#include "dg_kv8.cuh"

namespace dg {
namespace kv8 {
cudaError_t configure_code();
cudaError_t configure_attn();
cudaError_t configure_weights();
cudaError_t configure_token();
cudaError_t configure_evict();
cudaError_t configure() {
  cudaError_t e = configure_code();
  if (e == cudaSuccess) e = configure_attn();
  if (e == cudaSuccess) e = configure_weights();
  if (e == cudaSuccess) e = configure_token();
  if (e == cudaSuccess) e = configure_evict();
  return e;
}
}  // namespace kv8
}  // namespace dg

using kv8::BLK;

struct dg_kv8 {
  dg_ctx* ctx = nullptr;
  int device = 0;
  uint8_t* k = nullptr;        // [Hkv][blocks][D / 128][128][128]
  uint8_t* v = nullptr;
  int32_t* exps = nullptr;     // [Hkv][blocks][2]: exponents of the scales of K and V
  uint32_t blocks = 0, Hkv = 0, D = 0;
};

static int32_t check_desc8(const dg_layer_desc* d) {
  const int32_t r = check_desc(d);
  if (r != DG_OK) return r;
  if (d->head_dim != 256 && d->head_dim != 512) return fail(DG_ERR_UNSUPPORTED, "caches in 8 bits: head_dim must be 256 or 512");
  if (d->rotary_dim % 16 != 0) return fail(DG_ERR_UNSUPPORTED, "caches in 8 bits: rotary_dim must be a multiple of 16");
  if (!(d->rms_eps >= 0.f)) return fail(DG_ERR_INVALID_ARG, "rms_eps must not be negative");
  return DG_OK;
}
static int32_t check_cache8(const dg_ctx* c, const dg_layer_desc& d, const dg_kv8* kv) {
  if (!kv) return fail(DG_ERR_INVALID_ARG, "kv is NULL");
  if (kv->Hkv != d.n_kv_heads || kv->D != d.head_dim) return fail(DG_ERR_INVALID_ARG, "kv geometry differs from desc");
  if (kv->device != c->device) return fail(DG_ERR_INVALID_ARG, "the cache lives on another device than the context");
  return DG_OK;
}
static int32_t check_aligned(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (!aligned16(p)) return fail(DG_ERR_ALIGNMENT, "device pointers must be 16-byte aligned");
  return DG_OK;
}
// Does [a, a + na) share a byte with [b, b + nb)?  (NULL: no memory.)
static bool overlap(const void* a, size_t na, const void* b, size_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a && b && x < y + nb && y < x + na;
}
static kv8::Rope make_rope8(const dg_layer_desc& d) {
  kv8::Rope r;
  r.half = d.rotary_dim / 2;
  r.dist = d.rope_pairing == DG_ROPE_SPLIT_HALF ? d.rotary_dim / 2 : d.head_dim / 2;
  r.log2_step = -2.0 / double(d.head_dim) * std::log2(double(d.rope_theta));
  return r;
}
static int32_t grow_bytes(dg_ctx* c, uint8_t** p, size_t* cap, size_t need) {
  uint8_t* none = nullptr;
  return grow_scratch(c, p, 1, &none, 0, cap, need);
}

extern "C" int32_t dg_kv8_create(dg_ctx* c, const dg_layer_desc* d, uint64_t capacity_tokens, dg_kv8** out) {
  if (!c || !out) return fail(DG_ERR_INVALID_ARG, "NULL argument");
  *out = nullptr;
  const int32_t r = check_desc8(d);
  if (r != DG_OK) return r;
  if (capacity_tokens == 0 || capacity_tokens > (1ull << 31) - BLK) return fail(DG_ERR_INVALID_ARG, "bad capacity");
  DG_CUDA(cudaSetDevice(c->device));
  dg_kv8* kv = new (std::nothrow) dg_kv8();
  if (!kv) return fail(DG_ERR_INVALID_ARG, "out of host memory");
  kv->ctx = c;
  kv->device = c->device;
  kv->blocks = uint32_t((capacity_tokens + BLK - 1) / BLK);
  kv->Hkv = d->n_kv_heads;
  kv->D = d->head_dim;
  const size_t tiles = size_t(kv->Hkv) * kv->blocks, bytes = tiles * BLK * kv->D;
  cudaError_t e = cudaMalloc(&kv->k, bytes);
  if (e == cudaSuccess) e = cudaMalloc(&kv->v, bytes);
  if (e == cudaSuccess) e = cudaMalloc(&kv->exps, tiles * 2 * sizeof(int32_t));
  // whole blocks are read and masked afterwards: every code is a finite number from the start
  if (e == cudaSuccess) e = cudaMemsetAsync(kv->k, 0, bytes, c->stream);
  if (e == cudaSuccess) e = cudaMemsetAsync(kv->v, 0, bytes, c->stream);
  if (e == cudaSuccess) e = cudaMemsetAsync(kv->exps, 0, tiles * 2 * sizeof(int32_t), c->stream);
  if (e != cudaSuccess) {
    dg_kv8_destroy(kv);
    return fail_cuda(e, "dg_kv8_create");
  }
  *out = kv;
  return DG_OK;
}

extern "C" int32_t dg_kv8_destroy(dg_kv8* kv) {
  if (!kv) return DG_OK;
  if (kv->ctx) {
    cudaSetDevice(kv->device);
    cudaStreamSynchronize(kv->ctx->stream);
  }
  cudaFree(kv->k);
  cudaFree(kv->v);
  cudaFree(kv->exps);
  delete kv;
  return DG_OK;
}

extern "C" uint64_t dg_kv8_capacity(const dg_kv8* kv) { return kv ? uint64_t(kv->blocks) * BLK : 0; }

static int32_t append8(dg_ctx* c, const dg_layer_desc* d, dg_kv8* kv, uint64_t n_keys, uint64_t pos, uint64_t n, const void* k,
                       const void* v, const void* kw) {
  if (n_keys > dg_kv8_capacity(kv) || n > dg_kv8_capacity(kv) - n_keys) return fail(DG_ERR_CAPACITY, "the tokens do not fit the cache");
  if (n == 0) return DG_OK;
  const int32_t r = check_aligned({k, v, kw});
  if (r != DG_OK) return r;
  DG_CUDA(cudaSetDevice(c->device));
  kv8::CodeParams p = {};
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.kw = static_cast<const __nv_bfloat16*>(kw);
  p.n = uint32_t(n);
  p.Hkv = kv->Hkv;
  p.D = kv->D;
  p.ready = d ? 0u : 1u;
  if (d) {
    p.v_norm = d->v_norm;
    p.eps = d->rms_eps;
    p.rope = make_rope8(*d);
  }
  p.status = c->d_status;
  p.k_codes = kv->k;
  p.v_codes = kv->v;
  p.exps = kv->exps;
  p.blocks = kv->blocks;
  p.n_keys = uint32_t(n_keys);
  p.pos = pos;
  c->last_launches = 1;
  DG_CUDA(kv8::launch_append(p, c->stream));
  return DG_OK;
}

extern "C" int32_t dg_kv8_append(dg_ctx* c, const dg_layer_desc* d, dg_kv8* kv, uint64_t n_keys, uint64_t pos, uint64_t n,
                                 const void* k, const void* v, const void* kw) {
  if (!c || !k || !v) return fail(DG_ERR_INVALID_ARG, "NULL argument");
  int32_t r = check_desc8(d);
  if (r == DG_OK) r = check_cache8(c, *d, kv);
  if (r != DG_OK) return r;
  if (pos > (1ull << 31) || n > (1ull << 31) || pos + n > (1ull << 31)) return fail(DG_ERR_CAPACITY, "position beyond 2^31");
  return append8(c, d, kv, n_keys, pos, n, k, v, kw);
}

static int32_t check_device_memory(const dg_kv8* kv, std::initializer_list<const void*> ps) {
  for (const void* p : ps) {
    cudaPointerAttributes at = {};
    if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
      cudaGetLastError();
      return fail(DG_ERR_INVALID_ARG, "not a device pointer");
    }
    if (!(at.type == cudaMemoryTypeDevice && at.device == kv->device) && at.type != cudaMemoryTypeManaged)
      return fail(DG_ERR_INVALID_ARG, "memory of the cache's device is needed");
  }
  return DG_OK;
}

extern "C" int32_t dg_kv8_load(dg_kv8* kv, uint64_t n_keys, uint64_t n, const void* k, const void* v) {
  if (!kv || !k || !v) return fail(DG_ERR_INVALID_ARG, "NULL argument");
  const int32_t r = check_device_memory(kv, {k, v});
  return r != DG_OK ? r : append8(kv->ctx, nullptr, kv, n_keys, 0, n, k, v, nullptr);
}

extern "C" int32_t dg_kv8_read(dg_kv8* kv, void* k_out, void* v_out, uint64_t slot0, uint64_t n) {
  if (!kv || !k_out || !v_out) return fail(DG_ERR_INVALID_ARG, "NULL argument");
  if (slot0 > dg_kv8_capacity(kv) || n > dg_kv8_capacity(kv) - slot0) return fail(DG_ERR_CAPACITY, "range outside the cache");
  if (n == 0) return DG_OK;
  int32_t r = check_aligned({k_out, v_out});
  if (r == DG_OK) r = check_device_memory(kv, {k_out, v_out});
  if (r != DG_OK) return r;
  DG_CUDA(cudaSetDevice(kv->device));
  kv8::ReadParams p = {};
  p.k = kv->k;
  p.v = kv->v;
  p.exps = kv->exps;
  p.blocks = kv->blocks;
  p.Hkv = kv->Hkv;
  p.D = kv->D;
  p.slot0 = uint32_t(slot0);
  p.n = uint32_t(n);
  p.k_out = static_cast<__nv_bfloat16*>(k_out);
  p.v_out = static_cast<__nv_bfloat16*>(v_out);
  kv->ctx->last_launches = 1;
  DG_CUDA(kv8::launch_read(p, kv->ctx->stream));
  return DG_OK;
}

// ------------------------------------------------------------------------------------------
// attention
// ------------------------------------------------------------------------------------------
namespace {

// Workspace of the rows of a step, in bytes from its start.
struct RowsLayout {
  size_t q, row, ck, cv, cexp, total;
};
RowsLayout rows_layout(const dg_layer_desc& d, uint32_t n_seq, uint32_t MT, uint32_t n_ctiles) {
  const size_t heads = size_t(n_seq) * d.n_kv_heads, D = d.head_dim;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  RowsLayout l;
  size_t at = 0;
  l.q = at;
  at = up(at + heads * MT * 2 * BLK * D);
  l.row = at;
  at = up(at + heads * MT * BLK * sizeof(float2));
  l.ck = at;
  at = up(at + heads * n_ctiles * 2 * BLK * D);
  l.cv = at;
  at = up(at + heads * n_ctiles * 2 * BLK * D);
  l.cexp = at;
  at = up(at + heads * n_ctiles * 2 * sizeof(int32_t));
  l.total = at;
  return l;
}

kv8::QueryParams query_params(const dg_layer_desc& d, uint8_t* ws, const RowsLayout& l, uint32_t MT) {
  kv8::QueryParams q = {};
  q.rows.codes = ws + l.q;
  q.rows.row = reinterpret_cast<float2*>(ws + l.row);
  q.rows.C = d.canvas;
  q.rows.Hq = d.n_q_heads;
  q.rows.Hkv = d.n_kv_heads;
  q.rows.G = d.n_q_heads / d.n_kv_heads;
  q.rows.D = d.head_dim;
  q.rows.MT = MT;
  q.eps = d.rms_eps;
  q.scale_log2 = d.softmax_scale * 1.4426950408889634f;
  q.rope = make_rope8(d);
  return q;
}

// How many splits the key tiles of each sequence are cut into, so that the launch's CTAs end together: `per` tiles a CTA at
// most, all CTAs of a wave side by side.  Costs in key tiles of a CTA (1.6 us): ten for what a wave costs beside its tiles; the
// merge, 2 us and the partial rows' way through memory, 0.33 ns for each row and split.  One canvas of 256 rows, us: 32,768 keys
// of 2 KV heads, splits 1 / 2 / 3 / 4 / 5 / 7 / 9: 456 / 248 / 176 / 142 / 226 / 183 / 154; head_dim 512, 1 / 2 / 3 / 4 / 9: 560 / 324 /
// 451 / 348 / 408; window 1024 of 8 KV heads, 1 / 2 / 3 / 4 / 5: 47 / 42 / 36 / 34 / 60; one token over 333 keys, 1 / 2 / 3: 11.8 /
// 12.1 / 11.5.
// Single tokens (dg_kv8_token_kernel) have all dims in one CTA and shorter tiles (1 us and less); the merge is a second launch of
// 3 us behind 10.
constexpr uint32_t kFixed8 = 10, kFixedToken = 6, kMerge8 = 1400, kMergeToken = 3500;
uint32_t plan_splits(const dg_ctx* c, kv8::Seq* seq, uint32_t n_seq, uint32_t base, uint64_t rows, uint32_t fixed, uint32_t merge,
                     const uint32_t* cost, uint32_t* most_splits) {
  const uint32_t sms = c->num_sms > 0 ? uint32_t(c->num_sms) : 148u;
  uint32_t most = 1;
  for (uint32_t b = 0; b < n_seq; ++b) most = cost[b] > most ? cost[b] : most;
  uint32_t best = most;
  uint64_t best_cost = ~0ull;
  for (uint32_t S = 1; S <= 128 && S <= most; ++S) {
    const uint32_t per = (most + S - 1) / S;
    uint64_t ctas = 0;
    for (uint32_t b = 0; b < n_seq; ++b) ctas += uint64_t(base) * (cost[b] <= per ? 1u : (cost[b] + per - 1) / per);
    const uint64_t waves = (ctas + sms - 1) / sms;
    const uint64_t t = waves * (per + fixed) * 1000 + (S == 1 ? 0 : merge + rows * S * 23 / 100);
    if (t < best_cost) {
      best_cost = t;
      best = per;
    }
  }
  uint32_t ctas = 0;
  *most_splits = 1;
  for (uint32_t b = 0; b < n_seq; ++b) {
    uint32_t s = cost[b] <= best ? 1u : (cost[b] + best - 1) / best;
    if (c->forced_splits) s = c->forced_splits < cost[b] ? c->forced_splits : (cost[b] ? cost[b] : 1u);
    seq[b].first_cta = ctas;
    seq[b].n_splits = s;
    ctas += base * s;
    *most_splits = s > *most_splits ? s : *most_splits;
  }
  return ctas;
}

}  // namespace

extern "C" int32_t dg_kv8_denoise(dg_ctx* c, const dg_layer_desc* d, dg_kv8* const* kv, const uint32_t* n_keys, const uint64_t* pos,
                                  uint32_t batch, const void* q, const void* k, const void* v, const void* qw, const void* kw,
                                  void* out, float* lse, void* q_rot) {
  if (!c || !kv || !n_keys || !q || !out) return fail(DG_ERR_INVALID_ARG, "NULL argument");
  if ((k == nullptr) != (v == nullptr)) return fail(DG_ERR_INVALID_ARG, "k and v are both given, or neither");
  int32_t r = check_desc8(d);
  if (r != DG_OK) return r;
  if (batch == 0) return fail(DG_ERR_INVALID_ARG, "batch must be positive");
  const bool windowed = d->mask_mode != DG_MASK_NONE && d->window != 0;
  for (uint32_t b = 0; b < batch; ++b) {
    r = check_cache8(c, *d, kv[b]);
    if (r != DG_OK) return r;
    if (n_keys[b] > dg_kv8_capacity(kv[b])) return fail(DG_ERR_CAPACITY, "n_keys exceeds the cache");
    const uint64_t at = pos ? pos[b] : n_keys[b];
    if (at > (1ull << 31) - d->canvas) return fail(DG_ERR_CAPACITY, "position beyond 2^31");
    if (windowed && at != n_keys[b])
      return fail(DG_ERR_INVALID_ARG, "a window counts positions: it needs pos = n_keys (no eviction)");
  }
  r = check_aligned({q, k, v, qw, kw, out, q_rot});
  if (r != DG_OK) return r;
  if (reinterpret_cast<uintptr_t>(lse) & 3u) return fail(DG_ERR_ALIGNMENT, "lse must be 4-byte aligned");
  const uint32_t C = d->canvas, G = d->n_q_heads / d->n_kv_heads, D = d->head_dim;
  {
    // several CTAs may read a row of q, k or v, and not all at the time when another writes outputs
    const size_t nq = size_t(batch) * C * d->n_q_heads * D * 2, nk = nq / G, nl = size_t(batch) * C * d->n_q_heads * 4;
    const struct { const void* p; size_t n; } outs[3] = {{out, nq}, {q_rot, nq}, {lse, nl}}, ins[5] = {{q, nq}, {k, nk}, {v, nk}, {qw, D * 2u}, {kw, D * 2u}};
    for (int i = 0; i < 3; ++i) {
      for (const auto& x : ins)
        if (overlap(outs[i].p, outs[i].n, x.p, x.n)) return fail(DG_ERR_INVALID_ARG, "an output overlaps an input");
      for (int j = 0; j < i; ++j)
        if (overlap(outs[i].p, outs[i].n, outs[j].p, outs[j].n)) return fail(DG_ERR_INVALID_ARG, "two outputs overlap");
    }
  }
  DG_CUDA(cudaSetDevice(c->device));
  const uint32_t MT = (C * G + BLK - 1) / BLK, n_ctiles = k ? (C + BLK - 1) / BLK : 0, KU = D / 256;
  const bool token = C * G <= kv8::TOKEN_ROWS && C <= kv8::TOKEN_CANVAS;
  const size_t q_elems = size_t(C) * d->n_q_heads * D, kv_elems = size_t(C) * d->n_kv_heads * D;
  c->last_launches = 0;
  for (uint32_t b0 = 0; b0 < batch; b0 += kv8::MAX_SEQ) {
    const uint32_t n = batch - b0 < kv8::MAX_SEQ ? batch - b0 : kv8::MAX_SEQ;
    kv8::AttnParams8 p = {};
    p.n_seq = n;
    p.C = C;
    p.Hq = d->n_q_heads;
    p.Hkv = d->n_kv_heads;
    p.G = G;
    p.D = D;
    p.MT = MT;
    p.include_canvas = k ? 1u : 0u;
    p.mode = d->mask_mode;
    p.windowed = windowed ? 1u : 0u;
    p.wm1 = windowed ? d->window - 1u : 0u;
    p.n_ctiles = n_ctiles;
    p.out = static_cast<__nv_bfloat16*>(out) + b0 * q_elems;
    p.lse = lse ? lse + size_t(b0) * C * d->n_q_heads : nullptr;
    p.status = c->d_status;
    uint64_t at[kv8::MAX_SEQ];
    uint32_t cost[kv8::MAX_SEQ];
    for (uint32_t b = 0; b < n; ++b) {
      const dg_kv8* x = kv[b0 + b];
      kv8::Seq& s = p.seq[b];
      s.k = x->k;
      s.v = x->v;
      s.exps = reinterpret_cast<const int2*>(x->exps);
      s.blocks = x->blocks;
      s.n_keys = n_keys[b0 + b];
      at[b] = pos ? pos[b0 + b] : s.n_keys;
      const kv8::Tiles t = kv8::tiles_of(kv8::seq_mask(p, s.n_keys), 0, C - 1);
      cost[b] = token ? t.nA : kv8::tile_cost(t);
    }
    uint32_t splits = 1;
    const uint64_t rows = uint64_t(n) * C * d->n_q_heads * KU;
    const uint32_t ctas = plan_splits(c, p.seq, n, token ? p.Hkv : p.Hkv * MT * KU, rows, token ? kFixedToken : kFixed8, token ? kMergeToken : kMerge8,
                                      cost, &splits);
    if (splits > 1) {
      const size_t slots = size_t(ctas) * (token ? KU : 1u) * BLK;
      r = grow_bytes(c, &c->kv8_part, &c->kv8_part_bytes, slots * (256 * sizeof(float) + sizeof(float2)));
      if (r != DG_OK) return r;
      p.ws_o = reinterpret_cast<float*>(c->kv8_part);
      p.ws_ml = reinterpret_cast<float2*>(c->kv8_part + slots * 256 * sizeof(float));
    }
    const __nv_bfloat16* qb = static_cast<const __nv_bfloat16*>(q) + b0 * q_elems;
    const __nv_bfloat16* kb = k ? static_cast<const __nv_bfloat16*>(k) + b0 * kv_elems : nullptr;
    const __nv_bfloat16* vb = v ? static_cast<const __nv_bfloat16*>(v) + b0 * kv_elems : nullptr;
    __nv_bfloat16* rot = q_rot ? static_cast<__nv_bfloat16*>(q_rot) + b0 * q_elems : nullptr;
    if (token) {
      kv8::TokenParams t = {};
      for (uint32_t b = 0; b < n; ++b) {
        t.seq[b] = p.seq[b];
        t.pos[b] = at[b];
        p.seq[b].first_cta *= KU;                 // the merge counts in 256 columns
      }
      t.n_seq = n;
      t.C = C;
      t.Hq = p.Hq;
      t.Hkv = p.Hkv;
      t.G = G;
      t.D = D;
      t.mode = p.mode;
      t.windowed = p.windowed;
      t.wm1 = p.wm1;
      t.v_norm = d->v_norm;
      t.q = qb;
      t.k = kb;
      t.v = vb;
      t.qw = static_cast<const __nv_bfloat16*>(qw);
      t.kw = static_cast<const __nv_bfloat16*>(kw);
      t.q_rot = rot;
      t.out = p.out;
      t.lse = p.lse;
      t.ws_o = p.ws_o;
      t.ws_ml = p.ws_ml;
      t.status = c->d_status;
      t.eps = d->rms_eps;
      t.scale_log2 = d->softmax_scale * 1.4426950408889634f;
      t.rope = make_rope8(*d);
      DG_CUDA(kv8::launch_token(t, D, ctas, c->stream));
      if (splits > 1) DG_CUDA(kv8::launch_merge(p, splits, c->stream));
      c->last_launches += splits > 1 ? 2 : 1;
      continue;
    }
    const RowsLayout l = rows_layout(*d, n, MT, n_ctiles);
    r = grow_bytes(c, &c->kv8_rows, &c->kv8_rows_bytes, l.total);
    if (r != DG_OK) return r;
    uint8_t* ws = c->kv8_rows;
    kv8::QueryParams qp = query_params(*d, ws, l, MT);
    qp.q = qb;
    qp.qw = static_cast<const __nv_bfloat16*>(qw);
    qp.q_rot = rot;
    kv8::CodeParams cp = {};
    cp.k = kb;
    cp.v = vb;
    cp.kw = static_cast<const __nv_bfloat16*>(kw);
    cp.n = C;
    cp.Hkv = d->n_kv_heads;
    cp.D = D;
    cp.v_norm = d->v_norm;
    cp.eps = d->rms_eps;
    cp.rope = qp.rope;
    cp.status = c->d_status;
    cp.k_codes = ws + l.ck;
    cp.v_codes = ws + l.cv;
    cp.exps = reinterpret_cast<int32_t*>(ws + l.cexp);
    cp.n_ctiles = n_ctiles;
    p.q_codes = ws + l.q;
    p.q_row = reinterpret_cast<const float2*>(ws + l.row);
    p.c_k = ws + l.ck;
    p.c_v = ws + l.cv;
    p.c_exps = reinterpret_cast<const int2*>(cp.exps);
    DG_CUDA(kv8::launch_rows(qp, cp, at, n, c->stream));
    DG_CUDA(kv8::launch_attention(p, D == 512 && MT % 2 == 0, ctas, splits, c->stream));
    c->last_launches += splits > 1 ? 3 : 2;
  }
  return DG_OK;
}

extern "C" int32_t dg_kv8_key_weights(dg_ctx* c, const dg_layer_desc* d, dg_kv8* kv, uint32_t n_keys, const void* q_rot, const float* lse,
                                      float* weights, uint64_t ld, float decay) {
  if (!c || !q_rot || !lse || !weights) return fail(DG_ERR_INVALID_ARG, "NULL argument");
  int32_t r = check_desc8(d);
  if (r == DG_OK) r = check_cache8(c, *d, kv);
  if (r != DG_OK) return r;
  if (n_keys > dg_kv8_capacity(kv)) return fail(DG_ERR_CAPACITY, "n_keys exceeds the cache");
  if (ld < n_keys) return fail(DG_ERR_INVALID_ARG, "ld is less than n_keys");
  if (!std::isfinite(decay) || decay < 0.f) return fail(DG_ERR_INVALID_ARG, "decay must be finite and not negative");
  r = check_aligned({q_rot});
  if (r != DG_OK) return r;
  if ((reinterpret_cast<uintptr_t>(lse) & 3u) || (reinterpret_cast<uintptr_t>(weights) & 3u))
    return fail(DG_ERR_ALIGNMENT, "lse and weights must be 4-byte aligned");
  {
    const size_t rows = size_t(d->canvas) * d->n_q_heads, n_w = ((d->n_kv_heads - 1) * ld + n_keys) * 4;
    if (overlap(weights, n_w, q_rot, rows * d->head_dim * 2) || overlap(weights, n_w, lse, rows * 4))
      return fail(DG_ERR_INVALID_ARG, "weights overlaps an input");
  }
  c->last_launches = 0;
  if (n_keys == 0) return DG_OK;
  DG_CUDA(cudaSetDevice(c->device));
  const uint32_t C = d->canvas, G = d->n_q_heads / d->n_kv_heads, D = d->head_dim, MT = (C * G + BLK - 1) / BLK;
  const RowsLayout l = rows_layout(*d, 1, MT, 0);
  r = grow_bytes(c, &c->kv8_rows, &c->kv8_rows_bytes, l.total);
  if (r != DG_OK) return r;
  kv8::QueryParams qp = query_params(*d, c->kv8_rows, l, MT);
  qp.q = static_cast<const __nv_bfloat16*>(q_rot);
  qp.lse = lse;
  qp.status = c->d_status;
  qp.prenormed = 1;
  qp.rope.half = 0;
  kv8::WeightParams p = {};
  p.q_codes = qp.rows.codes;
  p.q_row = qp.rows.row;
  p.k = kv->k;
  p.exps = reinterpret_cast<const int2*>(kv->exps);
  p.blocks = kv->blocks;
  p.n_keys = n_keys;
  p.C = C;
  p.Hkv = d->n_kv_heads;
  p.G = G;
  p.MT = MT;
  p.mode = d->mask_mode;
  p.windowed = d->mask_mode != DG_MASK_NONE && d->window != 0 ? 1u : 0u;
  p.wm1 = p.windowed ? d->window - 1u : 0u;
  p.w = weights;
  p.ld = ld;
  p.decay = decay;
  p.status = c->d_status;
  // One CTA a run of keys, or an even cut of all steps with the runs shared at the cuts and a second launch for the sums: by
  // steps a CTA (1.3 us and less), 2 for what a run costs beside its steps, 4 for the launch.  us by runs / cut evenly, a canvas
  // of 256 over 2 KV heads of head_dim 256: 2,000 keys 30.7 / 22.1, 8,191 33.4 / 27.6, 19,200 59.2 / 43.0, 32,768 60.4 / 61.8,
  // 45,000 86.8 / 80.0; a canvas of 64, head_dim 512: 8,191 15.6 / 20.7, 19,200 36.7 / 30.8.
  const uint32_t rows = C * G, blocks = (n_keys + BLK - 1) / BLK;
  const bool pair = D == 512 && rows >= 512;   // csrc/dg_kv8_weights.cu has both sides
  const uint32_t sms = (c->num_sms > 0 ? uint32_t(c->num_sms) : 148u) / (pair ? 2u : 1u), kt = 512 / D * (pair ? 2u : 1u);
  {
    MaskParams mk = make_mask(*d, n_keys, 0, n_keys, 0);
    const uint32_t lo = mask_row_lo(mk, 0), last = (blocks + kt - 1) / kt - 1;
    p.run0 = lo / BLK / kt < last ? lo / BLK / kt : last;
  }
  const uint32_t nr = D == 256 || pair ? 128u : 64u;   // rows of a step
  const uint32_t runs = ((blocks + kt - 1) / kt - p.run0) * p.Hkv, steps = (rows + nr - 1) / nr;
  const uint64_t units = uint64_t(runs) * steps;
  uint32_t ctas = runs;
  const uint32_t whole = (runs + sms - 1) / sms * (steps + 2);
  const uint32_t even = uint32_t(units < sms ? units : sms), per = uint32_t((units + even - 1) / even);
  if (per + 2u * (per / steps + 1u) + 4u < whole) {
    ctas = even;
    const uint32_t pieces = steps / uint32_t(units / even) + 2u;   // CTAs that a run's stages can be spread over
    r = grow_bytes(c, &c->kv8_part, &c->kv8_part_bytes, size_t(pieces) * p.Hkv * n_keys * sizeof(float));
    if (r != DG_OK) return r;
    p.part = reinterpret_cast<float*>(c->kv8_part);
  }
  const uint64_t at = 0;
  DG_CUDA(kv8::launch_rows(qp, kv8::CodeParams{}, &at, 1, c->stream));
  DG_CUDA(kv8::launch_weights(p, D, pair, ctas, c->stream));
  c->last_launches = p.part ? 3 : 2;
  return DG_OK;
}

extern "C" int32_t dg_kv8_evict(dg_ctx* c, dg_kv8* from, uint32_t n_keys, const float* weights, uint64_t ld, uint32_t n_keep,
                                uint32_t n_recent, dg_kv8* to, int32_t* kept, float* weights_out, uint64_t ld_out) {
  if (!c || !from || !to || !weights || !kept) return fail(DG_ERR_INVALID_ARG, "NULL argument");
  if (from == to) return fail(DG_ERR_INVALID_ARG, "a cache is evicted into another one");
  if (from->Hkv != to->Hkv || from->D != to->D) return fail(DG_ERR_INVALID_ARG, "the two caches differ in geometry");
  if (from->device != c->device || to->device != c->device)
    return fail(DG_ERR_INVALID_ARG, "the cache lives on another device than the context");
  if (n_keys > dg_kv8_capacity(from) || n_keep > dg_kv8_capacity(to)) return fail(DG_ERR_CAPACITY, "the tokens do not fit the cache");
  if (n_keep == 0 || n_keep > n_keys || n_recent > n_keep) return fail(DG_ERR_INVALID_ARG, "0 < n_keep <= n_keys and n_recent <= n_keep are needed");
  if (ld < n_keys || (weights_out && ld_out < n_keep)) return fail(DG_ERR_INVALID_ARG, "a row of weights is shorter than its tokens");
  for (const void* p : {static_cast<const void*>(weights), static_cast<const void*>(kept), static_cast<const void*>(weights_out)})
    if (reinterpret_cast<uintptr_t>(p) & 3u) return fail(DG_ERR_ALIGNMENT, "weights and kept must be 4-byte aligned");
  const size_t heads = from->Hkv - 1, n_w = (heads * ld + n_keys) * 4, n_o = (heads * ld_out + n_keep) * 4, n_i = (heads + 1) * n_keep * 4;
  if (overlap(weights, n_w, weights_out, n_o)) return fail(DG_ERR_INVALID_ARG, "weights_out overlaps weights");
  if (overlap(kept, n_i, weights, n_w) || overlap(kept, n_i, weights_out, n_o)) return fail(DG_ERR_INVALID_ARG, "kept overlaps weights");
  DG_CUDA(cudaSetDevice(c->device));
  kv8::EvictParams p = {};
  p.w = weights;
  p.ld = ld;
  p.n_keys = n_keys;
  p.n_keep = n_keep;
  p.n_recent = n_recent;
  p.Hkv = from->Hkv;
  p.D = from->D;
  p.kept = kept;
  p.w_out = weights_out;
  p.ld_out = ld_out;
  p.k = from->k;
  p.v = from->v;
  p.exps = from->exps;
  p.blocks = from->blocks;
  p.to_k = to->k;
  p.to_v = to->v;
  p.to_exps = to->exps;
  p.to_blocks = to->blocks;
  c->last_launches = 2;
  DG_CUDA(kv8::launch_evict(p, c->stream));
  return DG_OK;
}
