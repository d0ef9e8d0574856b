// What the host side's files share: error text, the context, checks of a layer, scratch.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cmath>
#include <deque>
#include <string>
#include <vector>

#include "dg_common.cuh"

using namespace dg;

// Not for other objects of the process: no name here leaves the library (an inline variable would otherwise be one for the whole
// process, whichever library defined it).
namespace dg {
namespace host __attribute__((visibility("hidden"))) {}
}  // namespace dg
using namespace dg::host;

// ------------------------------------------------------------------------------------------
// error plumbing
// ------------------------------------------------------------------------------------------
namespace dg {
namespace host {
std::string& last_error();           // this thread's (dg_api.cu)

inline int32_t fail_cuda(cudaError_t e, const char* what) {
  last_error() = std::string(what) + ": " + cudaGetErrorString(e);
  return DG_ERR_CUDA;
}
#define DG_CUDA(call)                                \
  do {                                               \
    cudaError_t e__ = (call);                        \
    if (e__ != cudaSuccess) return fail_cuda(e__, #call); \
  } while (0)

inline int32_t fail(int32_t code, const char* msg) {
  last_error() = msg;
  return code;
}
}  // namespace host
}  // namespace dg

// ------------------------------------------------------------------------------------------
// the context
// ------------------------------------------------------------------------------------------
struct dg_ctx {
  int device = 0;
  int num_sms = 0;
  cudaStream_t own_stream = nullptr;
  cudaStream_t stream = nullptr;
  DevStatus* d_status = nullptr;
  uint32_t concurrent = 1;             // canvases in flight together: the split heuristic counts their CTAs
  uint32_t* counters = nullptr;        // [kCounterSlots], zero between launches
  float* ws_o = nullptr;               // split partials
  float* ws_ml = nullptr;
  size_t ws_rows = 0;                  // capacity of ws_o / ws_ml: splits * rows (x 256 / x 2)
  std::vector<void*> outgrown;         // scratch that has been replaced by a larger buffer (grow_scratch)
  __nv_bfloat16* stage_q = nullptr;    // device staging for host-buffer calls / pre-normed Q
  __nv_bfloat16* stage_k = nullptr;
  __nv_bfloat16* stage_v = nullptr;
  __nv_bfloat16* stage_o = nullptr;
  size_t stage_q_elems = 0, stage_kv_elems = 0;
  float* nccl_pay = nullptr;           // [rows][D+1] payload of the cross-rank merge
  float* nccl_mg = nullptr;            // [rows]
  size_t nccl_rows = 0, nccl_d = 0;
  // dg_attn_block: activations between its kernels (normed input, Q, K, V, O, projected O, row sums of squares)
  __nv_bfloat16* blk_xn = nullptr;
  __nv_bfloat16* blk_q = nullptr;
  __nv_bfloat16* blk_k = nullptr;
  __nv_bfloat16* blk_v = nullptr;
  __nv_bfloat16* blk_o = nullptr;
  float* blk_part = nullptr;           // fp32 partial planes of the output projection, [4][rows][hidden]
  void* topk_plane = nullptr;          // dg_attn_denoise_topk: fp32 scores of a pass and their group maxima
  size_t topk_bytes = 0;
  uint4* bits = nullptr;               // dg_attn_denoise_bitmap: the packed bitmap [canvas][tiles] and its live-tile flags
  uint8_t* bits_live = nullptr;
  size_t bits_tiles = 0;               // capacity in 128-key tiles, for kMaxCanvas rows
  uint8_t* kv8_rows = nullptr;         // calls on 8-bit caches: the coded rows of a step
  uint8_t* kv8_part = nullptr;         // and the partial rows or sums of its splits
  size_t kv8_rows_bytes = 0, kv8_part_bytes = 0;
  size_t blk_rows = 0, blk_hidden = 0, blk_qe = 0, blk_ke = 0;
  CUtensorMap blk_tm_xn, blk_tm_o;
  struct WMap {
    const void* w;
    uint32_t n, k, bn;
    CUtensorMap tm;
  };
  std::deque<WMap> blk_wmaps;          // tensor maps of the weight matrices seen so far (a deque: growing it leaves
                                       // the addresses of its elements, which a call holds across two look-ups, alone)
  int q_from_prev_kernel = 0;          // 1 while dg_attn_block runs: Q is written by the kernel queued just ahead
  int force_general = 0;
  int fused_append = 1;                // 1: the canvas append runs inside the attention launch where it can
  int inputs_stable = 0;               // 1: the caller's q/k/v are not written by work queued ahead of a call
  int pair_mode = 2;                   // tensor path: 0 single-CTA kernel, 1 CTA-pair (cta_group::2) kernel, 2 automatic
  uint32_t forced_splits = 0;
  uint32_t last_launches = 0;
  // optional per-launch timing of the attention kernel (event pairs on the launching stream)
  unsigned long long* stamps = nullptr;   // caller-owned device buffer for per-CTA phase stamps
  bool timing = false;
  std::vector<cudaEvent_t> ev;
  size_t ev_used = 0;
};

// ------------------------------------------------------------------------------------------
// checks, scratch
// ------------------------------------------------------------------------------------------
namespace dg {
namespace host {
inline int32_t check_desc(const dg_layer_desc* d) {
  if (!d) return fail(DG_ERR_INVALID_ARG, "desc is NULL");
  if (d->n_q_heads == 0 || d->n_kv_heads == 0 || d->n_q_heads % d->n_kv_heads != 0)
    return fail(DG_ERR_INVALID_ARG, "n_q_heads must be a positive multiple of n_kv_heads");
  if (d->head_dim == 0 || d->head_dim % 8 != 0 || d->head_dim > kMaxHeadDim)
    return fail(DG_ERR_UNSUPPORTED, "head_dim must be a multiple of 8, at most 512");
  if (d->canvas == 0 || d->canvas > kMaxCanvas) return fail(DG_ERR_UNSUPPORTED, "canvas must be in 1..256");
  if (d->rotary_dim > d->head_dim || d->rotary_dim % 2 != 0)
    return fail(DG_ERR_INVALID_ARG, "rotary_dim must be even and <= head_dim");
  if (d->mask_mode > DG_MASK_CAUSAL) return fail(DG_ERR_INVALID_ARG, "unknown mask_mode");
  if (d->rope_pairing > DG_ROPE_PROPORTIONAL) return fail(DG_ERR_INVALID_ARG, "unknown rope_pairing");
  if (d->rope_pairing == DG_ROPE_SPLIT_HALF && d->rotary_dim / 2 + d->rotary_dim / 2 > d->head_dim)
    return fail(DG_ERR_INVALID_ARG, "rotary_dim too large");
  if (d->rope_pairing == DG_ROPE_PROPORTIONAL && d->rotary_dim / 2 > d->head_dim / 2)
    return fail(DG_ERR_INVALID_ARG, "rotary_dim too large for proportional pairing");
  if (!(d->softmax_scale > 0.f) || !std::isfinite(d->softmax_scale))
    return fail(DG_ERR_INVALID_ARG, "softmax_scale must be positive and finite");
  if (!(d->rope_theta > 0.f)) return fail(DG_ERR_INVALID_ARG, "rope_theta must be positive");
  return DG_OK;
}
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Scratch of the attention calls grows without a synchronisation and without freeing: a CUDA graph may hold the address of
// the buffer in use, work may be queued on it, and the stream may be under capture (the driver then allows the allocation
// only in the relaxed mode).  Buffers that became too small are kept until the context goes; their successors are twice as
// large where memory allows, so that a session that grows by a block at a time allocates rarely and all of them together
// stay below twice the last.  Two buffers of one capacity, na and nb elements of them per unit of it (nb = 0: one buffer).
template <class A, class B>
inline int32_t grow_scratch(dg_ctx* ctx, A** a, size_t na, B** b, size_t nb, size_t* cap, size_t need) {
  if (need <= *cap) return DG_OK;
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  DG_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
  cudaError_t e = cudaSuccess;
  for (const size_t n : {need > 2 * *cap ? need : 2 * *cap, need}) {
    A* fa = nullptr;
    B* fb = nullptr;
    e = cudaMalloc(&fa, n * na * sizeof(A));
    if (e == cudaSuccess && nb) e = cudaMalloc(&fb, n * nb * sizeof(B));
    if (e == cudaSuccess) {
      if (*a) ctx->outgrown.push_back(*a);
      if (*b) ctx->outgrown.push_back(*b);
      *a = fa;
      *b = fb;
      *cap = n;
      break;
    }
    cudaGetLastError();
    cudaFree(fa);
  }
  cudaThreadExchangeStreamCaptureMode(&mode);
  return e == cudaSuccess ? DG_OK : fail_cuda(e, "scratch allocation");
}
}  // namespace host
}  // namespace dg
