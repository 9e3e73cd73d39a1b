// extern "C" boundary of libsage_mi355x.so: argument validation, error
// reporting and dispatch to the gfx950 kernels.  See include/sage_mi355x.h.
#include <stdio.h>
#include <stdarg.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <chrono>
#include <cstdlib>
#include <mutex>

#include "../../include/sage_mi355x.h"
#include "sage_common.h"

#include "sage_launch.h"

namespace {

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int64_t kAttnMaxN = (int64_t)1 << 22;  // sage_attn_fwd's sequence-length limit
// Workgroups of one 1D launch of 256-thread workgroups (the dispatch packet
// holds the grid in work-items, a 32-bit count).
constexpr int64_t kMaxGridUnits = ((int64_t)1 << 24) - 1;

int check_common(int64_t bh, int64_t n, int64_t d, int qk, int pv, int gran) {
  if (bh <= 0 || n <= 0) return fail(SAGE_ERR_ARG, "bh=%lld and n=%lld must be positive", (long long)bh, (long long)n);
  if (d != 64 && d != 128) return fail(SAGE_ERR_ARG, "head_dim must be 64 or 128, got %lld", (long long)d);
  if (qk != SAGE_QK_INT8 && qk != SAGE_QK_FP8) return fail(SAGE_ERR_ARG, "unknown qk_kind %d", qk);
  if (pv != SAGE_PV_BF16 && pv != SAGE_PV_FP8) return fail(SAGE_ERR_ARG, "unknown pv_kind %d", pv);
  if (gran != SAGE_GRAN_TOKEN && gran != SAGE_GRAN_BLOCK64) return fail(SAGE_ERR_ARG, "unknown granularity %d", gran);
  if (bh > 65535) return fail(SAGE_ERR_ARG, "bh=%lld exceeds the grid limit 65535", (long long)bh);
  if (n > (int64_t)1 << 24) return fail(SAGE_ERR_ARG, "n=%lld exceeds 2^24", (long long)n);
  return SAGE_OK;
}

int launch_status(hipError_t e, const char* what) {
  if (e != hipSuccess) return fail(SAGE_ERR_LAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
  g_err[0] = '\0';
  return SAGE_OK;
}

}  // namespace

extern "C" {

int sage_abi_version(void) { return SAGE_ABI_VERSION; }

const char* sage_last_error(void) { return g_err; }

int64_t sage_padded_len(int64_t n) { return sage::padded_len(n); }

size_t sage_quant_workspace_bytes(int64_t bh, int64_t n, int64_t d) { return sage::quant_workspace_bytes(bh, n, d); }

size_t sage_attn_workspace_bytes(int64_t b, int64_t h, int64_t n, int64_t d) {
  return sage::attn_workspace_bytes(b, h, n, d);
}

size_t sage_attn_masked_workspace_bytes(int64_t b, int64_t h, int64_t n, int64_t d) {
  return sage::attn_workspace_bytes(b, h, n, d, true);
}

}  // extern "C"

namespace {

// Outputs and workspace of a quantization call.
int check_quant_outputs(int64_t bh, int64_t n, int64_t d, int64_t h_producer, int pv_kind, int smooth_k,
                        const void* q_codes,
                        const float* q_scale, const void* k_codes, const float* k_scale, const void* v_out,
                        const float* v_scale, const void* k_mean, const void* workspace, size_t workspace_bytes) {
  if (!q_codes || !q_scale || !k_codes || !k_scale || !v_out) return fail(SAGE_ERR_ARG, "null tensor pointer");
  if (pv_kind == SAGE_PV_FP8 && !v_scale) return fail(SAGE_ERR_ARG, "fp8 PV needs v_scale");
  const void* ptrs[] = {q_codes, q_scale, k_codes, k_scale, v_out};
  for (const void* p : ptrs)
    if (!aligned16(p)) return fail(SAGE_ERR_ALIGN, "tensor pointers must be 16-byte aligned");
  if (v_scale && !aligned16(v_scale)) return fail(SAGE_ERR_ALIGN, "v_scale must be 16-byte aligned");
  const int64_t units = sage::quant_grid_units(bh, n, d, h_producer);
  if (units > kMaxGridUnits)
    return fail(SAGE_ERR_ARG, "quantizing bh=%lld x n=%lld takes %lld workgroups, beyond one launch's %lld",
                (long long)bh, (long long)n, (long long)units, (long long)kMaxGridUnits);
  if (smooth_k) {
    if (!k_mean) return fail(SAGE_ERR_ARG, "smooth_k needs k_mean");
    const size_t need = sage::quant_workspace_bytes(bh, n, d);
    if (!workspace || workspace_bytes < need)
      return fail(SAGE_ERR_WORKSPACE, "workspace of %zu bytes needed, got %zu", need, workspace_bytes);
    if (!aligned16(workspace)) return fail(SAGE_ERR_ALIGN, "workspace must be 16-byte aligned");
  }
  return SAGE_OK;
}

// Inputs of the q/k/v producer.
int check_producer(const void* qkv, const float* q_norm_w, const float* k_norm_w, const float* freqs, int64_t b,
                   int64_t h, int64_t n, int64_t d, float norm_eps, sage::ProdArgs& prod) {
  if (b <= 0 || h <= 0) return fail(SAGE_ERR_ARG, "b=%lld and h=%lld must be positive", (long long)b, (long long)h);
  if (b * h > 65535) return fail(SAGE_ERR_ARG, "b*h=%lld exceeds the grid limit 65535", (long long)(b * h));
  if (n <= 0) return fail(SAGE_ERR_ARG, "n=%lld must be positive", (long long)n);
  if (n > (int64_t)1 << 24) return fail(SAGE_ERR_ARG, "n=%lld exceeds 2^24", (long long)n);
  if (d != 64 && d != 128) return fail(SAGE_ERR_ARG, "head_dim must be 64 or 128, got %lld", (long long)d);
  if (!qkv || !q_norm_w || !k_norm_w || !freqs) return fail(SAGE_ERR_ARG, "null tensor pointer");
  const void* ptrs[] = {qkv, q_norm_w, k_norm_w, freqs};
  for (const void* p : ptrs)
    if (!aligned16(p)) return fail(SAGE_ERR_ALIGN, "tensor pointers must be 16-byte aligned");
  if (!(norm_eps >= 0.0f)) return fail(SAGE_ERR_ARG, "norm_eps must be >= 0");
  // at most one launch's workgroups of one per (64-token block, head)
  if (b * h * ((n + 63) / 64) > kMaxGridUnits)
    return fail(SAGE_ERR_ARG, "b*h*ceil(n/64) = %lld exceeds the grid limit", (long long)(b * h * ((n + 63) / 64)));
  // the standalone producer and its backward: one per (pass of 256/(d/8) tokens, group of kSlabHeads heads)
  const int64_t rpp = 256 / (d / 8);
  const int64_t slabs = b * ((n + rpp - 1) / rpp) * ((h + sage::kSlabHeads - 1) / sage::kSlabHeads);
  if (slabs > kMaxGridUnits)
    return fail(SAGE_ERR_ARG, "%lld producer slabs exceed the grid limit", (long long)slabs);
  // 256 token rows of the projection output (3*h*d bf16 each) within 32-bit byte offsets
  if (3 * h * d * 2 * 256 > (int64_t)0xffffffff)
    return fail(SAGE_ERR_ARG, "3*h*d = %lld channels per token row is too wide for the producer", (long long)(3 * h * d));
  prod = sage::ProdArgs{static_cast<const uint16_t*>(qkv), q_norm_w, k_norm_w, freqs, (int)h, (int)(b * h),
                        norm_eps};
  return SAGE_OK;
}

// Backward workspace: byte offsets of the quantization's outputs (codes,
// scales, K mean, column-sum partials), the smoothed K rows, -D and the padded
// LSE.
struct BwdWorkspace {
  size_t qc, qs, kc, ks, kmean, quant, kt, neg_delta, lse_pad, sums, dq_part, dq_ctr, bytes;
};

BwdWorkspace bwd_workspace(int64_t b, int64_t bh, int64_t n, int64_t d) {
  const size_t np = (size_t)sage::padded_len(n), rows = (size_t)bh * np;
  BwdWorkspace w;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = (off + bytes + 255) & ~(size_t)255;
    return at;
  };
  w.qc = take(rows * d);
  w.qs = take(rows * 4);
  w.kc = take(rows * d);
  w.ks = take(rows * 4);
  w.kmean = take((size_t)bh * d * 2);
  w.quant = take(sage::quant_workspace_bytes(bh, n, d));
  w.kt = take(rows * d * 2);
  w.lse_pad = take(rows * 4);
  w.neg_delta = take(rows * 4);
  // document-id summaries (used with doc_ids): key tiles, 32- and 128-row blocks
  w.sums = take((size_t)b * ((n + 63) / 64 + np / 32 + np / 128) * sizeof(int4));
  // fp32 partial dQ of the cut items' two key-tile halves, their counters
  w.dq_part = take((size_t)sage::kBwdDqSplit * 2 * 128 * d * sizeof(float));
  w.dq_ctr = take((size_t)sage::kBwdDqSplit * sizeof(uint64_t));
  w.bytes = off;
  return w;
}

// Workspace of sage_forward: the quantization's outputs (sized for per-token
// scales, the larger granularity), its workspace, the attention's workspace.
struct ForwardWorkspace {
  size_t qc, qs, kc, ks, vop, vs, kmean, quant, attn, bytes;
};

ForwardWorkspace forward_workspace(int64_t b, int64_t h, int64_t n, int64_t d, int pv_kind, bool doc_ids) {
  const int64_t bh = b * h;
  const size_t np = (size_t)sage::padded_len(n), rows = (size_t)bh * np;
  ForwardWorkspace w;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = (off + bytes + 255) & ~(size_t)255;
    return at;
  };
  w.qc = take(rows * d);
  w.qs = take(rows * 4);
  w.kc = take(rows * d);
  w.ks = take(rows * 4);
  w.vop = take(rows * d * (pv_kind == SAGE_PV_FP8 ? 1 : 2));
  w.vs = take(pv_kind == SAGE_PV_FP8 ? rows / 64 * d * 4 : 0);
  w.kmean = take((size_t)bh * d * 2);
  w.quant = take(sage::quant_workspace_bytes(bh, n, d));
  w.attn = off;
  w.bytes = off + sage::attn_workspace_bytes(b, h, n, d, doc_ids);
  return w;
}

}  // namespace

extern "C" {

int sage_quantize_qkv(const void* q, const void* k, const void* v, int64_t bh, int64_t n, int64_t d, int qk_kind,
                      int pv_kind, int granularity, int smooth_k, float sm_scale_log2e, void* q_codes,
                      float* q_scale, void* k_codes, float* k_scale, void* v_out, float* v_scale, void* k_mean,
                      void* workspace, size_t workspace_bytes, hipStream_t stream) {
  int st = check_common(bh, n, d, qk_kind, pv_kind, granularity);
  if (st) return st;
  if (!q || !k || !v) return fail(SAGE_ERR_ARG, "null tensor pointer");
  const void* ins[] = {q, k, v};
  for (const void* p : ins)
    if (!aligned16(p)) return fail(SAGE_ERR_ALIGN, "tensor pointers must be 16-byte aligned");
  st = check_quant_outputs(bh, n, d, 0, pv_kind, smooth_k, q_codes, q_scale, k_codes, k_scale, v_out, v_scale, k_mean,
                           workspace, workspace_bytes);
  if (st) return st;
  hipError_t e = sage::launch_quantize(
      qk_kind, pv_kind, granularity, smooth_k != 0, static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k),
      static_cast<const uint16_t*>(v), bh, n, d, sm_scale_log2e, static_cast<double*>(workspace),
      static_cast<uint8_t*>(q_codes), q_scale, static_cast<uint8_t*>(k_codes), k_scale, static_cast<uint8_t*>(v_out),
      v_scale, static_cast<uint16_t*>(k_mean), sage::ProdArgs{}, stream);
  return launch_status(e, "sage_quantize_qkv");
}

int sage_qkv_postprocess(const void* qkv, const float* q_norm_w, const float* k_norm_w, const float* freqs,
                         int64_t b, int64_t h, int64_t n, int64_t d, float norm_eps, void* q_out, void* k_out,
                         void* v_out, hipStream_t stream) {
  sage::ProdArgs prod;
  int st = check_producer(qkv, q_norm_w, k_norm_w, freqs, b, h, n, d, norm_eps, prod);
  if (st) return st;
  if (!q_out || !k_out || !v_out) return fail(SAGE_ERR_ARG, "null tensor pointer");
  const void* outs[] = {q_out, k_out, v_out};
  for (const void* p : outs)
    if (!aligned16(p)) return fail(SAGE_ERR_ALIGN, "tensor pointers must be 16-byte aligned");
  return launch_status(sage::launch_qkv_postprocess(prod, b * h, n, d, static_cast<uint16_t*>(q_out),
                                                    static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out),
                                                    stream),
                       "sage_qkv_postprocess");
}

int sage_qkv_postprocess_bwd(const void* qkv, const float* q_norm_w, const float* k_norm_w, const float* freqs,
                             const void* grad_q, const void* grad_k, const void* grad_v, int64_t b, int64_t h,
                             int64_t n, int64_t d, float norm_eps, void* dqkv, hipStream_t stream) {
  sage::ProdArgs prod;
  int st = check_producer(qkv, q_norm_w, k_norm_w, freqs, b, h, n, d, norm_eps, prod);
  if (st) return st;
  if (!grad_q || !grad_k || !grad_v || !dqkv) return fail(SAGE_ERR_ARG, "null tensor pointer");
  const void* ptrs[] = {grad_q, grad_k, grad_v, dqkv};
  for (const void* p : ptrs)
    if (!aligned16(p)) return fail(SAGE_ERR_ALIGN, "tensor pointers must be 16-byte aligned");
  return launch_status(sage::launch_qkv_postprocess_bwd(prod, b * h, n, d, static_cast<const uint16_t*>(grad_q),
                                                        static_cast<const uint16_t*>(grad_k),
                                                        static_cast<const uint16_t*>(grad_v),
                                                        static_cast<uint16_t*>(dqkv), stream),
                       "sage_qkv_postprocess_bwd");
}

int sage_quantize_from_qkv(const void* qkv, const float* q_norm_w, const float* k_norm_w, const float* freqs,
                           int64_t b, int64_t h, int64_t n, int64_t d, float norm_eps, int qk_kind, int pv_kind,
                           int granularity, int smooth_k, float sm_scale_log2e, void* q_codes, float* q_scale,
                           void* k_codes, float* k_scale, void* v_out, float* v_scale, void* k_mean, void* workspace,
                           size_t workspace_bytes, hipStream_t stream) {
  sage::ProdArgs prod;
  int st = check_producer(qkv, q_norm_w, k_norm_w, freqs, b, h, n, d, norm_eps, prod);
  if (st) return st;
  st = check_common(b * h, n, d, qk_kind, pv_kind, granularity);
  if (st) return st;
  st = check_quant_outputs(b * h, n, d, h, pv_kind, smooth_k, q_codes, q_scale, k_codes, k_scale, v_out, v_scale,
                           k_mean, workspace, workspace_bytes);
  if (st) return st;
  hipError_t e = sage::launch_quantize(
      qk_kind, pv_kind, granularity, smooth_k != 0, nullptr, nullptr, nullptr, b * h, n, d, sm_scale_log2e,
      static_cast<double*>(workspace), static_cast<uint8_t*>(q_codes), q_scale, static_cast<uint8_t*>(k_codes),
      k_scale, static_cast<uint8_t*>(v_out), v_scale, static_cast<uint16_t*>(k_mean), prod, stream);
  return launch_status(e, "sage_quantize_from_qkv");
}

}  // extern "C"

namespace {

// A 56-bit tag never passed to an earlier attention launch of this process (a
// clock reading at first use, plus a call counter): the split items' arrival
// counters of other calls never match it (AttnParams::merge_ctr).
uint64_t next_merge_tag() {
  static std::atomic<uint64_t> counter{0};
  static const uint64_t base =
      (uint64_t)std::chrono::steady_clock::now().time_since_epoch().count() * 0x9E3779B97F4A7C15ull;
  return (base + counter.fetch_add(1, std::memory_order_relaxed) * 2 + 1) & (((uint64_t)1 << 56) - 1);
}

// The split items of unmasked launches merge in the attention kernel, unless
// SAGE_MERGE=kernel asks for the separate merge kernel (tests compare both).
bool merge_in_kernel() {
  const char* e = std::getenv("SAGE_MERGE");
  return e == nullptr || strcmp(e, "kernel") != 0;
}

// The backward cuts its last dQ items in two key halves unless
// SAGE_BWD_SPLIT=off (tests compare both).
bool bwd_split_enabled() {
  const char* e = std::getenv("SAGE_BWD_SPLIT");
  return e == nullptr || strcmp(e, "off") != 0;
}

// sage_attn_fwd and its variants: validation, workspace layout and launch.
// s_dump (int8 QK, per-token scales, no mask only) receives the S^T
// accumulators the kernel's loop consumes.
int attn_fwd_impl(const void* q_codes, const float* q_scale, const void* k_codes, const float* k_scale,
                  const void* v_in, const float* v_scale, int64_t b, int64_t h, int64_t n, int64_t d, int qk_kind,
                  int pv_kind, int granularity, const uint8_t* tile_mask, int64_t mask_stride_z, int64_t mask_nq,
                  int64_t mask_nkv, const int32_t* doc_ids, void* workspace, size_t workspace_bytes, void* out,
                  int out_layout, float* lse, int32_t* s_dump, const char* name, hipStream_t stream) {
  if (b <= 0 || h <= 0) return fail(SAGE_ERR_ARG, "b=%lld and h=%lld must be positive", (long long)b, (long long)h);
  int st = check_common(b * h, n, d, qk_kind, pv_kind, granularity);
  if (st) return st;
  if (!q_codes || !q_scale || !k_codes || !k_scale || !v_in || !out || !lse)
    return fail(SAGE_ERR_ARG, "null tensor pointer");
  if (pv_kind == SAGE_PV_FP8 && !v_scale) return fail(SAGE_ERR_ARG, "fp8 PV needs v_scale");
  const void* ptrs[] = {q_codes, q_scale, k_codes, k_scale, v_in, out};
  for (const void* p : ptrs)
    if (!aligned16(p)) return fail(SAGE_ERR_ALIGN, "tensor pointers must be 16-byte aligned");
  if (v_scale && !aligned16(v_scale)) return fail(SAGE_ERR_ALIGN, "v_scale must be 16-byte aligned");
  if (out_layout != SAGE_OUT_BHND && out_layout != SAGE_OUT_BNHD)
    return fail(SAGE_ERR_ARG, "out_layout must be 0 ([B,H,N,D]) or 1 ([B,N,H,D]), got %d", out_layout);
  // one head's operands are addressed through buffer resources with 32-bit
  // byte offsets: Np*D*2 bytes of bf16 V must stay below 2^31
  if (n > kAttnMaxN) return fail(SAGE_ERR_ARG, "n=%lld exceeds %lld for the attention", (long long)n, (long long)kAttnMaxN);
  // The epilogue addresses 32 output rows of one head in 32-bit byte offsets:
  // at most 32 * h*d*2 bytes, under 2^31 since b*h <= 65535 and d <= 128.
  const int64_t nq = (n + 127) / 128, nkv = (n + 63) / 64;
  int mask = 0;
  if (tile_mask) {
    if (mask_nq != nq || mask_nkv != nkv)
      return fail(SAGE_ERR_ARG, "block_mask must be %lld x %lld tiles, got %lld x %lld", (long long)nq,
                  (long long)nkv, (long long)mask_nq, (long long)mask_nkv);
    if (mask_stride_z != 0 && mask_stride_z != nq * nkv)
      return fail(SAGE_ERR_ARG, "mask_stride_z must be 0 (2D mask) or %lld (3D mask)", (long long)(nq * nkv));
    mask |= 1;
  }
  if (doc_ids) mask |= 2;
  sage::AttnParams p;
  memset(&p, 0, sizeof(p));
  // Masked launches need no partial slots.  With a tile mask alone and a
  // workspace that has room for them all the same (sage_attn_workspace_bytes,
  // or the scratch of the allocation-free entry point), items are
  // split as in an unmasked launch: the production op is always masked, and at
  // 1x30x4416 its 1050 items leave a third round of 26.  The pieces' slots stay
  // within kMaskedSplitBytes, so every entry point that has the room cuts the
  // same items.
  sage::AttnWorkspace ws = sage::attn_workspace(b, h, n, d, mask != 0);
  // a launch whose every item is cut runs whole in a workspace of the summaries
  // alone, the size it needs without the cut
  if (mask == 0 && ws.split.whole == 0 && workspace_bytes < ws.bytes) ws = sage::attn_workspace(b, h, n, d, true);
  sage::MaskedSplit shares{sage::TailSplit{b * h * nq, 1}, 0, 1};
  if (mask == 1 && merge_in_kernel()) {
    const sage::AttnWorkspace split = sage::attn_workspace(b, h, n, d, false, sage::kMaskedSplitBytes);
    if (workspace_bytes >= split.bytes) {
      ws = split;
      shares = sage::masked_split(split.split, b * h * nq, nkv);
    }
  }
  if (!workspace || workspace_bytes < ws.bytes)
    return fail(SAGE_ERR_WORKSPACE, "workspace of %zu bytes needed, got %zu", ws.bytes, workspace_bytes);
  if (!aligned16(workspace)) return fail(SAGE_ERR_ALIGN, "workspace must be 16-byte aligned");
  uint8_t* wsp = static_cast<uint8_t*>(workspace);
  if (doc_ids) {
    const int64_t nt = nkv;
    p.kv_sum = reinterpret_cast<const int4*>(wsp + ws.doc_off);
    p.q_sum = p.kv_sum + b * nt;
    p.q_sum128 = p.q_sum + b * (sage::padded_len(n) / 32);
    p.doc_range = p.q_sum128 + b * (sage::padded_len(n) / 128);
    p.heavy = reinterpret_cast<int4*>(wsp + ws.heavy_off);
    p.heavy_max = sage::kHeavyMax;
  }
  p.qc = static_cast<const uint8_t*>(q_codes);
  p.qs = q_scale;
  p.kc = static_cast<const uint8_t*>(k_codes);
  p.ks = k_scale;
  p.vin = static_cast<const uint8_t*>(v_in);
  p.vs = v_scale;
  p.tile_mask = tile_mask;
  p.mask_stride_z = mask_stride_z;
  p.mask_nkv = mask_nkv;
  p.doc = doc_ids;
  p.out = static_cast<uint16_t*>(out);
  if (out_layout == SAGE_OUT_BNHD) {
    p.out_bs = n * h * d;
    p.out_hs = d;
    p.out_rs = h * d;
  } else {
    p.out_bs = h * n * d;
    p.out_hs = n * d;
    p.out_rs = d;
  }
  p.lse = lse;
  p.n = n;
  p.np = sage::padded_len(n);
  p.h = (int)h;
  p.bh = (int)(b * h);
  p.nt = (int)nkv;
  p.light_last = (nq > 1 && n - (nq - 1) * 128 <= 64) ? 1 : 0;
  // cut the items of the last, partial dispatch round
  const sage::TailSplit split = mask == 0 ? ws.split : shares.split;
  p.n_whole = (int)split.whole;
  p.split_parts = split.parts;
  p.share_from = shares.share_from;
  p.share_min = shares.share_min;
  if (split.parts > 1) {
    p.part = reinterpret_cast<float*>(wsp + ws.part_off);
    if (merge_in_kernel()) {
      p.merge_ctr = reinterpret_cast<uint64_t*>(wsp + ws.ctr_off);
      p.merge_tag = next_merge_tag();
    }
  }
  if ((int64_t)p.bh * nq + (int64_t)sage::kHeavyMax * h + 8 * sage::kResidentWGs > kMaxGridUnits)
    return fail(SAGE_ERR_ARG, "b*h*ceil(n/128) = %lld exceeds the grid limit", (long long)(p.bh * nq));
  p.s_dump = s_dump;
  hipError_t e = sage::launch_attn(qk_kind, pv_kind, granularity, mask, p, d, (int)b, stream);
  return launch_status(e, name);
}

}  // namespace

extern "C" {

int sage_attn_fwd(const void* q_codes, const float* q_scale, const void* k_codes, const float* k_scale,
                  const void* v_in, const float* v_scale, int64_t b, int64_t h, int64_t n, int64_t d, int qk_kind,
                  int pv_kind, int granularity, const uint8_t* tile_mask, int64_t mask_stride_z, int64_t mask_nq,
                  int64_t mask_nkv, const int32_t* doc_ids, void* workspace, size_t workspace_bytes, void* out,
                  int out_layout, float* lse, hipStream_t stream) {
  return attn_fwd_impl(q_codes, q_scale, k_codes, k_scale, v_in, v_scale, b, h, n, d, qk_kind, pv_kind, granularity,
                       tile_mask, mask_stride_z, mask_nq, mask_nkv, doc_ids, workspace, workspace_bytes, out,
                       out_layout, lse, nullptr, "sage_attn_fwd", stream);
}

}  // extern "C"

namespace {

// Device scratch of sage_attn_fwd_noalloc: the document-id summaries and the
// split-tail partials that sage_attn_fwd keeps in its workspace argument.  An
// unmasked call may need SAGE_NOALLOC_SCRATCH_BYTES of it; the rest is for the
// pieces of tile-masked items.
// Each GPU the library runs on holds its own copy until the process ends.
// Host code never uses the array's name as an address: its device address
// comes from hipGetSymbolAddress, once per device, with that device current.
__device__ __align__(256) uint8_t scratch[sage::kMaskedSplitBytes];

constexpr int kMaxDevices = 64;
std::mutex g_scratch_mu;
void* g_scratch_ptr[kMaxDevices];

// Scratch address on the device of `stream`, which must be the current device.
int scratch_of_stream(hipStream_t stream, void** ptr) {
  int cur = -1, sdev = -1;
  hipError_t e = hipGetDevice(&cur);
  if (e == hipSuccess) e = hipStreamGetDevice(stream, &sdev);
  if (e != hipSuccess) return fail(SAGE_ERR_LAUNCH, "device of the stream: %s", hipGetErrorString(e));
  if (sdev != cur)
    return fail(SAGE_ERR_ARG, "the stream belongs to device %d, the current device is %d", sdev, cur);
  if (cur < 0 || cur >= kMaxDevices) return fail(SAGE_ERR_ARG, "device %d beyond the first %d", cur, kMaxDevices);
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (!g_scratch_ptr[cur]) {
    void* p = nullptr;
    e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    if (e != hipSuccess || !p)
      return fail(SAGE_ERR_LAUNCH, "hipGetSymbolAddress(scratch) failed: %s", hipGetErrorString(e));
    g_scratch_ptr[cur] = p;
  }
  *ptr = g_scratch_ptr[cur];
  return SAGE_OK;
}

}  // namespace

extern "C" {

int sage_attn_fwd_noalloc(const void* q_codes, const float* q_scale, const void* k_codes, const float* k_scale,
                          const void* v_in, const float* v_scale, int64_t b, int64_t h, int64_t n, int64_t d,
                          int qk_kind, int pv_kind, int granularity, const uint8_t* tile_mask, int64_t mask_stride_z,
                          int64_t mask_nq, int64_t mask_nkv, const int32_t* doc_ids, void* out, int out_layout,
                          float* lse, hipStream_t stream) {
  if (b <= 0 || h <= 0) return fail(SAGE_ERR_ARG, "b=%lld and h=%lld must be positive", (long long)b, (long long)h);
  int st = check_common(b * h, n, d, qk_kind, pv_kind, granularity);
  if (st) return st;
  const size_t need = sage::attn_workspace_bytes(b, h, n, d, tile_mask != nullptr || doc_ids != nullptr);
  if (need > (size_t)SAGE_NOALLOC_SCRATCH_BYTES)
    return fail(SAGE_ERR_WORKSPACE,
                "b=%lld h=%lld n=%lld d=%lld needs %zu bytes of workspace, beyond the %zu-byte scratch of the "
                "allocation-free entry point; use sage_attn_fwd with a workspace",
                (long long)b, (long long)h, (long long)n, (long long)d, need, (size_t)SAGE_NOALLOC_SCRATCH_BYTES);
  void* ws = nullptr;
  st = scratch_of_stream(stream, &ws);
  if (st) return st;
  return attn_fwd_impl(q_codes, q_scale, k_codes, k_scale, v_in, v_scale, b, h, n, d, qk_kind, pv_kind, granularity,
                       tile_mask, mask_stride_z, mask_nq, mask_nkv, doc_ids, ws, sage::kMaskedSplitBytes, out,
                       out_layout, lse, nullptr, "sage_attn_fwd_noalloc", stream);
}

size_t sage_forward_workspace_bytes(int64_t b, int64_t h, int64_t n, int64_t d, int pv_kind, int with_doc_ids) {
  // shapes sage_forward refuses: no size, and no division by a chunk count of zero
  if (b <= 0 || h <= 0 || n <= 0 || (d != 64 && d != 128)) return 0;
  return forward_workspace(b, h, n, d, pv_kind, with_doc_ids != 0).bytes;
}

int sage_forward(const void* q, const void* k, const void* v, int64_t b, int64_t h, int64_t n, int64_t d, int qk_kind,
                 int pv_kind, int granularity, int smooth_k, float sm_scale_log2e, const uint8_t* tile_mask,
                 int64_t mask_stride_z, int64_t mask_nq, int64_t mask_nkv, const int32_t* doc_ids, void* workspace,
                 size_t workspace_bytes, void* out, int out_layout, float* lse, hipStream_t stream) {
  if (b <= 0 || h <= 0) return fail(SAGE_ERR_ARG, "b=%lld and h=%lld must be positive", (long long)b, (long long)h);
  int st = check_common(b * h, n, d, qk_kind, pv_kind, granularity);
  if (st) return st;
  const ForwardWorkspace w = forward_workspace(b, h, n, d, pv_kind, doc_ids != nullptr);
  if (!workspace || workspace_bytes < w.bytes)
    return fail(SAGE_ERR_WORKSPACE, "workspace of %zu bytes needed, got %zu", w.bytes, workspace_bytes);
  if (!aligned16(workspace)) return fail(SAGE_ERR_ALIGN, "workspace must be 16-byte aligned");
  uint8_t* p = static_cast<uint8_t*>(workspace);
  float* qs = reinterpret_cast<float*>(p + w.qs);
  float* ks = reinterpret_cast<float*>(p + w.ks);
  float* vs = pv_kind == SAGE_PV_FP8 ? reinterpret_cast<float*>(p + w.vs) : nullptr;
  st = sage_quantize_qkv(q, k, v, b * h, n, d, qk_kind, pv_kind, granularity, smooth_k, sm_scale_log2e, p + w.qc, qs,
                         p + w.kc, ks, p + w.vop, vs, p + w.kmean, p + w.quant, w.attn - w.quant, stream);
  if (st) return st;
  return attn_fwd_impl(p + w.qc, qs, p + w.kc, ks, p + w.vop, vs, b, h, n, d, qk_kind, pv_kind, granularity, tile_mask,
                       mask_stride_z, mask_nq, mask_nkv, doc_ids, p + w.attn, w.bytes - w.attn, out, out_layout, lse,
                       nullptr, "sage_forward", stream);
}

int sage_attn_qk_accumulators(const void* q_codes, const float* q_scale, const void* k_codes, const float* k_scale,
                              const void* v_in, const float* v_scale, int64_t b, int64_t h, int64_t n, int64_t d,
                              int qk_kind, int pv_kind, void* workspace, size_t workspace_bytes, void* out, float* lse,
                              int32_t* s_out, hipStream_t stream) {
  if (!s_out) return fail(SAGE_ERR_ARG, "null tensor pointer");
  return attn_fwd_impl(q_codes, q_scale, k_codes, k_scale, v_in, v_scale, b, h, n, d, qk_kind, pv_kind,
                       SAGE_GRAN_TOKEN, nullptr, 0, 0, 0, nullptr, workspace, workspace_bytes, out, SAGE_OUT_BHND,
                       lse, s_out, "sage_attn_qk_accumulators", stream);
}

size_t sage_attn_bwd_workspace_bytes(int64_t b, int64_t h, int64_t n, int64_t d) {
  return bwd_workspace(b, b * h, n, d).bytes;
}

int sage_attn_bwd(const void* q, const void* k, const void* v, const void* out, const float* lse, const void* dout,
                  int64_t b, int64_t h, int64_t n, int64_t d, int qk_kind, int smooth_k, float sm_scale,
                  float sm_scale_log2e, const uint8_t* tile_mask, int64_t mask_stride_z, int64_t mask_nq, int64_t mask_nkv,
                  const int32_t* doc_ids, void* workspace, size_t workspace_bytes, void* dq, void* dk, void* dv,
                  hipStream_t stream) {
  return sage_attn_bwd_layout(q, k, v, out, SAGE_OUT_BHND, lse, dout, SAGE_OUT_BHND, b, h, n, d, qk_kind, smooth_k,
                              sm_scale, sm_scale_log2e, tile_mask, mask_stride_z, mask_nq, mask_nkv, doc_ids,
                              workspace, workspace_bytes, dq, dk, dv, stream);
}

int sage_attn_bwd_layout(const void* q, const void* k, const void* v, const void* out, int out_layout,
                         const float* lse, const void* dout, int dout_layout, int64_t b, int64_t h, int64_t n,
                         int64_t d, int qk_kind, int smooth_k, float sm_scale, float sm_scale_log2e,
                         const uint8_t* tile_mask, int64_t mask_stride_z, int64_t mask_nq, int64_t mask_nkv,
                         const int32_t* doc_ids, void* workspace, size_t workspace_bytes, void* dq, void* dk, void* dv,
                         hipStream_t stream) {
  if (b <= 0 || h <= 0) return fail(SAGE_ERR_ARG, "b=%lld and h=%lld must be positive", (long long)b, (long long)h);
  int st = check_common(b * h, n, d, qk_kind, SAGE_PV_BF16, SAGE_GRAN_TOKEN);
  if (st) return st;
  if (!q || !k || !v || !out || !lse || !dout || !dq || !dk || !dv) return fail(SAGE_ERR_ARG, "null tensor pointer");
  const void* ptrs[] = {q, k, v, out, dout, dq, dk, dv};
  for (const void* p : ptrs)
    if (!aligned16(p)) return fail(SAGE_ERR_ALIGN, "tensor pointers must be 16-byte aligned");
  if (!(sm_scale > 0.0f) || !(sm_scale_log2e > 0.0f))
    return fail(SAGE_ERR_ARG, "sm_scale and sm_scale_log2e must be positive");
  for (const int layout : {out_layout, dout_layout})
    if (layout != SAGE_OUT_BHND && layout != SAGE_OUT_BNHD)
      return fail(SAGE_ERR_ARG, "out and dout layouts must be 0 ([B,H,N,D]) or 1 ([B,N,H,D]), got %d", layout);
  const int64_t nq = (n + 127) / 128, nkv = (n + 63) / 64;
  int mask = 0;
  if (tile_mask) {
    if (mask_nq != nq || mask_nkv != nkv)
      return fail(SAGE_ERR_ARG, "block_mask must be %lld x %lld tiles, got %lld x %lld", (long long)nq,
                  (long long)nkv, (long long)mask_nq, (long long)mask_nkv);
    if (mask_stride_z != 0 && mask_stride_z != nq * nkv)
      return fail(SAGE_ERR_ARG, "mask_stride_z must be 0 (2D mask) or %lld (3D mask)", (long long)(nq * nkv));
    mask |= 1;
  }
  if (doc_ids) mask |= 2;
  // one launch of a dK/dV and a dQ workgroup (256 threads) per 128-row tile; the
  // quantization's limit below leaves room for the rounding and the cut items
  if ((b * h) * ((n + 127) / 128) > kMaxGridUnits / 2)
    return fail(SAGE_ERR_ARG, "b*h*ceil(n/128) = %lld exceeds the grid limit", (long long)(b * h * ((n + 127) / 128)));
  if (sage::quant_grid_units(b * h, n, d, 0) > kMaxGridUnits)
    return fail(SAGE_ERR_ARG, "quantizing b*h=%lld x n=%lld exceeds one launch's %lld workgroups", (long long)(b * h),
                (long long)n, (long long)kMaxGridUnits);
  const BwdWorkspace ws = bwd_workspace(b, b * h, n, d);
  if (!workspace || workspace_bytes < ws.bytes)
    return fail(SAGE_ERR_WORKSPACE, "workspace of %zu bytes needed, got %zu", ws.bytes, workspace_bytes);
  if (!aligned16(workspace)) return fail(SAGE_ERR_ALIGN, "workspace must be 16-byte aligned");
  uint8_t* w = static_cast<uint8_t*>(workspace);
  const int64_t bh = b * h;
  const auto* q16 = static_cast<const uint16_t*>(q);
  const auto* k16 = static_cast<const uint16_t*>(k);
  const auto* do16 = static_cast<const uint16_t*>(dout);
  // codes, scales and the K mean of the forward's per-token quantization, and
  // the backward's own operands, in one launch
  auto strides = [&](int layout, int64_t& bs, int64_t& hs, int64_t& rs) {
    bs = h * n * d;
    hs = layout == SAGE_OUT_BNHD ? d : n * d;
    rs = layout == SAGE_OUT_BNHD ? h * d : d;
  };
  sage::BwdPrep prep{};
  prep.kt = reinterpret_cast<uint16_t*>(w + ws.kt);
  prep.dout = do16;
  strides(dout_layout, prep.dout_bs, prep.dout_hs, prep.dout_rs);
  prep.out = static_cast<const uint16_t*>(out);
  strides(out_layout, prep.out_bs, prep.out_hs, prep.out_rs);
  prep.lse = lse;
  prep.neg_delta = reinterpret_cast<float*>(w + ws.neg_delta);
  prep.lse_pad = reinterpret_cast<float*>(w + ws.lse_pad);
  prep.h = (int)h;
  hipError_t e = sage::launch_quantize_bwd(
      qk_kind, smooth_k != 0, q16, k16, bh, n, d, sm_scale_log2e, reinterpret_cast<double*>(w + ws.quant), w + ws.qc,
      reinterpret_cast<float*>(w + ws.qs), w + ws.kc, reinterpret_cast<float*>(w + ws.ks),
      reinterpret_cast<uint16_t*>(w + ws.kmean), prep, stream);
  if (e != hipSuccess) return launch_status(e, "sage_attn_bwd (quantize)");
  const int4* sums = reinterpret_cast<const int4*>(w + ws.sums);
  const int64_t np = sage::padded_len(n);
  if (doc_ids) {
    e = sage::launch_doc_summaries(doc_ids, n, (int)b, const_cast<int4*>(sums), const_cast<int4*>(sums + b * nkv),
                                   const_cast<int4*>(sums + b * nkv + b * (np / 32)), nullptr, stream);
    if (e != hipSuccess) return launch_status(e, "sage_attn_bwd (summaries)");
  }
  sage::BwdParams p;
  memset(&p, 0, sizeof(p));
  p.qc = w + ws.qc;
  p.qs = reinterpret_cast<const float*>(w + ws.qs);
  p.kc = w + ws.kc;
  p.ks = reinterpret_cast<const float*>(w + ws.ks);
  p.q = q16;
  p.kt = smooth_k ? reinterpret_cast<const uint16_t*>(w + ws.kt) : k16;
  p.v = static_cast<const uint16_t*>(v);
  p.dout = do16;
  p.dout_bs = prep.dout_bs;
  p.dout_hs = prep.dout_hs;
  p.dout_rs = prep.dout_rs;
  p.lse_pad = reinterpret_cast<const float*>(w + ws.lse_pad);
  p.neg_delta = reinterpret_cast<const float*>(w + ws.neg_delta);
  p.tile_mask = tile_mask;
  p.mask_stride_z = mask_stride_z;
  p.mask_nkv = mask_nkv;
  p.doc = doc_ids;
  p.kv_sum = sums;
  p.q_sum = sums + b * nkv;
  p.q_sum128 = sums + b * nkv + b * (np / 32);
  p.dq = static_cast<uint16_t*>(dq);
  p.dk = static_cast<uint16_t*>(dk);
  p.dv = static_cast<uint16_t*>(dv);
  p.n = n;
  p.np = np;
  p.h = (int)h;
  p.sm_scale = sm_scale;
  // the last dQ items (up to kBwdDqSplit, a multiple of 8) in two key halves:
  // the backward at 1x30x4416x128 919 -> 880 us, 1x30x1280 115.7 -> 110.0,
  // 2x4x333x64 18.0 either way; 1x30x3071, whose last round is fuller, 442 -> 449
  const int64_t items = bh * (np / 128);
  p.dq_split = nkv >= 2 && bwd_split_enabled() ? (int)std::min<int64_t>(sage::kBwdDqSplit, items / 8 * 8) : 0;
  p.dq_part = reinterpret_cast<float*>(w + ws.dq_part);
  p.dq_ctr = reinterpret_cast<uint64_t*>(w + ws.dq_ctr);
  p.dq_tag = next_merge_tag();
  return launch_status(sage::launch_bwd(qk_kind, mask, p, d, bh, stream), "sage_attn_bwd");
}

int sage_build_tile_mask(const int32_t* doc_ids, int64_t b, int64_t n, int32_t pad_fill, uint8_t* mask,
                         hipStream_t stream) {
  if (b <= 0 || n <= 0) return fail(SAGE_ERR_ARG, "b=%lld and n=%lld must be positive", (long long)b, (long long)n);
  if (b > 65535) return fail(SAGE_ERR_ARG, "b=%lld exceeds the grid limit 65535", (long long)b);
  if (n > (int64_t)1 << 24) return fail(SAGE_ERR_ARG, "n=%lld exceeds 2^24", (long long)n);
  if (!doc_ids || !mask) return fail(SAGE_ERR_ARG, "null tensor pointer");
  return launch_status(sage::launch_tile_mask(doc_ids, b, n, pad_fill, mask, stream), "sage_build_tile_mask");
}

int sage_doc_ids_from_cu_seqlens(const int32_t* cu_seqlens, int64_t b, int64_t n_segments, int64_t n,
                                 int32_t* doc_ids, hipStream_t stream) {
  if (b <= 0 || n <= 0) return fail(SAGE_ERR_ARG, "b=%lld and n=%lld must be positive", (long long)b, (long long)n);
  if (n_segments < 0) return fail(SAGE_ERR_ARG, "n_segments=%lld must not be negative", (long long)n_segments);
  if (b > 65535) return fail(SAGE_ERR_ARG, "b=%lld exceeds the grid limit 65535", (long long)b);
  if (n > (int64_t)1 << 24) return fail(SAGE_ERR_ARG, "n=%lld exceeds 2^24", (long long)n);
  if (!cu_seqlens || !doc_ids) return fail(SAGE_ERR_ARG, "null tensor pointer");
  return launch_status(sage::launch_doc_from_cu(cu_seqlens, b, n_segments, n, doc_ids, stream),
                       "sage_doc_ids_from_cu_seqlens");
}

}  // extern "C"

namespace {

int check_norm(const sage::NormArgs& a, int64_t b, int64_t n, int64_t c, int64_t groups, int dtype, int fp32_params) {
  if (b <= 0 || n <= 0 || c <= 0)
    return fail(SAGE_ERR_ARG, "b=%lld, n=%lld and c=%lld must be positive", (long long)b, (long long)n, (long long)c);
  if (c > sage::kNormMaxC) return fail(SAGE_ERR_ARG, "c=%lld exceeds %lld", (long long)c, (long long)sage::kNormMaxC);
  if (b > 65535 || n >= (int64_t)1 << 23 || b * n >= (int64_t)1 << 23)
    return fail(SAGE_ERR_ARG, "b=%lld x n=%lld exceeds the grid limit 2^23", (long long)b, (long long)n);
  if (groups <= 0 || groups > 32767 || b * groups > 32767)
    return fail(SAGE_ERR_ARG, "b=%lld x groups=%lld must be between 1 and 32767", (long long)b, (long long)groups);
  if (!a.doc && groups != 1) return fail(SAGE_ERR_ARG, "groups=%lld needs doc_ids", (long long)groups);
  if (dtype != SAGE_DTYPE_BF16 && dtype != SAGE_DTYPE_FP16) return fail(SAGE_ERR_ARG, "unknown dtype %d", dtype);
  if (fp32_params < 0 || fp32_params > 15) return fail(SAGE_ERR_ARG, "unknown fp32_params %d", fp32_params);
  if (!(a.eps >= 0.0f)) return fail(SAGE_ERR_ARG, "eps must be >= 0");
  return SAGE_OK;
}

sage::NormArgs norm_args(const void* x, int64_t x_bs, int64_t x_rs, const void* w, const void* cond, int64_t cond_bs,
                         int64_t cond_gs, int64_t groups, const int32_t* doc, int64_t b, int64_t n, int64_t c,
                         int fp32_params, float eps) {
  sage::NormArgs a{};
  a.x = {x, x_bs, x_rs};
  a.w = {w, fp32_params & SAGE_FP32_WEIGHT ? 1 : 0};
  a.cond = {cond, fp32_params & SAGE_FP32_COND ? 1 : 0, (int)groups, cond_bs, cond_gs};
  a.doc = doc;
  a.groups = (int)groups;
  a.b = (int)b;
  a.n = n;
  a.c = (int)c;
  a.eps = eps;
  return a;
}

// Element alignment of a call's pointers: 2 bytes, fp32 parameters 4.
int check_norm_align(const sage::NormArgs& a) {
  const void* two[] = {a.x.p, a.res.p, a.dout.p, a.dhidden.p, a.out, a.hidden, a.dx, a.dres};
  for (const void* p : two)
    if (reinterpret_cast<uintptr_t>(p) & 1u) return fail(SAGE_ERR_ALIGN, "tensor pointers must be aligned to their elements");
  const struct { const void* p; int f32; } params[] = {
      {a.w.p, a.w.f32},   {a.w2.p, a.w2.f32}, {a.cond.p, a.cond.f32},   {a.cond2.p, a.cond2.f32},
      {a.dw, a.w.f32},    {a.dw2, a.w2.f32},  {a.dcond, a.cond.f32},    {a.dcond2, a.cond2.f32}};
  for (const auto& q : params)
    if (reinterpret_cast<uintptr_t>(q.p) & (q.f32 ? 3u : 1u))
      return fail(SAGE_ERR_ALIGN, "parameter pointers must be aligned to their elements");
  return SAGE_OK;
}

size_t norm_workspace(int64_t b, const sage::NormChunks& k, int sets, size_t* id_off) {
  const size_t part = (size_t)(b * k.chunks * k.slots * sets * k.cp) * sizeof(float);
  *id_off = part;
  return part + (size_t)(b * k.chunks * k.slots) * sizeof(int32_t);
}

// The backward's chunks and workspace, and its launch.
int run_norm_bwd(int op, sage::NormArgs& a, int dtype, void* workspace, size_t workspace_bytes, hipStream_t stream,
                 const char* what) {
  const sage::NormChunks k = sage::norm_chunks(a.b, a.n, a.c, a.groups, a.doc != nullptr);
  a.chunks = (int)k.chunks;
  a.chunk = k.chunk;
  a.slots = (int)k.slots;
  a.cp = k.cp;
  if (a.dw || a.dw2 || a.dcond || a.dcond2) {
    size_t id_off;
    const size_t need = norm_workspace(a.b, k, op == sage::kNormGateModulate ? 2 : 1, &id_off);
    if (!workspace || workspace_bytes < need)
      return fail(SAGE_ERR_WORKSPACE, "workspace of %zu bytes needed, got %zu", need, workspace_bytes);
    if (!aligned16(workspace)) return fail(SAGE_ERR_ALIGN, "workspace must be 16-byte aligned");
    a.part = static_cast<float*>(workspace);
    a.part_id = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(workspace) + id_off);
  }
  return launch_status(sage::launch_norm_bwd(op, dtype, a, stream), what);
}

}  // namespace

extern "C" {

int sage_rms_norm_modulate(const void* x, int64_t x_bs, int64_t x_rs, const void* weight, const void* scale,
                           int64_t scale_bs, int64_t scale_gs, int64_t groups, const int32_t* doc_ids, int64_t b,
                           int64_t n, int64_t c, int dtype, int fp32_params, float eps, void* out,
                           hipStream_t stream) {
  sage::NormArgs a = norm_args(x, x_bs, x_rs, weight, scale, scale_bs, scale_gs, groups, doc_ids, b, n, c,
                               fp32_params, eps);
  if (const int e = check_norm(a, b, n, c, groups, dtype, fp32_params)) return e;
  if (!x || !out) return fail(SAGE_ERR_ARG, "null tensor pointer");
  a.out = out;
  if (const int e = check_norm_align(a)) return e;
  return launch_status(sage::launch_norm_fwd(sage::kNormModulate, dtype, a, stream), "sage_rms_norm_modulate");
}

int sage_rms_norm_gate_residual(const void* residual, int64_t r_bs, int64_t r_rs, const void* x, int64_t x_bs,
                                int64_t x_rs, const void* weight, const void* gate, int64_t gate_bs, int64_t gate_gs,
                                int64_t groups, const int32_t* doc_ids, int64_t b, int64_t n, int64_t c, int dtype,
                                int fp32_params, float eps, void* out, hipStream_t stream) {
  sage::NormArgs a = norm_args(x, x_bs, x_rs, weight, gate, gate_bs, gate_gs, groups, doc_ids, b, n, c, fp32_params,
                               eps);
  if (const int e = check_norm(a, b, n, c, groups, dtype, fp32_params)) return e;
  if (!residual || !x || !out) return fail(SAGE_ERR_ARG, "null tensor pointer");
  a.res = {residual, r_bs, r_rs};
  a.out = out;
  if (const int e = check_norm_align(a)) return e;
  return launch_status(sage::launch_norm_fwd(sage::kNormGate, dtype, a, stream), "sage_rms_norm_gate_residual");
}

int sage_rms_norm_gate_residual_modulate(const void* residual, int64_t r_bs, int64_t r_rs, const void* x,
                                         int64_t x_bs, int64_t x_rs, const void* weight, const void* gate,
                                         int64_t gate_bs, int64_t gate_gs, const void* next_weight,
                                         const void* next_scale, int64_t scale_bs, int64_t scale_gs, int64_t groups,
                                         const int32_t* doc_ids, int64_t b, int64_t n, int64_t c, int dtype,
                                         int fp32_params, float eps, void* hidden, void* out, hipStream_t stream) {
  sage::NormArgs a = norm_args(x, x_bs, x_rs, weight, gate, gate_bs, gate_gs, groups, doc_ids, b, n, c, fp32_params,
                               eps);
  if (const int e = check_norm(a, b, n, c, groups, dtype, fp32_params)) return e;
  if (!residual || !x || !hidden || !out) return fail(SAGE_ERR_ARG, "null tensor pointer");
  a.res = {residual, r_bs, r_rs};
  a.w2 = {next_weight, fp32_params & SAGE_FP32_NEXT_WEIGHT ? 1 : 0};
  a.cond2 = {next_scale, fp32_params & SAGE_FP32_NEXT_SCALE ? 1 : 0, (int)groups, scale_bs, scale_gs};
  a.hidden = hidden;
  a.out = out;
  if (const int e = check_norm_align(a)) return e;
  return launch_status(sage::launch_norm_fwd(sage::kNormGateModulate, dtype, a, stream),
                       "sage_rms_norm_gate_residual_modulate");
}

size_t sage_rms_norm_bwd_workspace_bytes(int64_t b, int64_t n, int64_t c, int64_t groups, int with_doc_ids,
                                         int fused) {
  if (b <= 0 || n <= 0 || c <= 0 || groups <= 0 || b > 65535 || groups > 32767 || b * groups > 32767 ||
      c > sage::kNormMaxC || n >= (int64_t)1 << 23 || b * n >= (int64_t)1 << 23)
    return 0;
  size_t id_off;
  return norm_workspace(b, sage::norm_chunks(b, n, c, groups, with_doc_ids != 0), fused ? 2 : 1, &id_off);
}

int sage_rms_norm_modulate_bwd(const void* dout, int64_t d_bs, int64_t d_rs, const void* x, int64_t x_bs,
                               int64_t x_rs, const void* weight, const void* scale, int64_t scale_bs,
                               int64_t scale_gs, int64_t groups, const int32_t* doc_ids, int64_t b, int64_t n,
                               int64_t c, int dtype, int fp32_params, float eps, void* workspace,
                               size_t workspace_bytes, void* dx, void* dweight, void* dscale, hipStream_t stream) {
  sage::NormArgs a = norm_args(x, x_bs, x_rs, weight, scale, scale_bs, scale_gs, groups, doc_ids, b, n, c,
                               fp32_params, eps);
  if (const int e = check_norm(a, b, n, c, groups, dtype, fp32_params)) return e;
  if (!dout || !x) return fail(SAGE_ERR_ARG, "null tensor pointer");
  a.dout = {dout, d_bs, d_rs};
  a.dx = dx;
  a.dw = dweight;
  a.dcond = dscale;
  if (const int e = check_norm_align(a)) return e;
  return run_norm_bwd(sage::kNormModulate, a, dtype, workspace, workspace_bytes, stream, "sage_rms_norm_modulate_bwd");
}

int sage_rms_norm_gate_residual_bwd(const void* dout, int64_t d_bs, int64_t d_rs, const void* x, int64_t x_bs,
                                    int64_t x_rs, const void* weight, const void* gate, int64_t gate_bs,
                                    int64_t gate_gs, int64_t groups, const int32_t* doc_ids, int64_t b, int64_t n,
                                    int64_t c, int dtype, int fp32_params, float eps, void* workspace,
                                    size_t workspace_bytes, void* dx, void* dweight, void* dgate,
                                    hipStream_t stream) {
  sage::NormArgs a = norm_args(x, x_bs, x_rs, weight, gate, gate_bs, gate_gs, groups, doc_ids, b, n, c, fp32_params,
                               eps);
  if (const int e = check_norm(a, b, n, c, groups, dtype, fp32_params)) return e;
  if (!dout || !x) return fail(SAGE_ERR_ARG, "null tensor pointer");
  a.dout = {dout, d_bs, d_rs};
  a.dx = dx;
  a.dw = dweight;
  a.dcond = dgate;
  if (const int e = check_norm_align(a)) return e;
  return run_norm_bwd(sage::kNormGate, a, dtype, workspace, workspace_bytes, stream,
                      "sage_rms_norm_gate_residual_bwd");
}

int sage_rms_norm_gate_residual_modulate_bwd(
    const void* dhidden, int64_t dh_bs, int64_t dh_rs, const void* dout, int64_t d_bs, int64_t d_rs,
    const void* residual, int64_t r_bs, int64_t r_rs, const void* x, int64_t x_bs, int64_t x_rs, const void* weight,
    const void* gate, int64_t gate_bs, int64_t gate_gs, const void* next_weight, const void* next_scale,
    int64_t scale_bs, int64_t scale_gs, int64_t groups, const int32_t* doc_ids, int64_t b, int64_t n, int64_t c,
    int dtype, int fp32_params, float eps, void* workspace, size_t workspace_bytes, void* dresidual, void* dx,
    void* dweight, void* dgate, void* dnext_weight, void* dnext_scale, hipStream_t stream) {
  sage::NormArgs a = norm_args(x, x_bs, x_rs, weight, gate, gate_bs, gate_gs, groups, doc_ids, b, n, c, fp32_params,
                               eps);
  if (const int e = check_norm(a, b, n, c, groups, dtype, fp32_params)) return e;
  if (!dhidden || !dout || !residual || !x || !dresidual) return fail(SAGE_ERR_ARG, "null tensor pointer");
  a.dhidden = {dhidden, dh_bs, dh_rs};
  a.dout = {dout, d_bs, d_rs};
  a.res = {residual, r_bs, r_rs};
  a.w2 = {next_weight, fp32_params & SAGE_FP32_NEXT_WEIGHT ? 1 : 0};
  a.cond2 = {next_scale, fp32_params & SAGE_FP32_NEXT_SCALE ? 1 : 0, (int)groups, scale_bs, scale_gs};
  a.dres = dresidual;
  a.dx = dx;
  a.dw = dweight;
  a.dcond = dgate;
  a.dw2 = dnext_weight;
  a.dcond2 = dnext_scale;
  if (const int e = check_norm_align(a)) return e;
  return run_norm_bwd(sage::kNormGateModulate, a, dtype, workspace, workspace_bytes, stream,
                      "sage_rms_norm_gate_residual_modulate_bwd");
}

}  // extern "C"

namespace {

int64_t up8(int64_t x) { return (x + 7) / 8 * 8; }
size_t up256(size_t x) { return (x + 255) / 256 * 256; }

int check_linear(int64_t m, int64_t n, int64_t k, int64_t w_rs, int dtype, int activation) {
  if (m <= 0 || n <= 0 || k <= 0)
    return fail(SAGE_ERR_ARG, "m=%lld, n=%lld and k=%lld must be positive", (long long)m, (long long)n, (long long)k);
  if (activation < SAGE_ACT_NONE || activation > SAGE_ACT_SWIGLU)
    return fail(SAGE_ERR_ARG, "unknown activation %d", activation);
  if (dtype != SAGE_DTYPE_BF16 && dtype != SAGE_DTYPE_FP16) return fail(SAGE_ERR_ARG, "unknown dtype %d", dtype);
  const int64_t rows = activation == SAGE_ACT_SWIGLU ? 2 * n : n;
  if (m >= (int64_t)1 << 24 || n >= (int64_t)1 << 22 || k >= (int64_t)1 << 22)
    return fail(SAGE_ERR_ARG, "m=%lld, n=%lld or k=%lld exceeds 2^24, 2^22, 2^22", (long long)m, (long long)n,
                (long long)k);
  if (rows >= (int64_t)1 << 22)
    return fail(SAGE_ERR_ARG, "a weight of %lld rows, 2^22 or more", (long long)rows);
  if (rows * up8(k) * 2 >= (int64_t)1 << 31 || (rows - 1) * w_rs * 2 + k * 2 >= (int64_t)1 << 31)
    return fail(SAGE_ERR_ARG, "a weight of %lld x %lld has 2^31 bytes or more", (long long)rows, (long long)k);
  return SAGE_OK;
}

// Row strides: at least the columns, and panels of 256 rows under 2^31 bytes (one row: any).
int check_rows(int64_t rs, int64_t rows, int64_t cols, const char* what) {
  if (rows == 1) return SAGE_OK;
  if (rs < cols) return fail(SAGE_ERR_ARG, "%s rows are %lld apart, under %lld", what, (long long)rs, (long long)cols);
  if (rs >= (int64_t)1 << 22) return fail(SAGE_ERR_ARG, "%s rows are %lld apart, 2^22 or more", what, (long long)rs);
  return SAGE_OK;
}

// Rows a product can read in place: from 16-byte boundaries, `cols` a multiple of 8 where the
// contraction runs along them.
bool in_place(const void* p, int64_t rs, int64_t rows, int64_t cols) {
  return aligned16(p) && (rows == 1 || rs % 8 == 0) && cols % 8 == 0;
}

// An operand in place, or its copy in the workspace (packed on run).
struct LinearOperand {
  const void* src;
  int64_t rs, rows, cols, pc;
  bool copy;
  size_t off;
  LinearOperand(const void* p, int64_t rs_, int64_t rows_, int64_t cols_, size_t& at)
      : src(p), rs(rs_), rows(rows_), cols(cols_), pc(up8(cols_)), copy(!in_place(p, rs_, rows_, cols_)), off(at) {
    if (copy) at += up256((size_t)(rows * pc) * 2);
  }
  const void* ptr(void* ws) const { return copy ? static_cast<uint8_t*>(ws) + off : src; }
  int64_t ld() const { return copy ? pc : rows == 1 ? up8(cols) : rs; }
  sage::PackArgs pack(void* ws) const {
    return {copy ? src : nullptr, rs, rows, cols, static_cast<uint8_t*>(ws) + off, pc};
  }
};

sage::GemmArgs forward_gemm(int64_t m, int64_t n, int64_t k, int act, bool vec) {
  sage::GemmArgs g{};
  g.vec = vec;
  g.m = m;
  g.n = (int)n;
  g.k = up8(k);
  g.kv = k;
  g.a_kc = g.b_kc = 1;
  g.act = act;
  sage::gemm_plan(g);
  return g;
}

// The backward's steps and their places in its workspace.
struct LinearBwd {
  int64_t rows;
  bool form_dz;     // dz is formed (an activation, or rows that no product can read in place)
  bool dz_in_place; // dout itself is the products' operand
  int64_t ldz;
  int64_t plane;    // elements between dz's two parts; 0: it has one
  size_t dz_off, sum_off, part_off, bytes;
  int64_t chunks, chunk;
  sage::GemmArgs gx{}, gw{};
  // x and weight as rows whose columns the products read 16 bytes at a time
  size_t x_off, w_off;
  bool copy_x, copy_w;
  // form_w: the weight's rows are formed in the workspace, whatever w is, and the dz of an
  // activation is two bf16 matrices
  LinearBwd(const void* dout, int64_t d_rs, const void* x, int64_t x_rs, const void* w, int64_t w_rs, int64_t m,
            int64_t n, int64_t k, int act, int want, bool form_w = false) {
    rows = act == SAGE_ACT_SWIGLU ? 2 * n : n;
    const bool products = want & 3;
    form_dz = products && (act != SAGE_ACT_NONE || !in_place(dout, d_rs, m, n));
    dz_in_place = products && !form_dz;
    ldz = form_dz ? up8(rows) : m == 1 ? up8(rows) : d_rs;
    size_t at = 0;
    dz_off = at;
    plane = form_w && form_dz && act != SAGE_ACT_NONE ? (int64_t)(up256((size_t)(m * ldz) * 2) / 2) : 0;
    if (form_dz) at += up256((size_t)(m * ldz) * 2) * (plane ? 2 : 1);
    // bias: chunks of at least 32 rows, at most 256 of them
    chunk = (m + 255) / 256 < 32 ? 32 : (m + 255) / 256;
    chunks = (m + chunk - 1) / chunk;
    sum_off = at;
    if (want & 4) at += up256((size_t)(chunks * rows) * 4);
    copy_x = (want & 2) && !in_place(x, x_rs, m, k);
    copy_w = (want & 1) && (form_w || !in_place(w, w_rs, rows, k));
    x_off = at;
    if (copy_x) at += up256((size_t)(m * up8(k)) * 2);
    w_off = at;
    if (copy_w) at += up256((size_t)(rows * up8(k)) * 2);
    size_t part = 0;
    if (want & 1) {
      gx.m = m;
      gx.n = (int)k;
      gx.k = up8(rows);
      gx.kv = rows;
      gx.a_kc = 1;
      gx.lda = ldz;
      gx.ldb = copy_w ? up8(k) : rows == 1 ? up8(k) : w_rs;
      gx.vec = k % 8 == 0;  // dx and dweight start on 16-byte boundaries
      gx.half = plane ? (rows + 63) / 64 * 64 : 0;
      gx.plane = plane;
      sage::gemm_plan(gx);
      part = (size_t)gx.part_floats * 4;
    }
    if (want & 2) {
      gw.m = rows;
      gw.n = (int)k;
      gw.k = gw.kv = m;
      gw.lda = ldz;
      gw.ldb = copy_x ? up8(k) : m == 1 ? up8(k) : x_rs;
      gw.vec = k % 8 == 0;
      sage::gemm_plan(gw);
      part = std::max(part, (size_t)gw.part_floats * 4);
    }
    part_off = at;
    bytes = at + up256(part);
  }
};

// The backward's launches.  w_codes (with w_scales): the weight is MXFP4, and its rows are formed
// in the workspace; else `weight` is read or copied.
int run_linear_bwd(const LinearBwd& plan, const void* dout, int64_t d_rs, const void* x, int64_t x_rs,
                   const void* weight, int64_t w_rs, const uint8_t* w_codes, const uint8_t* w_scales, const float* z,
                   int64_t m, int64_t n, int64_t k, int dtype, int activation, int bias_fp32, void* workspace,
                   size_t workspace_bytes, void* dx, void* dweight, void* dbias, hipStream_t stream) {
  LinearBwd p = plan;
  if (p.bytes && (!workspace || workspace_bytes < p.bytes))
    return fail(SAGE_ERR_WORKSPACE, "workspace of %zu bytes needed, got %zu", p.bytes, workspace_bytes);
  if (p.bytes && !aligned16(workspace)) return fail(SAGE_ERR_ALIGN, "workspace must be 16-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (p.form_dz || dbias) {
    sage::DactArgs d{};
    d.dout = dout;
    d.z = z;
    d.ldd = m == 1 ? n : d_rs;
    d.m = m;
    d.n = (int)n;
    d.act = activation;
    d.dz = p.form_dz ? ws + p.dz_off : nullptr;
    d.ldz = p.ldz;
    d.plane = d.dz ? p.plane : 0;
    d.vec = in_place(dout, d_rs, m, n) && aligned16(z);
    d.part = dbias ? reinterpret_cast<float*>(ws + p.sum_off) : nullptr;
    d.chunks = p.chunks;
    d.chunk = p.chunk;
    d.dbias = dbias;
    d.bias_f32 = bias_fp32 != 0;
    const hipError_t e = sage::launch_dact(dtype, d, stream);
    if (e != hipSuccess) return launch_status(e, "sage_linear_bwd (activation)");
  }
  const void* dz = p.form_dz ? ws + p.dz_off : dout;
  if (dx && w_codes) {
    const sage::MxDequantArgs q{w_codes, w_scales,      p.rows, (int)up8(k), (int)sage::mx_cols(k),
                                ws + p.w_off, up8(k), 1};
    const hipError_t e = sage::launch_mx_dequantize(q, p.plane ? SAGE_DTYPE_BF16 : dtype, stream);
    if (e != hipSuccess) return launch_status(e, "sage_mxfp4_linear_bwd (weight)");
  } else if (p.copy_x || p.copy_w) {
    const hipError_t e = sage::launch_pack({p.copy_x ? x : nullptr, x_rs, m, k, ws + p.x_off, up8(k)},
                                           {p.copy_w ? weight : nullptr, w_rs, p.rows, k, ws + p.w_off, up8(k)}, stream);
    if (e != hipSuccess) return launch_status(e, "sage_linear_bwd (copy)");
  }
  if (dx) {
    p.gx.a = dz;
    p.gx.b = p.copy_w ? ws + p.w_off : weight;
    p.gx.out = dx;
    p.gx.part = reinterpret_cast<float*>(ws + p.part_off);
    const hipError_t e = sage::launch_gemm(p.gx, dtype, stream);
    if (e != hipSuccess) return launch_status(e, "sage_linear_bwd (dx)");
  }
  if (dweight) {
    p.gw.a = dz;
    p.gw.b = p.copy_x ? ws + p.x_off : x;
    p.gw.out = dweight;
    p.gw.part = reinterpret_cast<float*>(ws + p.part_off);
    const hipError_t e = sage::launch_gemm(p.gw, dtype, stream);
    if (e != hipSuccess) return launch_status(e, "sage_linear_bwd (dweight)");
  }
  return launch_status(hipSuccess, "sage_linear_bwd");
}

}  // namespace

extern "C" {

size_t sage_linear_workspace_bytes(const void* x, int64_t x_rs, const void* weight, int64_t w_rs, int64_t m,
                                   int64_t n, int64_t k, int activation, int other_rows) {
  if (m <= 0 || n <= 0 || k <= 0 || m >= (int64_t)1 << 24 || n >= (int64_t)1 << 22 || k >= (int64_t)1 << 22) return 0;
  size_t at = 0;
  const LinearOperand xo(x, x_rs, m, k, at);
  const LinearOperand wo(weight, w_rs, activation == SAGE_ACT_SWIGLU ? 2 * n : n, k, at);
  // outputs, residual and bias on 16-byte boundaries or not: room for either
  return at + (size_t)std::max(forward_gemm(m, n, k, activation, n % 8 == 0).part_floats,
                               other_rows ? forward_gemm(m, n, k, activation, false).part_floats : 0) * 4;
}

int sage_linear(const void* x, int64_t x_rs, const void* weight, int64_t w_rs, const void* bias, int bias_fp32,
                const void* residual, int64_t r_rs, int64_t m, int64_t n, int64_t k, int dtype, int activation,
                void* workspace, size_t workspace_bytes, float* z, void* out, hipStream_t stream) {
  if (const int e = check_linear(m, n, k, w_rs, dtype, activation)) return e;
  const int64_t rows = activation == SAGE_ACT_SWIGLU ? 2 * n : n;
  if (!x || !weight || !out) return fail(SAGE_ERR_ARG, "null tensor pointer");
  if (const int e = check_rows(x_rs, m, k, "x")) return e;
  if (const int e = check_rows(w_rs, rows, k, "weight")) return e;
  if (residual)
    if (const int e = check_rows(r_rs, m, n, "residual")) return e;
  for (const void* p : {x, weight, residual, (const void*)out})
    if (reinterpret_cast<uintptr_t>(p) & 1u) return fail(SAGE_ERR_ALIGN, "tensor pointers must be aligned to their elements");
  if (reinterpret_cast<uintptr_t>(z) & 3u || reinterpret_cast<uintptr_t>(bias) & (bias_fp32 ? 3u : 1u))
    return fail(SAGE_ERR_ALIGN, "bias must be aligned to its elements, z to 4 bytes");
  size_t at = 0;
  const LinearOperand xo(x, x_rs, m, k, at);
  const LinearOperand wo(weight, w_rs, rows, k, at);
  const bool vec = n % 8 == 0 && aligned16(out) && aligned16(z) && aligned16(bias) && aligned16(residual) &&
                   (!residual || m == 1 || r_rs % 8 == 0);
  sage::GemmArgs g = forward_gemm(m, n, k, activation, vec);
  const size_t need = at + (size_t)g.part_floats * 4;
  if (need && (!workspace || workspace_bytes < need))
    return fail(SAGE_ERR_WORKSPACE, "workspace of %zu bytes needed, got %zu", need, workspace_bytes);
  if (need && !aligned16(workspace)) return fail(SAGE_ERR_ALIGN, "workspace must be 16-byte aligned");
  const hipError_t e = sage::launch_pack(xo.pack(workspace), wo.pack(workspace), stream);
  if (e != hipSuccess) return launch_status(e, "sage_linear (copy)");
  g.a = xo.ptr(workspace);
  g.lda = xo.ld();
  g.b = wo.ptr(workspace);
  g.ldb = wo.ld();
  g.bias = bias;
  g.bias_f32 = bias_fp32 != 0;
  g.res = residual;
  g.ldr = m == 1 ? n : r_rs;
  g.z = z;
  g.out = out;
  g.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + at);
  return launch_status(sage::launch_gemm(g, dtype, stream), "sage_linear");
}

size_t sage_linear_bwd_workspace_bytes(const void* dout, int64_t d_rs, const void* x, int64_t x_rs,
                                       const void* weight, int64_t w_rs, int64_t m, int64_t n, int64_t k,
                                       int activation, int want) {
  if (m <= 0 || n <= 0 || k <= 0 || m >= (int64_t)1 << 24 || n >= (int64_t)1 << 22 || k >= (int64_t)1 << 22) return 0;
  return LinearBwd(dout, d_rs, x, x_rs, weight, w_rs, m, n, k, activation, want).bytes;
}

int sage_linear_bwd(const void* dout, int64_t d_rs, const void* x, int64_t x_rs, const void* weight, int64_t w_rs,
                    const float* z, int64_t m, int64_t n, int64_t k, int dtype, int activation, int bias_fp32,
                    void* workspace, size_t workspace_bytes, void* dx, void* dweight, void* dbias,
                    hipStream_t stream) {
  if (const int e = check_linear(m, n, k, dx ? w_rs : 0, dtype, activation)) return e;
  const int64_t rows = activation == SAGE_ACT_SWIGLU ? 2 * n : n;
  const int want = (dx ? 1 : 0) | (dweight ? 2 : 0) | (dbias ? 4 : 0);
  if (!dout || (dweight && !x) || (dx && !weight) || (activation != SAGE_ACT_NONE && !z))
    return fail(SAGE_ERR_ARG, "null tensor pointer");
  if (!want) return SAGE_OK;
  if (const int e = check_rows(d_rs, m, n, "dout")) return e;
  if (dweight)
    if (const int e = check_rows(x_rs, m, k, "x")) return e;
  if (dx)
    if (const int e = check_rows(w_rs, rows, k, "weight")) return e;
  if (reinterpret_cast<uintptr_t>(z) & 3u) return fail(SAGE_ERR_ALIGN, "z must be aligned to 4 bytes");
  for (const void* p : {dout, x, weight, (const void*)dx, (const void*)dweight})
    if (reinterpret_cast<uintptr_t>(p) & 1u) return fail(SAGE_ERR_ALIGN, "tensor pointers must be aligned to their elements");
  if (reinterpret_cast<uintptr_t>(dbias) & (bias_fp32 ? 3u : 1u))
    return fail(SAGE_ERR_ALIGN, "dbias must be aligned to its elements");
  if (!aligned16(dx) || !aligned16(dweight)) return fail(SAGE_ERR_ALIGN, "dx and dweight must be 16-byte aligned");
  const LinearBwd p(dout, d_rs, x, x_rs, weight, w_rs, m, n, k, activation, want);
  return run_linear_bwd(p, dout, d_rs, x, x_rs, weight, w_rs, nullptr, nullptr, z, m, n, k, dtype, activation, bias_fp32,
                        workspace, workspace_bytes, dx, dweight, dbias, stream);
}

}  // extern "C"

namespace {

// ---- MXFP4

int check_mx_rows(int64_t m, int64_t k, int dtype, const void* codes, const void* scales) {
  if (m <= 0 || k <= 0) return fail(SAGE_ERR_ARG, "m=%lld and k=%lld must be positive", (long long)m, (long long)k);
  if (m >= (int64_t)1 << 24 || k >= (int64_t)1 << 22)
    return fail(SAGE_ERR_ARG, "m=%lld or k=%lld exceeds 2^24, 2^22", (long long)m, (long long)k);
  if (dtype != SAGE_DTYPE_BF16 && dtype != SAGE_DTYPE_FP16) return fail(SAGE_ERR_ARG, "unknown dtype %d", dtype);
  if (!codes || !scales) return fail(SAGE_ERR_ARG, "null tensor pointer");
  if (!aligned16(codes) || reinterpret_cast<uintptr_t>(scales) & 7u)
    return fail(SAGE_ERR_ALIGN, "codes must be 16-byte and scales 8-byte aligned");
  return SAGE_OK;
}

int check_mx_linear(int64_t m, int64_t n, int64_t k, int dtype, int activation) {
  if (m <= 0 || n <= 0 || k <= 0)
    return fail(SAGE_ERR_ARG, "m=%lld, n=%lld and k=%lld must be positive", (long long)m, (long long)n, (long long)k);
  if (activation < SAGE_ACT_NONE || activation > SAGE_ACT_SWIGLU)
    return fail(SAGE_ERR_ARG, "unknown activation %d", activation);
  if (dtype != SAGE_DTYPE_BF16 && dtype != SAGE_DTYPE_FP16) return fail(SAGE_ERR_ARG, "unknown dtype %d", dtype);
  if (m >= (int64_t)1 << 24 || n >= (int64_t)1 << 22 || k >= (int64_t)1 << 22)
    return fail(SAGE_ERR_ARG, "m=%lld, n=%lld or k=%lld exceeds 2^24, 2^22, 2^22", (long long)m, (long long)n,
                (long long)k);
  const int64_t rows = activation == SAGE_ACT_SWIGLU ? 2 * n : n;
  if (rows >= (int64_t)1 << 22)
    return fail(SAGE_ERR_ARG, "a weight of %lld rows, 2^22 or more", (long long)rows);
  if (rows * (sage::mx_cols(k) / 2) >= (int64_t)1 << 31)
    return fail(SAGE_ERR_ARG, "a weight of %lld x %lld has 2^31 bytes of codes or more", (long long)rows, (long long)k);
  return SAGE_OK;
}

// What a product's x is: codes, 16-bit rows, or such rows on 16-byte boundaries and near enough for 32-bit
// offsets, which it quantizes itself where they are few and short.
enum { kMxCodes = 0, kMxRows = 1, kMxNearRows = 2 };
int mx_rows(const void* x, int64_t rs, int64_t m, int64_t k) {
  return !x ? kMxCodes
         : in_place(x, rs, m, k) && (m == 1 || (rs >= 0 && rs < (int64_t)1 << 22)) ? kMxNearRows : kMxRows;
}

// Codes and scales of x in the workspace, and what follows them.
struct MxLinear {
  size_t scales, part;
  bool quantizes;  // the product itself
  sage::GemmArgs g{};
  MxLinear(int64_t m, int64_t n, int64_t k, int act, int x, bool vec) {
    const int64_t kp = sage::mx_cols(k);
    g.vec = vec;
    g.m = m;
    g.n = (int)n;
    g.k = g.kv = g.lda = g.ldb = kp / 4;
    g.a_kc = g.b_kc = 1;
    g.act = act;
    sage::mx_gemm_plan(g);
    quantizes = x == kMxNearRows && g.skinny && m <= sage::kMxQuantRows && k <= sage::kMxQuantCols;
    const bool quantize = x != kMxCodes && !quantizes;
    scales = quantize ? up256((size_t)m * (kp / 2)) : 0;
    part = quantize ? scales + up256((size_t)m * (kp / 32)) : 0;
  }
  size_t bytes() const { return part + (size_t)g.part_floats * 4; }
};

}  // namespace

extern "C" {

int sage_mxfp4_quantize(const void* x, int64_t x_rs, int64_t m, int64_t k, int dtype, void* codes, void* scales,
                        hipStream_t stream) {
  if (const int e = check_mx_rows(m, k, dtype, codes, scales)) return e;
  if (!x) return fail(SAGE_ERR_ARG, "null tensor pointer");
  if (reinterpret_cast<uintptr_t>(x) & 1u) return fail(SAGE_ERR_ALIGN, "x must be aligned to its elements");
  const sage::MxQuantArgs a{x, m == 1 ? k : x_rs, m, (int)k, (int)sage::mx_cols(k), in_place(x, x_rs, m, k),
                            static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales)};
  return launch_status(sage::launch_mx_quantize(a, dtype, stream), "sage_mxfp4_quantize");
}

int sage_mxfp4_dequantize(const void* codes, const void* scales, int64_t m, int64_t k, int dtype, void* out,
                          hipStream_t stream) {
  if (const int e = check_mx_rows(m, k, dtype, codes, scales)) return e;
  if (!out) return fail(SAGE_ERR_ARG, "null tensor pointer");
  if (reinterpret_cast<uintptr_t>(out) & 1u) return fail(SAGE_ERR_ALIGN, "out must be aligned to its elements");
  const sage::MxDequantArgs a{static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), m, (int)k,
                              (int)sage::mx_cols(k), out, k, aligned16(out) && k % 8 == 0};
  return launch_status(sage::launch_mx_dequantize(a, dtype, stream), "sage_mxfp4_dequantize");
}

size_t sage_mxfp4_linear_workspace_bytes(int64_t m, int64_t n, int64_t k, int activation, int quantize_x,
                                         int other_rows) {
  if (check_mx_linear(m, n, k, SAGE_DTYPE_BF16, activation)) return 0;
  // outputs, residual and bias on 16-byte boundaries or not: room for either
  const size_t bytes = MxLinear(m, n, k, activation, quantize_x, n % 8 == 0).bytes();
  return other_rows ? std::max(bytes, MxLinear(m, n, k, activation, quantize_x, false).bytes()) : bytes;
}

int sage_mxfp4_linear(const void* x, int64_t x_rs, const void* x_codes, const void* x_scales, const void* w_codes,
                      const void* w_scales, const void* bias, int bias_fp32, const void* residual, int64_t r_rs,
                      int64_t m, int64_t n, int64_t k, int dtype, int activation, void* workspace,
                      size_t workspace_bytes, float* z, void* out, hipStream_t stream) {
  if (const int e = check_mx_linear(m, n, k, dtype, activation)) return e;
  if (!out || !w_codes || !w_scales || (!x && (!x_codes || !x_scales)))
    return fail(SAGE_ERR_ARG, "null tensor pointer");
  if (residual)
    if (const int e = check_rows(r_rs, m, n, "residual")) return e;
  for (const void* p : {x, residual, (const void*)out})
    if (reinterpret_cast<uintptr_t>(p) & 1u) return fail(SAGE_ERR_ALIGN, "tensor pointers must be aligned to their elements");
  if (reinterpret_cast<uintptr_t>(z) & 3u || reinterpret_cast<uintptr_t>(bias) & (bias_fp32 ? 3u : 1u))
    return fail(SAGE_ERR_ALIGN, "bias must be aligned to its elements, z to 4 bytes");
  if (!aligned16(w_codes) || reinterpret_cast<uintptr_t>(w_scales) & 7u ||
      (!x && (!aligned16(x_codes) || reinterpret_cast<uintptr_t>(x_scales) & 7u)))
    return fail(SAGE_ERR_ALIGN, "codes must be 16-byte and scales 8-byte aligned");
  const bool vec = n % 8 == 0 && aligned16(out) && aligned16(z) && aligned16(bias) && aligned16(residual) &&
                   (!residual || m == 1 || r_rs % 8 == 0);
  MxLinear p(m, n, k, activation, mx_rows(x, x_rs, m, k), vec);
  if (p.bytes() && (!workspace || workspace_bytes < p.bytes()))
    return fail(SAGE_ERR_WORKSPACE, "workspace of %zu bytes needed, got %zu", p.bytes(), workspace_bytes);
  if (p.bytes() && !aligned16(workspace)) return fail(SAGE_ERR_ALIGN, "workspace must be 16-byte aligned");
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  sage::MxGemmArgs a{};
  if (x && p.quantizes) {
    a.x = x;
    a.ldx = m == 1 ? k : x_rs;
    a.kx = (int)k;
  } else if (x) {
    const int e = sage_mxfp4_quantize(x, x_rs, m, k, dtype, ws, ws + p.scales, stream);
    if (e) return e;
  }
  a.g = p.g;
  a.g.a = x ? ws : x_codes;
  a.g.b = w_codes;
  a.sa = x ? ws + p.scales : static_cast<const uint8_t*>(x_scales);
  a.sb = static_cast<const uint8_t*>(w_scales);
  a.g.bias = bias;
  a.g.bias_f32 = bias_fp32 != 0;
  a.g.res = residual;
  a.g.ldr = m == 1 ? n : r_rs;
  a.g.z = z;
  a.g.out = out;
  a.g.part = reinterpret_cast<float*>(ws + p.part);
  return launch_status(sage::launch_mx_gemm(a, dtype, stream), "sage_mxfp4_linear");
}

size_t sage_mxfp4_linear_bwd_workspace_bytes(const void* dout, int64_t d_rs, int64_t m, int64_t n, int64_t k,
                                             int activation, int want) {
  if (check_mx_linear(m, n, k, SAGE_DTYPE_BF16, activation)) return 0;
  if (want & 1 && check_linear(m, n, k, 0, SAGE_DTYPE_BF16, activation)) return 0;
  return LinearBwd(dout, d_rs, nullptr, 0, nullptr, 0, m, n, k, activation, want & 5, true).bytes;
}

int sage_mxfp4_linear_bwd(const void* dout, int64_t d_rs, const void* w_codes, const void* w_scales, const float* z,
                          int64_t m, int64_t n, int64_t k, int dtype, int activation, int bias_fp32, void* workspace,
                          size_t workspace_bytes, void* dx, void* dbias, hipStream_t stream) {
  if (const int e = check_mx_linear(m, n, k, dtype, activation)) return e;
  if (dx)
    if (const int e = check_linear(m, n, k, 0, dtype, activation)) return e;  // the weight's 16-bit rows
  const int want = (dx ? 1 : 0) | (dbias ? 4 : 0);
  if (!dout || (dx && (!w_codes || !w_scales)) || (activation != SAGE_ACT_NONE && !z))
    return fail(SAGE_ERR_ARG, "null tensor pointer");
  if (!want) return SAGE_OK;
  if (const int e = check_rows(d_rs, m, n, "dout")) return e;
  if (reinterpret_cast<uintptr_t>(z) & 3u) return fail(SAGE_ERR_ALIGN, "z must be aligned to 4 bytes");
  if (reinterpret_cast<uintptr_t>(dout) & 1u || reinterpret_cast<uintptr_t>(dbias) & (bias_fp32 ? 3u : 1u))
    return fail(SAGE_ERR_ALIGN, "tensor pointers must be aligned to their elements");
  if (!aligned16(dx) || !aligned16(w_codes) || reinterpret_cast<uintptr_t>(w_scales) & 7u)
    return fail(SAGE_ERR_ALIGN, "dx and codes must be 16-byte and scales 8-byte aligned");
  const LinearBwd p(dout, d_rs, nullptr, 0, nullptr, 0, m, n, k, activation, want, true);
  return run_linear_bwd(p, dout, d_rs, nullptr, 0, nullptr, 0, static_cast<const uint8_t*>(w_codes),
                        static_cast<const uint8_t*>(w_scales), z, m, n, k, dtype, activation, bias_fp32, workspace,
                        workspace_bytes, dx, nullptr, dbias, stream);
}

int sage_rms_norm_modulate_mxfp4(const void* x, int64_t x_bs, int64_t x_rs, const void* weight, const void* scale,
                                 int64_t scale_bs, int64_t scale_gs, int64_t groups, const int32_t* doc_ids, int64_t b,
                                 int64_t n, int64_t c, int dtype, int fp32_params, double eps, void* codes,
                                 void* scales, hipStream_t stream) {
  sage::NormArgs a = norm_args(x, x_bs, x_rs, weight, scale, scale_bs, scale_gs, groups, doc_ids, b, n, c,
                               fp32_params, (float)eps);
  a.eps64 = eps;
  if (!(eps >= 0.0)) return fail(SAGE_ERR_ARG, "eps must be >= 0");
  if (const int e = check_norm(a, b, n, c, groups, dtype, fp32_params)) return e;
  if (!x) return fail(SAGE_ERR_ARG, "null tensor pointer");
  if (const int e = check_norm_align(a)) return e;
  if (const int e = check_mx_rows(b * n, c, dtype, codes, scales)) return e;
  return launch_status(sage::launch_norm_mx(sage::kNormModulate, dtype, a, static_cast<uint8_t*>(codes),
                                            static_cast<uint8_t*>(scales), stream),
                       "sage_rms_norm_modulate_mxfp4");
}

int sage_rms_norm_gate_residual_modulate_mxfp4(
    const void* residual, int64_t r_bs, int64_t r_rs, const void* x, int64_t x_bs, int64_t x_rs, const void* weight,
    const void* gate, int64_t gate_bs, int64_t gate_gs, const void* next_weight, const void* next_scale,
    int64_t scale_bs, int64_t scale_gs, int64_t groups, const int32_t* doc_ids, int64_t b, int64_t n, int64_t c,
    int dtype, int fp32_params, double eps, void* hidden, void* codes, void* scales, hipStream_t stream) {
  sage::NormArgs a = norm_args(x, x_bs, x_rs, weight, gate, gate_bs, gate_gs, groups, doc_ids, b, n, c, fp32_params,
                               (float)eps);
  a.eps64 = eps;
  if (!(eps >= 0.0)) return fail(SAGE_ERR_ARG, "eps must be >= 0");
  if (const int e = check_norm(a, b, n, c, groups, dtype, fp32_params)) return e;
  if (!residual || !x || !hidden) return fail(SAGE_ERR_ARG, "null tensor pointer");
  a.res = {residual, r_bs, r_rs};
  a.w2 = {next_weight, fp32_params & SAGE_FP32_NEXT_WEIGHT ? 1 : 0};
  a.cond2 = {next_scale, fp32_params & SAGE_FP32_NEXT_SCALE ? 1 : 0, (int)groups, scale_bs, scale_gs};
  a.hidden = hidden;
  if (const int e = check_norm_align(a)) return e;
  if (const int e = check_mx_rows(b * n, c, dtype, codes, scales)) return e;
  return launch_status(sage::launch_norm_mx(sage::kNormGateModulate, dtype, a, static_cast<uint8_t*>(codes),
                                            static_cast<uint8_t*>(scales), stream),
                       "sage_rms_norm_gate_residual_modulate_mxfp4");
}

}  // extern "C"
