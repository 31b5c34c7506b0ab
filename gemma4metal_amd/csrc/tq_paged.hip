// Attention over the paged int4 cache (single tokens, batches that share a
// prefix, prompts), with a sliding window and first tokens that stay visible.
#include <math.h>

#include <algorithm>

#include "tq_sdpa_common.h"

namespace tq {
namespace {

// A wave per (query, head) row: lane i holds dims i E .. i E + E - 1, E = D / 64,
// and walks the row's keys one by one with a running maximum and sum.
template <int D, typename SB>
__global__ __launch_bounds__(256) void paged_rows_kernel(SdpaParams p, int64_t rows) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int b = static_cast<int>(row / p.Hq), h = static_cast<int>(row - static_cast<int64_t>(b) * p.Hq);
  const int kvh = h / p.gqa;
  const int n = p.prefill ? p.n + b + 1 : min(p.seq_lens[b], p.n_clamp);
  const int W = p.windows ? p.windows[b] : p.window;
  const int lo = W > 0 ? max(0, n - W) : 0;
  const int64_t mine = p.prefill ? 0 : static_cast<int64_t>(b) * p.max_pages;
  float q[E], o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = load_any(p.q, p.q_dtype, row * D + lane * E + e) * p.scale_log2;
    o[e] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int t = 0; t < n; ++t) {
    if (t < lo && t >= p.sinks) t = lo;
    const int page = p.tables[(t < p.shared ? 0 : mine) + (t >> p.page_shift)];
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.num_pages)) continue;
    const int64_t r = ((static_cast<int64_t>(page) * p.Hkv + kvh) << p.page_shift) + (t & ((1 << p.page_shift) - 1));
    const int64_t g = r * (D / 64) + lane * E / 64, w = r * (D / 8) + lane * E / 8;
    const int sh = 4 * (lane * E % 8);
    const float ks = sb_to_f32(static_cast<const SB*>(p.ks)[g]), kb = sb_to_f32(static_cast<const SB*>(p.kb)[g]);
    const float vs = sb_to_f32(static_cast<const SB*>(p.vs)[g]), vb = sb_to_f32(static_cast<const SB*>(p.vb)[g]);
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], fmaf(ks, static_cast<float>(p.kq[w] >> (sh + 4 * e) & 15u), kb), s);
    s = group_sum<64>(s);
    const float mn = fmaxf(m, s), f = merge_factor(m, mn), x = fast_exp2(s - mn);
    l = fmaf(l, f, x);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(o[e], f, x * fmaf(vs, static_cast<float>(p.vq[w] >> (sh + 4 * e) & 15u), vb));
    m = mn;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) p.out[row * D + lane * E + e] = normalise(o[e], l, 0.0f);
}

template <int D>
int launch_rows(const SdpaParams& p, int sb_dtype, int64_t rows, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>((rows + 3) / 4);
  if (sb_dtype == TQ_F16) paged_rows_kernel<D, __half><<<grid, 256, 0, s>>>(p, rows);
  else paged_rows_kernel<D, float><<<grid, 256, 0, s>>>(p, rows);
  TQ_CHECK_LAUNCH("paged_rows_kernel");
  return TQ_OK;
}

// What both calls refuse; fills the parameters that they share.
int paged_params(SdpaParams& p, const void* q, int q_dtype, const uint32_t* kq, const void* ks, const void* kb,
                 const uint32_t* vq, const void* vs, const void* vb, int sb_dtype, float* out, int batch, int Hq,
                 int Hkv, int D, int page_size, int num_pages, const int32_t* tables, int max_pages, int gqa,
                 float scale, int window, int sinks, const char* fn) {
  TQ_CHECK_ARG(valid_dtype(q_dtype), "%s: bad q_dtype %d", fn, q_dtype);
  TQ_CHECK_ARG(sb_dtype == TQ_F16 || sb_dtype == TQ_F32, "%s: sb_dtype must be f16 or f32", fn);
  if (D != 128 && D != 256 && D != 512) {
    set_error("%s: head_dim must be 128, 256 or 512 (got %d)", fn, D);
    return TQ_ERR_UNSUPPORTED;
  }
  TQ_CHECK_ARG(Hkv >= 1 && gqa >= 1, "%s: num_kv_heads and gqa_factor must be >= 1", fn);
  TQ_CHECK_ARG(Hq == static_cast<int64_t>(Hkv) * gqa, "%s: num_heads (%d) != num_kv_heads (%d) * gqa_factor (%d)", fn, Hq, Hkv, gqa);
  TQ_CHECK_ARG(Hq <= 65535, "%s: at most 65535 heads", fn);
  TQ_CHECK_ARG(window >= 0 && sinks >= 0, "%s: sliding_window and num_sinks must be >= 0", fn);
  TQ_CHECK_ARG(std::isfinite(scale), "%s: scale must be finite", fn);
  if (int r = check_paging(page_size, num_pages, max_pages, fn)) return r;
  TQ_CHECK_ARG(q && kq && ks && kb && vq && vs && vb && out && tables, "%s: null tensor pointer", fn);
  const struct { const void* t; const char* what; } aligned[] = {
      {q, "queries"}, {kq, "k_quant"}, {ks, "k_scales"}, {kb, "k_biases"}, {vq, "v_quant"}, {vs, "v_scales"},
      {vb, "v_biases"}, {out, "out"}};
  for (const auto& a : aligned)
    TQ_CHECK_ARG(reinterpret_cast<uintptr_t>(a.t) % 16 == 0, "%s: %s must be 16-byte aligned", fn, a.what);
  p.q = q;
  p.q_dtype = q_dtype;
  p.kq = kq; p.ks = ks; p.kb = kb;
  p.vq = vq; p.vs = vs; p.vb = vb;
  p.out = out;
  p.Hq = Hq; p.Hkv = Hkv; p.gqa = gqa;
  p.window = window;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.nq = batch;
  p.cus = target_wgs();
  p.tables = tables;
  p.max_pages = max_pages;
  p.num_pages = num_pages;
  p.page_shift = __builtin_ctz(static_cast<unsigned>(page_size));
  p.sinks = sinks;
  return TQ_OK;
}

int launch_any(const SdpaParams& p, int D, int sb_dtype, int64_t rows, hipStream_t s) {
  if (D == 128) return launch_rows<128>(p, sb_dtype, rows, s);
  if (D == 256) return launch_rows<256>(p, sb_dtype, rows, s);
  return launch_rows<512>(p, sb_dtype, rows, s);
}

}  // namespace
}  // namespace tq

using namespace tq;

extern "C" size_t tq_sdpa_int4_paged_workspace_size(int batch, int num_heads, int num_kv_heads, int head_dim,
                                                    int max_kv_len, int shared_prefix) {
  return 0;
}

extern "C" int tq_sdpa_int4_paged(const void* q, tq_dtype q_dtype, const uint32_t* k_quant, const void* k_scales,
                                  const void* k_biases, const uint32_t* v_quant, const void* v_scales,
                                  const void* v_biases, tq_dtype sb_dtype, float* out, int batch, int num_heads,
                                  int num_kv_heads, int head_dim, int page_size, int num_pages,
                                  const int32_t* block_tables, int max_pages, const int32_t* seq_lens,
                                  const int32_t* windows, int max_kv_len, int gqa_factor, float scale,
                                  int sliding_window, int num_sinks, int shared_prefix, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  clear_error();
  const char* fn = "tq_sdpa_int4_paged";
  TQ_CHECK_ARG(batch >= 0 && batch <= 65535, "%s: batch must be 0 to 65535", fn);
  if (batch == 0) return TQ_OK;
  SdpaParams p{};
  if (int r = paged_params(p, q, q_dtype, k_quant, k_scales, k_biases, v_quant, v_scales, v_biases, sb_dtype, out,
                           batch, num_heads, num_kv_heads, head_dim, page_size, num_pages, block_tables, max_pages,
                           gqa_factor, scale, sliding_window, num_sinks, fn))
    return r;
  TQ_CHECK_ARG(seq_lens != nullptr, "%s: seq_lens is NULL", fn);
  TQ_CHECK_ARG(max_kv_len >= 0 && max_kv_len <= max_pages * page_size,
               "%s: need 0 <= max_kv_len <= max_pages * page_size (got %d, %d)", fn, max_kv_len, max_pages * page_size);
  TQ_CHECK_ARG(shared_prefix >= 0 && shared_prefix % page_size == 0 && shared_prefix <= max_kv_len,
               "%s: shared_prefix (%d) must be a multiple of page_size (%d) from 0 to max_kv_len (%d)", fn,
               shared_prefix, page_size, max_kv_len);
  p.seq_lens = seq_lens;
  p.windows = windows;
  p.n_clamp = max_kv_len;
  p.shared = shared_prefix;
  return launch_any(p, head_dim, sb_dtype, static_cast<int64_t>(batch) * num_heads, static_cast<hipStream_t>(stream));
}

extern "C" size_t tq_sdpa_int4_paged_prefill_workspace_size(int num_heads, int num_kv_heads, int head_dim,
                                                            int n_prior, int n_new) {
  return 0;
}

extern "C" int tq_sdpa_int4_paged_prefill(const void* q, tq_dtype q_dtype, const uint32_t* k_quant,
                                          const void* k_scales, const void* k_biases, const uint32_t* v_quant,
                                          const void* v_scales, const void* v_biases, tq_dtype sb_dtype, float* out,
                                          int num_heads, int num_kv_heads, int head_dim, int page_size, int num_pages,
                                          const int32_t* block_table, int max_pages, int n_prior, int n_new,
                                          int gqa_factor, float scale, int sliding_window, int num_sinks,
                                          void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  const char* fn = "tq_sdpa_int4_paged_prefill";
  TQ_CHECK_ARG(n_prior >= 0 && n_new >= 0, "%s: n_prior and n_new must be >= 0", fn);
  if (n_new == 0) return TQ_OK;
  SdpaParams p{};
  if (int r = paged_params(p, q, q_dtype, k_quant, k_scales, k_biases, v_quant, v_scales, v_biases, sb_dtype, out,
                           n_new, num_heads, num_kv_heads, head_dim, page_size, num_pages, block_table, max_pages,
                           gqa_factor, scale, sliding_window, num_sinks, fn))
    return r;
  TQ_CHECK_ARG(static_cast<int64_t>(n_prior) + n_new <= static_cast<int64_t>(max_pages) * page_size,
               "%s: n_prior + n_new (%d + %d) exceeds max_pages * page_size (%d)", fn, n_prior, n_new,
               max_pages * page_size);
  TQ_CHECK_ARG(n_new <= 65535, "%s: at most 65535 queries per call", fn);
  p.prefill = 1;
  p.n = n_prior;
  return launch_any(p, head_dim, sb_dtype, static_cast<int64_t>(n_new) * num_heads, static_cast<hipStream_t>(stream));
}
