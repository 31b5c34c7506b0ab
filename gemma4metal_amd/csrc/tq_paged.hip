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
__global__ __launch_bounds__(256) void paged_rows_kernel(PagedParams p, int64_t rows) {
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
int launch_rows(const PagedParams& p, int sb_dtype, int64_t rows, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>((rows + 3) / 4);
  if (sb_dtype == TQ_F16) paged_rows_kernel<D, __half><<<grid, 256, 0, s>>>(p, rows);
  else paged_rows_kernel<D, float><<<grid, 256, 0, s>>>(p, rows);
  TQ_CHECK_LAUNCH("paged_rows_kernel");
  return TQ_OK;
}

// What both calls refuse; fills the parameters that they share.
int paged_params(PagedParams& p, const void* q, int q_dtype, const uint32_t* kq, const void* ks, const void* kb,
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

// Kernel and split plan of a decode call: sdpa_int4_hc2_kernel for D 512 with
// GQA a multiple of 8, else sdpa_int4_mfma_kernel, on blocks of 32 keys.
struct PagedPlan {
  bool hc;
  int G, n_sub, chunk, max_splits;
  bool lpt;
  WsLayout wl;
};

// max_len: what any sequence attends beside the shared rows, at most.
PagedPlan plan_paged(int batch, int Hq, int Hkv, int D, int sb_dtype, int max_len) {
  PagedPlan pl{};
  const int gqa = Hq / Hkv;
  pl.hc = D == 512 && gqa % 8 == 0;
  pl.G = head_subgroup(gqa);
  while (!pl.hc && pl.G > 1 && !mfma_serves(D, pl.G, sb_dtype)) pl.G /= 2;
  pl.n_sub = gqa / pl.G;
  const int64_t groups = static_cast<int64_t>(batch) * Hkv * pl.n_sub;
  const int len = static_cast<int>(std::min<int64_t>((static_cast<int64_t>(max_len) + 31) / 32 * 32, 0x7FFFFFE0));
  const int min_splits = min_splits_for(batch);
  pl.chunk = (plan_chunk(len, groups, min_splits) + 31) / 32 * 32;
  pl.max_splits = max_splits_bound(len, groups, min_splits);
  // the device chooses the chunk (see plan_sdpa)
  pl.lpt = batch <= 64 && !pl.hc;
  if (pl.lpt && groups >= 2 * static_cast<int64_t>(target_wgs()) && pl.max_splits > 2) {
    pl.max_splits = 2;
    pl.chunk = std::max(pl.chunk, ((len + 1) / 2 + 127) / 128 * 128);
  }
  pl.wl = ws_layout(batch, Hq, D, pl.max_splits);
  return pl;
}

// Keys a sequence attends at most, in whole blocks.
int attended_bound(int max_kv_len, int window, bool windows, int sinks) {
  if (windows || window == 0) return max_kv_len;
  const int64_t most = static_cast<int64_t>(window) + 62 + (static_cast<int64_t>(sinks) + 31) / 32 * 32;
  return static_cast<int>(std::min<int64_t>(most, max_kv_len));
}

int launch_any(const PagedParams& p, int D, int sb_dtype, int64_t rows, hipStream_t s) {
  if (D == 128) return launch_rows<128>(p, sb_dtype, rows, s);
  if (D == 256) return launch_rows<256>(p, sb_dtype, rows, s);
  return launch_rows<512>(p, sb_dtype, rows, s);
}

}  // namespace
}  // namespace tq

using namespace tq;

extern "C" size_t tq_sdpa_int4_paged_workspace_size(int batch, int num_heads, int num_kv_heads, int head_dim,
                                                    int max_kv_len, int shared_prefix) {
  if (batch < 1 || num_kv_heads < 1 || num_heads < num_kv_heads || max_kv_len < 0 || shared_prefix < 0) return 0;
  // (every plan of a call with these sizes: a window only shortens the splits)
  const int gqa = num_heads / num_kv_heads;
  const int64_t groups = static_cast<int64_t>(batch) * num_kv_heads * (gqa / head_subgroup(gqa));
  return ws_layout(batch, num_heads, head_dim, max_splits_bound(max_kv_len, groups, min_splits_for(batch))).total;
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
  PagedParams p{};
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
  if (shared_prefix > 0)
    return launch_any(p, head_dim, sb_dtype, static_cast<int64_t>(batch) * num_heads, static_cast<hipStream_t>(stream));
  const PagedPlan pl = plan_paged(batch, num_heads, num_kv_heads, head_dim, sb_dtype,
                                  attended_bound(max_kv_len, sliding_window, windows != nullptr, num_sinks));
  TQ_CHECK_ARG(num_kv_heads * static_cast<int64_t>(pl.n_sub) <= 65535, "%s: grid too large", fn);
  TQ_CHECK_ARG(static_cast<int64_t>(batch) * num_heads <= kMaxCounters, "%s: batch * num_heads must be <= %lld", fn,
               static_cast<long long>(kMaxCounters));
  p.n_sub = pl.n_sub;
  p.chunk = pl.chunk;
  p.max_splits = pl.max_splits;
  p.lpt = pl.lpt ? 1 : 0;
  if (pl.max_splits > 1) {
    if (!workspace || workspace_bytes < pl.wl.total) {
      set_error("%s: workspace of %zu bytes needed (got %zu)", fn, pl.wl.total, workspace_bytes);
      return TQ_ERR_WORKSPACE;
    }
    TQ_CHECK_ARG(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "%s: workspace must be 16-byte aligned", fn);
    // the split partials are addressed with 32-bit byte offsets
    TQ_CHECK_ARG(pl.wl.total - pl.wl.o_off < (size_t{1} << 31), "%s: split-K partials exceed 2 GiB", fn);
    char* ws = static_cast<char*>(workspace);
    p.ws_cnt = reinterpret_cast<int*>(ws + pl.wl.cnt_off);
    p.ws_ml = reinterpret_cast<float*>(ws + pl.wl.ml_off);
    p.ws_o = reinterpret_cast<float*>(ws + pl.wl.o_off);
  }
  const dim3 grid(pl.max_splits, num_kv_heads * pl.n_sub, batch);
  p.cnt_stride = counter_stride(static_cast<int64_t>(batch) * num_heads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (!pl.hc) return launch_sdpa_mfma(p, head_dim, pl.G, sb_dtype, grid, s);
  p.ext_merge = pl.max_splits > 1 ? 1 : 0;
  const int r = launch_sdpa_hc(p, sb_dtype, grid, s);
  return r != TQ_OK || !p.ext_merge ? r : launch_merge_splits(p, head_dim, batch, s);
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
  PagedParams p{};
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
