// Attention over the paged int4 cache (single tokens, batches that share a
// prefix, prompts), with a sliding window and first tokens that stay visible:
// argument checks, split plans and launches.  Single tokens run the decode
// kernels in their paged form (tq_sdpa_mfma.hip, tq_sdpa_hc.hip); prompts, and
// the part of a batch's keys that all its sequences share, run the K/V-tile
// kernel (tq_paged_tiles.hip), whose partials the decode kernel joins with those
// of each sequence's own keys.
#include <math.h>

#include <algorithm>
#include <cstdio>

#include "tq_sdpa_common.h"

namespace tq {
namespace {

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
  int G, n_sub, chunk;
  int max_splits;  // of any sequence
  int grid_x;      // workgroups per (sequence, head) of the grid, on average
  bool lpt;        // the device chooses the chunk and orders the jobs (paged_job)
  int waves;       // of a workgroup
  int slots;       // workgroups that the chip runs at once
};

// Splits of a sequence that the device may choose (see plan_paged), from those of
// equal sequences.
int lpt_splits(int splits, int len, int64_t groups, int64_t slots) {
  return static_cast<int>(std::min<int64_t>({2 * static_cast<int64_t>(splits), std::max((static_cast<int64_t>(len) + 127) / 128, int64_t{1}),
                                             kMaxSplits, 1 + (2 * slots + groups - 1) / groups}));
}

// max_len: what any sequence attends beside the shared rows, at most.
PagedPlan plan_paged(int batch, int Hq, int Hkv, int D, int sb_dtype, int max_len) {
  PagedPlan pl{};
  const int gqa = Hq / Hkv;
  pl.hc = D == 512 && gqa % 8 == 0;
  pl.G = head_subgroup(gqa);
  while (!pl.hc && pl.G > 1 && !mfma_serves(D, pl.G, sb_dtype)) pl.G /= 2;
  pl.n_sub = gqa / pl.G;
  const int64_t groups = static_cast<int64_t>(batch) * Hkv * pl.n_sub, cus = target_wgs();
  const int len = static_cast<int>(std::min<int64_t>((static_cast<int64_t>(max_len) + 31) / 32 * 32, 0x7FFFFFE0));
  const int min_splits = min_splits_for(batch);
  pl.chunk = (plan_chunk(len, groups, min_splits) + 31) / 32 * 32;
  pl.grid_x = pl.max_splits = max_splits_bound(len, groups, min_splits);
  // Four waves a workgroup, two workgroups a CU: one streams under the other's
  // prologue and merge.  64 sequences of 256 .. 1,024 keys (Hq 32 Hkv 16 D 256) 38
  // against 52 us, 32 with a window of 1,024 33 against 42; eight waves once every CU
  // has 24,576 keys to stream: 64 of 4,096 .. 16,384 keys (Hq 16 Hkv 8 D 128) 136
  // against 150 us, 16 such sequences of D 256 140 both.
  pl.waves = D != 512 && !(len >= 12288 && groups * len >= cus * 24576) ? 4 : 8;
  pl.slots = static_cast<int>(pl.waves == 4 ? 2 * cus : cus);
  // Batches of up to 64 sequences, where there is something to choose or to order.
  // The longest sequences may then be split twice as far as equal ones would be;
  // the grid holds a job per sequence and one per slot beside (workgroups without
  // a job cost 2 to 3 us of a slot each round).
  pl.lpt = batch > 1 && batch <= 64 && (pl.max_splits > 1 || groups > pl.slots);
  if (pl.lpt) {
    pl.max_splits = lpt_splits(pl.max_splits, len, groups, pl.slots);
    pl.grid_x = static_cast<int>(std::min<int64_t>(pl.max_splits, 1 + (pl.slots + groups - 1) / groups));
  }
  // every sequence's keys fit its splits
  const int64_t least = (static_cast<int64_t>(len) + pl.max_splits - 1) / pl.max_splits;
  pl.chunk = static_cast<int>(std::max<int64_t>(pl.chunk, (least + 31) / 32 * 32));
  return pl;
}

// Splits of any plan of these sizes, whatever its window.
int max_paged_splits(int batch, int Hq, int Hkv, int D, int max_len) {
  const PagedPlan pl = plan_paged(batch, Hq, Hkv, D, TQ_F16, max_len);
  const int64_t groups = static_cast<int64_t>(batch) * Hkv * pl.n_sub;
  const int s = max_splits_bound(max_len, groups, min_splits_for(batch));
  return std::max({pl.max_splits, s, lpt_splits(s, max_len, groups, 2 * target_wgs())});
}

// Keys a sequence attends at most, in whole blocks.
int attended_bound(int max_kv_len, int window, bool windows, int sinks) {
  if (windows || window == 0) return max_kv_len;
  const int64_t most = static_cast<int64_t>(window) + 62 + (static_cast<int64_t>(sinks) + 31) / 32 * 32;
  return static_cast<int>(std::min<int64_t>(most, max_kv_len));
}

// The split partials of a call in its workspace, and behind them the chunk that a
// launch chose.
constexpr size_t kWsTail = 256;

int set_workspace(PagedParams& p, void* workspace, size_t bytes, const WsLayout& wl, const char* fn) {
  const size_t need = wl.total + kWsTail;
  if (!workspace || bytes < need) {
    set_error("%s: workspace of %zu bytes needed (got %zu)", fn, need, workspace ? bytes : size_t{0});
    return TQ_ERR_WORKSPACE;
  }
  TQ_CHECK_ARG(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "%s: workspace must be 16-byte aligned", fn);
  // the split partials are addressed with 32-bit byte offsets
  TQ_CHECK_ARG(wl.total - wl.o_off < (size_t{1} << 31), "%s: split partials exceed 2 GiB", fn);
  char* ws = static_cast<char*>(workspace);
  p.ws_cnt = reinterpret_cast<int*>(ws + wl.cnt_off);
  p.ws_ml = reinterpret_cast<float*>(ws + wl.ml_off);
  p.ws_o = reinterpret_cast<float*>(ws + wl.o_off);
  p.lpt_chunk = reinterpret_cast<int*>(ws + wl.total);
  return TQ_OK;
}

// Keys that a prompt's workgroup attends that ends at position n, about.
int64_t prompt_keys(int64_t n, int window, int sinks) {
  return window > 0 ? std::min<int64_t>(n, static_cast<int64_t>(window) + sinks + 64) : n;
}

}  // namespace
}  // namespace tq

using namespace tq;

extern "C" size_t tq_sdpa_int4_paged_workspace_size(int batch, int num_heads, int num_kv_heads, int head_dim,
                                                    int max_kv_len, int shared_prefix) {
  if (batch < 1 || num_kv_heads < 1 || num_heads < num_kv_heads || max_kv_len < 0 || shared_prefix < 0) return 0;
  // (every plan of a call with these sizes: a window only shortens the splits)
  if (num_heads % num_kv_heads != 0) return 0;
  const int gqa = num_heads / num_kv_heads;
  int splits = max_paged_splits(batch, num_heads, num_kv_heads, head_dim, max_kv_len);
  if (shared_prefix > 0)
    splits += std::max(plan_paged_tiles(static_cast<int64_t>(batch) * gqa, num_kv_heads, head_dim, shared_prefix, shared_prefix, false).splits,
                       plan_paged_tiles(static_cast<int64_t>(batch) * gqa, num_kv_heads, head_dim, shared_prefix, shared_prefix, true).splits);
  return ws_layout(batch, num_heads, head_dim, splits).total + kWsTail;
}

namespace {

// prefix_table: the pages of the shared rows; NULL: sequence 0's.
int paged_decode(const void* q, int q_dtype, const uint32_t* k_quant, const void* k_scales, const void* k_biases,
                 const uint32_t* v_quant, const void* v_scales, const void* v_biases, int sb_dtype, float* out, int batch,
                 int num_heads, int num_kv_heads, int head_dim, int page_size, int num_pages, const int32_t* block_tables,
                 int max_pages, const int32_t* seq_lens, const int32_t* windows, int max_kv_len, int gqa_factor,
                 float scale, int sliding_window, int num_sinks, const int32_t* prefix_table, int shared_prefix,
                 void* workspace, size_t workspace_bytes, void* stream, const char* fn) {
  clear_error();
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
  // of the rows behind the shared ones
  const PagedPlan pl = plan_paged(batch, num_heads, num_kv_heads, head_dim, sb_dtype,
                                  std::min(attended_bound(max_kv_len, sliding_window, windows != nullptr, num_sinks),
                                           max_kv_len - shared_prefix));
  TQ_CHECK_ARG(num_kv_heads * static_cast<int64_t>(pl.n_sub) <= 65535, "%s: grid too large", fn);
  TQ_CHECK_ARG(static_cast<int64_t>(batch) * num_heads <= kMaxCounters, "%s: batch * num_heads must be <= %lld", fn,
               static_cast<long long>(kMaxCounters));
  p.n_sub = pl.n_sub;
  p.chunk = pl.chunk;
  p.lpt = pl.lpt ? 1 : 0;
  p.lpt_jobs = pl.grid_x * batch;
  p.waves = pl.waves;
  p.cus = pl.slots;
  TilesPlan tiles{0, 0};
  if (shared_prefix > 0)
    tiles = plan_paged_tiles(static_cast<int64_t>(batch) * gqa_factor, num_kv_heads, head_dim, shared_prefix, shared_prefix,
                             q_dtype == TQ_F32 && sb_dtype == TQ_F32);
  p.pre = tiles.splits;
  p.max_splits = pl.max_splits + p.pre;
  if (p.max_splits > 1) {
    if (int r = set_workspace(p, workspace, workspace_bytes, ws_layout(batch, num_heads, head_dim, p.max_splits), fn)) return r;
  }
  const dim3 grid(pl.grid_x, num_kv_heads * pl.n_sub, batch);
  p.cnt_stride = counter_stride(static_cast<int64_t>(batch) * num_heads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p.pre > 0) {
    PagedParams t = p;
    if (prefix_table) t.tables = prefix_table;
    t.max_pages = shared_prefix / page_size;
    if (int r = launch_paged_tiles(t, head_dim, sb_dtype, tiles, true, s)) return r;
  }
  if (!pl.hc) return launch_sdpa_mfma(p, head_dim, pl.G, sb_dtype, grid, s);
  p.ext_merge = p.max_splits > 1 ? 1 : 0;
  const int r = launch_sdpa_hc(p, sb_dtype, grid, s);
  return r != TQ_OK || !p.ext_merge ? r : launch_merge_splits(p, head_dim, batch, s);
}

}  // namespace

extern "C" int tq_sdpa_int4_paged(const void* q, tq_dtype q_dtype, const uint32_t* k_quant, const void* k_scales,
                                  const void* k_biases, const uint32_t* v_quant, const void* v_scales,
                                  const void* v_biases, tq_dtype sb_dtype, float* out, int batch, int num_heads,
                                  int num_kv_heads, int head_dim, int page_size, int num_pages,
                                  const int32_t* block_tables, int max_pages, const int32_t* seq_lens,
                                  const int32_t* windows, int max_kv_len, int gqa_factor, float scale,
                                  int sliding_window, int num_sinks, int shared_prefix, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  return paged_decode(q, q_dtype, k_quant, k_scales, k_biases, v_quant, v_scales, v_biases, sb_dtype, out, batch, num_heads,
                      num_kv_heads, head_dim, page_size, num_pages, block_tables, max_pages, seq_lens, windows,
                      max_kv_len, gqa_factor, scale, sliding_window, num_sinks, nullptr, shared_prefix, workspace,
                      workspace_bytes, stream, "tq_sdpa_int4_paged");
}

extern "C" int tq_sdpa_int4_paged_prefix(const void* q, tq_dtype q_dtype, const uint32_t* k_quant,
                                         const void* k_scales, const void* k_biases, const uint32_t* v_quant,
                                         const void* v_scales, const void* v_biases, tq_dtype sb_dtype, float* out,
                                         int batch, int num_heads, int num_kv_heads, int head_dim, int page_size,
                                         int num_pages, const int32_t* block_tables, int max_pages,
                                         const int32_t* seq_lens, const int32_t* windows, int max_kv_len,
                                         int gqa_factor, float scale, int sliding_window, int num_sinks,
                                         const int32_t* prefix_table, int shared_prefix, void* workspace,
                                         size_t workspace_bytes, void* stream) {
  return paged_decode(q, q_dtype, k_quant, k_scales, k_biases, v_quant, v_scales, v_biases, sb_dtype, out, batch, num_heads,
                      num_kv_heads, head_dim, page_size, num_pages, block_tables, max_pages, seq_lens, windows,
                      max_kv_len, gqa_factor, scale, sliding_window, num_sinks, prefix_table, shared_prefix, workspace,
                      workspace_bytes, stream, "tq_sdpa_int4_paged_prefix");
}

extern "C" int tq_sdpa_int4_paged_plan(int batch, int num_heads, int num_kv_heads, int head_dim, int max_kv_len,
                                       int sliding_window, int num_sinks, int shared_prefix, int* splits,
                                       int* chunk_keys, int* shared_splits, int* on_device, char* kernel,
                                       size_t kernel_bytes) {
  clear_error();
  const char* fn = "tq_sdpa_int4_paged_plan";
  TQ_CHECK_ARG(head_dim == 128 || head_dim == 256 || head_dim == 512, "%s: bad head_dim %d", fn, head_dim);
  TQ_CHECK_ARG(batch >= 1 && num_kv_heads >= 1 && num_heads >= num_kv_heads && num_heads % num_kv_heads == 0 &&
                   max_kv_len >= 0 && sliding_window >= 0 && num_sinks >= 0 && shared_prefix >= 0 &&
                   shared_prefix <= max_kv_len,
               "%s: bad shape", fn);
  const PagedPlan pl = plan_paged(batch, num_heads, num_kv_heads, head_dim, TQ_F16,
                                  std::min(attended_bound(max_kv_len, sliding_window, false, num_sinks),
                                           max_kv_len - shared_prefix));
  if (splits) *splits = pl.max_splits;
  if (chunk_keys) *chunk_keys = pl.chunk;
  if (shared_splits)
    *shared_splits = shared_prefix > 0 ? plan_paged_tiles(static_cast<int64_t>(batch) * (num_heads / num_kv_heads),
                                                          num_kv_heads, head_dim, shared_prefix, shared_prefix,
                                                          false).splits
                                       : 0;
  if (on_device) *on_device = pl.lpt ? 1 : 0;
  if (kernel && kernel_bytes > 0)
    std::snprintf(kernel, kernel_bytes, "%s", pl.hc ? "sdpa_int4_hc2_kernel" : "sdpa_int4_mfma_kernel");
  return TQ_OK;
}

extern "C" size_t tq_sdpa_int4_paged_prefill_workspace_size(int num_heads, int num_kv_heads, int head_dim,
                                                            int n_prior, int n_new) {
  if (num_kv_heads < 1 || num_heads < num_kv_heads || n_prior < 0 || n_new < 1) return 0;
  // (a window only shortens the splits)
  const int splits = paged_tiles_max_splits(static_cast<int64_t>(n_new) * (num_heads / num_kv_heads), num_kv_heads,
                                            head_dim, static_cast<int64_t>(n_prior) + (n_new + 1) / 2);
  return splits > 1 ? ws_layout(n_new, num_heads, head_dim, splits).total + kWsTail : 0;
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
  const int64_t rows = static_cast<int64_t>(n_new) * gqa_factor;
  TQ_CHECK_ARG(rows < (int64_t{1} << 31) && (rows + 63) / 64 * num_kv_heads < (int64_t{1} << 31), "%s: grid too large", fn);
  const TilesPlan tiles = plan_paged_tiles(
      rows, num_kv_heads, head_dim, prompt_keys(static_cast<int64_t>(n_prior) + (n_new + 1) / 2, sliding_window, num_sinks),
      prompt_keys(static_cast<int64_t>(n_prior) + n_new, sliding_window, num_sinks), q_dtype == TQ_F32 && sb_dtype == TQ_F32);
  p.max_splits = tiles.splits;
  if (tiles.splits > 1)
    if (int r = set_workspace(p, workspace, workspace_bytes, ws_layout(n_new, num_heads, head_dim, tiles.splits), fn)) return r;
  return launch_paged_tiles(p, head_dim, sb_dtype, tiles, false, static_cast<hipStream_t>(stream));
}

namespace {

// Sequences of a launch.  A job is found by a pass over them all, a wave's 64 at a time, and
// splits by up to six more: us a sequence of calls of 64, 1,024, 2,048 and 4,096 sequences
// (Hkv 8 D 128, up to 6,000 keys), one token 1.5, 1.0, 1.1, 1.3, 40 tokens 11.9, 11.5, 13.6,
// 17.6; it would be the square of them.
constexpr int kChunkSeqs = 1024;

// The partials of a batch's split blocks, behind the counters that other calls keep
// zeroed in the same workspace.
struct ChunksLayout {
  size_t ml, o, few_ml, few_o, total;
};

ChunksLayout chunks_layout(const ChunksPlan& pl, int D) {
  size_t at = ws_layout(0, 0, D, 0).ml_off;
  const auto take = [&](int64_t rows, int64_t floats) {
    const size_t from = at;
    at += (sizeof(float) * rows * floats + 255) / 256 * 256;
    return from;
  };
  ChunksLayout w;
  w.ml = take(pl.tiles.slots * 16 * pl.rs, 2);
  w.o = take(pl.tiles.slots * 16 * pl.rs, D);
  w.few_ml = take(pl.few_rows.slots * 16, 2);
  w.few_o = take(pl.few_rows.slots * 16, D);
  w.total = at;
  return w;
}

}  // namespace

extern "C" size_t tq_sdpa_int4_paged_chunks_workspace_size(int batch, int queries, int num_heads, int num_kv_heads,
                                                           int head_dim, int max_new, int max_kv_len) {
  if (batch < 1 || queries < 1 || num_kv_heads < 1 || num_heads < num_kv_heads || num_heads % num_kv_heads != 0 ||
      (head_dim != 128 && head_dim != 256 && head_dim != 512) || max_new < 0 || max_kv_len < 0)
    return 0;
  // (a window only takes keys away; where it leaves so few that nothing is split, none)
  size_t most = 0;
  for (int seqs : {std::min(batch, kChunkSeqs), batch % kChunkSeqs})
    for (int wide : {0, 1, 3}) {  // of the queries (1), and the scales
      if (seqs == 0) continue;
      const ChunksPlan pl = plan_chunks(seqs, batch, queries, num_heads / num_kv_heads, num_kv_heads, head_dim, max_new,
                                        max_kv_len, 0, 0, (wide & 1) != 0, (wide & 2) != 0);
      if (pl.tiles.slots + pl.few_rows.slots > 0) most = std::max(most, chunks_layout(pl, head_dim).total);
    }
  return most;
}

extern "C" int tq_sdpa_int4_paged_chunks(const void* q, tq_dtype q_dtype, const uint32_t* k_quant,
                                         const void* k_scales, const void* k_biases, const uint32_t* v_quant,
                                         const void* v_scales, const void* v_biases, tq_dtype sb_dtype, float* out,
                                         int batch, int queries, int num_heads, int num_kv_heads, int head_dim,
                                         int page_size, int num_pages, const int32_t* block_tables, int max_pages,
                                         const int32_t* starts, const int32_t* seq_lens, int max_new, int max_kv_len,
                                         int gqa_factor, float scale, int sliding_window, int num_sinks,
                                         void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  const char* fn = "tq_sdpa_int4_paged_chunks";
  TQ_CHECK_ARG(batch >= 0 && batch <= 65535, "%s: batch must be 0 to 65535", fn);
  TQ_CHECK_ARG(queries >= 0, "%s: queries must be >= 0", fn);
  TQ_CHECK_ARG(max_new >= 0, "%s: max_new must be >= 0", fn);
  if (batch == 0 || queries == 0) return TQ_OK;
  PagedParams p{};
  if (int r = paged_params(p, q, q_dtype, k_quant, k_scales, k_biases, v_quant, v_scales, v_biases, sb_dtype, out,
                           batch, num_heads, num_kv_heads, head_dim, page_size, num_pages, block_tables, max_pages,
                           gqa_factor, scale, sliding_window, num_sinks, fn))
    return r;
  TQ_CHECK_ARG(starts && seq_lens, "%s: null pointer", fn);
  TQ_CHECK_ARG(max_kv_len >= 0 && max_kv_len <= max_pages * page_size,
               "%s: need 0 <= max_kv_len <= max_pages * page_size (got %d, %d)", fn, max_kv_len, max_pages * page_size);
  TQ_CHECK_ARG(static_cast<int64_t>(queries) * num_heads < (int64_t{1} << 30), "%s: too many queries", fn);
  p.n_clamp = max_kv_len;
  const auto plan_of = [&](int seqs) {
    return plan_chunks(seqs, batch, queries, gqa_factor, num_kv_heads, head_dim, max_new, max_kv_len, sliding_window,
                       num_sinks, q_dtype == TQ_F32, sb_dtype == TQ_F32);
  };
  // (all checks before the first launch)
  for (int seqs : {std::min(batch, kChunkSeqs), batch % kChunkSeqs}) {
    if (seqs == 0) continue;
    const ChunksPlan plan = plan_of(seqs);
    TQ_CHECK_ARG(chunk_threads(plan, head_dim) < (int64_t{1} << 32), "%s: grid too large", fn);
    if (plan.tiles.slots + plan.few_rows.slots == 0) continue;
    const size_t need = chunks_layout(plan, head_dim).total;
    if (!workspace || workspace_bytes < need) {
      set_error("%s: workspace of %zu bytes needed (got %zu)", fn, need, workspace ? workspace_bytes : size_t{0});
      return TQ_ERR_WORKSPACE;
    }
    TQ_CHECK_ARG(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "%s: workspace must be 16-byte aligned", fn);
  }
  for (int b0 = 0; b0 < batch; b0 += kChunkSeqs) {  // (one after the other on the stream: one workspace)
    const ChunksPlan plan = plan_of(std::min(batch - b0, kChunkSeqs));
    const ChunksLayout wl = chunks_layout(plan, head_dim);
    const auto at = [&](size_t off) { return reinterpret_cast<float*>(static_cast<char*>(workspace) + off); };
    PagedParams part = p;
    part.nq = std::min(batch - b0, kChunkSeqs);
    part.tables = block_tables + static_cast<int64_t>(b0) * max_pages;
    part.seq_lens = seq_lens + b0;
    PagedParams few = part;
    if (plan.tiles.slots + plan.few_rows.slots > 0) {
      part.ws_ml = at(wl.ml);
      part.ws_o = at(wl.o);
      few.ws_ml = at(wl.few_ml);
      few.ws_o = at(wl.few_o);
    }
    if (int r = launch_chunks(part, few, head_dim, sb_dtype, plan, starts + b0, queries, max_new, static_cast<hipStream_t>(stream))) return r;
  }
  return TQ_OK;
}
