// Chunks of new tokens of a batch's sequences over pages: the kernel for sequences of
// few rows (queries x heads of a kv head), the merge of split jobs, and the plan.
// Sequences of more rows run paged_tiles_kernel, or both kinds paged_mixed_kernel
// (tq_paged_tiles.hip).
#include "tq_paged_few.h"

#include <climits>

#include <algorithm>

namespace tq {
namespace {

// Rows of a sequence up to which it is one of few.  In us, this kernel against the tile
// kernel, 32 sequences of 300 to 6,000 keys, bf16 queries and fp16 scales / fp32 queries /
// fp32 scales / both:
// D 128 (Hkv 8)  64 rows 144 : 169 / 150 : 181 / 148 : 187 / 157 : 194
//               128 rows 257 : 259 / 264 : 280 / 258 : 285 / 267 : 299
// D 256 (Hkv 16, window 1,024)
//                32 rows  93 : 124 / 123 : 133 / 109 : 129 / 146 : 154
//                48 rows 129 : 132 / 176 : 142 / 155 : 138 / 208 : 163
//                64 rows 167 : 137
// D 512 (Hkv 4)  16 rows 144 : 209 / 209 : 230 / 186 : 225 / 239 : 256
//                24 rows 284 : 216 / 403 : 237 / 353 : 232 / 456 : 263
// (fp32 queries are twice the operands, and fp32 scales twice the words, of registers that
// D 256 and 512 do not have: 19 to 79 and 95 to 208 of them are spilled.)
constexpr int few_rows(int D, bool wide) { return D == 512 ? 16 : D == 256 ? (wide ? 32 : 48) : 128; }
template <int D, bool F32, bool Q32>
__global__ __launch_bounds__((FewGeom<D, F32>::NT)) __attribute__((amdgpu_waves_per_eu(D == 512 ? 1 : 2, D == 512 ? 1 : 2)))
void paged_few_kernel(TileParams p) {
  __shared__ __attribute__((aligned(16))) typename FewGeom<D, F32>::Lds lds;
  few_job<D, F32, Q32>(p, blockIdx.x, threadIdx.x, lds);
}

// The outputs of split block j of one kernel's jobs, by workgroup y of ny.
constexpr int kMergeThreads = 256;
constexpr int kMergeParts = 4;  // workgroups of a block of paged_tiles_kernel

template <int D, int ROWS, int TK, bool FEW>
__device__ __forceinline__ void merge_job(const TileParams& p, int j, int y, int ny) {
  constexpr int D4 = D / 4;
  __shared__ int told[kJobInts];
  const ChunkJob job = chunk_job<ROWS, TK, FEW, true>(p, j, threadIdx.x, told);
  if (job.splits == 0) return;
  const int rows = min(job.n * p.gqa - job.blk * ROWS, ROWS);
  const float2* ml = reinterpret_cast<const float2*>(p.ws_ml) + static_cast<int64_t>(job.slot) * ROWS;
  const v4f* po = reinterpret_cast<const v4f*>(p.ws_o) + static_cast<int64_t>(job.slot) * ROWS * D4;
  for (int u = y * kMergeThreads + threadIdx.x; u < rows * D4; u += ny * kMergeThreads) {
    const int r = u / D4;
    float M = -INFINITY, L = 0.0f;
    v4f O = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = 0; k0 < job.splits; k0 += 4) {  // four in flight (past the end: the last one again, of weight 0)
      float2 x[4];
      v4f v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = min(k0 + i, job.splits - 1);
        x[i] = ml[k * ROWS + r];
        v[i] = po[static_cast<int64_t>(k) * ROWS * D4 + u];
      }
      float now = M;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (k0 + i >= job.splits) x[i].x = -INFINITY;
        now = fmaxf(now, x[i].x);
      }
      const float f = merge_factor(M, now);
      L *= f;
      O *= f;
      M = now;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float fk = merge_factor(x[i].x, M);
        L = fmaf(x[i].y, fk, L);
        O += fk * v[i];
      }
    }
    v4f y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = chunk_result(O[e], L);
    const int row = job.blk * ROWS + r, q = row / p.gqa;
    reinterpret_cast<v4f*>(p.out)[(static_cast<int64_t>(job.s0 + q) * p.Hq + job.kvh * p.gqa + (row - q * p.gqa)) * D4 + u % D4] = y;
  }
}

// few: the parameters of paged_few_kernel's jobs (the first few_n workgroups); tiles: the
// others'.  (Most workgroups find no split block: as many as the chip runs at once.)
template <int D, int ROWS>
__global__ __launch_bounds__(kMergeThreads) void merge_chunks_kernel(TileParams few, TileParams tiles, int few_n) {
  const int i = blockIdx.x;
  if (i < few_n) merge_job<D, kFewBlock, 32, true>(few, i, 0, 1);
  else merge_job<D, ROWS, D == 512 ? 32 : 64, false>(tiles, (i - few_n) / kMergeParts, (i - few_n) % kMergeParts, kMergeParts);
}

template <bool F32>
void launch_few(const TileParams& p, int D, dim3 grid, hipStream_t s) {
  const bool q32 = p.q_dtype == TQ_F32;
  const auto run = [&](auto d) {
    constexpr int kD = decltype(d)::value;
    if (q32) paged_few_kernel<kD, F32, true><<<grid, FewGeom<kD, F32>::NT, 0, s>>>(p);
    else paged_few_kernel<kD, F32, false><<<grid, FewGeom<kD, F32>::NT, 0, s>>>(p);
  };
  if (D == 512) run(std::integral_constant<int, 512>{});
  else if (D == 256) run(std::integral_constant<int, 256>{});
  else run(std::integral_constant<int, 128>{});
}

template <int D>
void launch_merge(const TileParams& few, const TileParams& tiles, int few_n, int rs, unsigned grid, hipStream_t s) {
  if constexpr (D < 512) {
    if (rs == 8) {
      merge_chunks_kernel<D, 128><<<grid, kMergeThreads, 0, s>>>(few, tiles, few_n);
      return;
    }
  }
  merge_chunks_kernel<D, 64><<<grid, kMergeThreads, 0, s>>>(few, tiles, few_n);
}

// The jobs of `blocks` blocks of rows of at most `keys` keys on `cus` workgroups at once,
// and the slots for the partials of split ones (chunk_tiles has both bounds).  Where the
// blocks, or those of the other kernel beside them (filled), fill the chip and none is
// longer than kEven keys, none is split: the merge's launch is 4 us (5 tokens of 32
// sequences behind a window of 1,024 53 us with it, 50 without), and jobs that there might
// be and are not, 11 ns each (2 chunks of 700 and 6 of 300, D 256, 214 us with splits of
// few rows in the grid, 209 without).
constexpr int kEven = 2048;

ChunkJobs jobs_of(int64_t blocks, int64_t keys, int tile, int least, int64_t cus, bool filled) {
  const int64_t tiles = (keys + tile - 1) / tile;
  const int64_t splits = std::min<int64_t>((tiles + least - 1) / least, kMostSplits);
  if (blocks == 0 || splits <= 1 || ((filled || blocks >= cus) && keys <= kEven)) return {blocks, 0};
  return {blocks + std::min(cus, blocks * (splits - 1)), std::min(2 * cus, blocks * splits)};
}

int64_t few_cus(int D) { return D == 512 ? target_wgs() : 2 * target_wgs(); }

}  // namespace

ChunksPlan plan_chunks(int batch, int of, int queries, int gqa, int Hkv, int D, int max_new, int64_t max_kv_len, int64_t window,
                       int64_t sinks, bool q32, bool s32) {
  ChunksPlan pl{};
  const int few = few_rows(D, q32 || s32);
  const int64_t rows = static_cast<int64_t>(std::min(max_new, queries)) * gqa, all = static_cast<int64_t>(queries) * gqa;
  const int64_t seqs = std::min(batch, queries);
  // keys of a block of R rows at most, in whole tiles of either kernel (no fewer than chunk_seq counts)
  const auto keys = [&](int64_t R) {
    return window > 0 ? std::min<int64_t>(max_kv_len, window + R + 256 + (sinks + 63) / 64 * 64) : max_kv_len;
  };
  pl.rs = D == 512 || (D == 256 && q32 && s32) || rows <= 64 ? 4 : 8;
  // sequences of few rows alone, or a batch that may hold some, or none.  (Us without and
  // with them apart, D 256: 3 chunks of 1,000 among 24 sequences 686, 549; 2 of 700 and 6 of
  // 300, none of them few, 207, 209.  At D 512, where a launch of its own without work takes
  // up to 10, only where chunks are short on average.)
  pl.few = rows <= few ? INT_MAX : batch > 1 && (D < 512 || all / of < 4 * few) ? few : 0;
  // blocks of rows of any chunks that add up to `queries`
  if (pl.few != INT_MAX) {
    const int64_t n = std::min(seqs, all / (pl.few + 1)), R = 16 * pl.rs;
    pl.tiles = jobs_of(std::min(all / R + n, n * ((rows + R - 1) / R)) * Hkv, keys(R), D == 512 ? 32 : 64,
                       kLeastTiles<false>, target_wgs(), false);
  }
  if (pl.few != 0) {
    const int64_t blocks = (std::min<int64_t>(rows, pl.few) + kFewBlock - 1) / kFewBlock;
    pl.few_rows = jobs_of(std::min(all / kFewBlock + seqs, seqs * blocks) * Hkv, keys(kFewBlock), 32,
                          kLeastTiles<true>, few_cus(D), D < 512 && pl.tiles.jobs > 0);
  }
  return pl;
}

int64_t chunk_threads(const ChunksPlan& plan, int D) {
  constexpr int64_t kTiles = kTileThreads, kFew = FewGeom<128, false>::NT;
  const bool one = D < 512 && plan.tiles.jobs > 0;  // (launch_chunks)
  return one ? kTiles * plan.tiles.jobs + kFew * (plan.few_rows.jobs + 1) : std::max(kTiles * plan.tiles.jobs, kFew * plan.few_rows.jobs);
}

int launch_chunks(const PagedParams& p0, const PagedParams& few0, int D, int sb_dtype, const ChunksPlan& plan,
                  const int* starts, int queries, int max_new, hipStream_t s) {
  TileParams p{}, few{};
  static_cast<PagedParams&>(p) = p0;
  static_cast<PagedParams&>(few) = few0;
  p.splits = few.splits = 1;
  p.starts = few.starts = starts;
  p.queries = few.queries = queries;
  p.few = few.few = plan.few;
  p.max_new = few.max_new = max_new;
  p.slots = static_cast<int>(plan.tiles.slots);
  few.slots = static_cast<int>(plan.few_rows.slots);
  few.cus = static_cast<int>(few_cus(D));
  const bool one = D < 512 && plan.tiles.jobs > 0;  // launch for both
  if (plan.tiles.jobs > 0)
    if (int r = launch_chunk_tiles(p, D, sb_dtype, plan.rs, plan.tiles.jobs, few, one ? plan.few_rows.jobs : 0, s)) return r;
  if (plan.few_rows.jobs > 0 && !one) {
    const dim3 grid(static_cast<unsigned>(plan.few_rows.jobs));
    if (sb_dtype == TQ_F32) launch_few<true>(few, D, grid, s);
    else launch_few<false>(few, D, grid, s);
    TQ_CHECK_LAUNCH("paged_few_kernel");
  }
  if (plan.few_rows.slots + plan.tiles.slots == 0) return TQ_OK;
  // (a split block has two slots at least)
  const int few_n = static_cast<int>(plan.few_rows.slots / 2);
  const unsigned grid = static_cast<unsigned>(few_n + plan.tiles.slots / 2 * kMergeParts);
  if (D == 512) launch_merge<512>(few, p, few_n, plan.rs, grid, s);
  else if (D == 256) launch_merge<256>(few, p, few_n, plan.rs, grid, s);
  else launch_merge<128>(few, p, few_n, plan.rs, grid, s);
  TQ_CHECK_LAUNCH("merge_chunks_kernel");
  return TQ_OK;
}

}  // namespace tq
