// Chunks of new tokens of a batch's sequences (tq_paged_chunks.hip): the parameters of
// the multi-query kernels over pages, and the jobs of a launch, which the device lays
// out from the lengths.
#pragma once

#include "tq_sdpa_common.h"

namespace tq {

struct TileParams : PagedParams {
  int splits;  // workgroups along the tiles (grid y); 1: write p.out
  // chunks of a batch (nq sequences): their queries are rows starts[b] .. starts[b + 1] - 1
  // of q and out, of `queries` in all.  Sequences of at most `few` rows (queries x heads of
  // a kv head) are the business of few_job, the others of tiles_job.
  const int* starts;
  int queries, few;
  int max_new;  // queries of a sequence that are served
  int slots;    // of the workspace; 0: no splits
};

constexpr int kTileThreads = 512;  // of paged_tiles_kernel and paged_mixed_kernel

// few_jobs > 0: both kernels' jobs in one launch (D < 512).
int launch_chunk_tiles(const TileParams& p, int D, int sb_dtype, int rs, int64_t jobs, const TileParams& few,
                       int64_t few_jobs, hipStream_t s);

namespace {

// Largest of 64 lanes, by the steps of wave_max_dpp (wave_max_i goes through the
// LDS: six of them were 1.5 us of a launch's start).
__device__ __forceinline__ int max_of_wave(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false));
  const auto a = __builtin_amdgcn_permlane16_swap(static_cast<unsigned>(v), static_cast<unsigned>(v), false, false);
  v = max(static_cast<int>(a[0]), static_cast<int>(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(static_cast<unsigned>(v), static_cast<unsigned>(v), false, false);
  return __builtin_amdgcn_readfirstlane(max(static_cast<int>(b[0]), static_cast<int>(b[1])));
}
__device__ __forceinline__ int min_of_wave(int v) { return -max_of_wave(-v); }

// A row's result: 0 where it attends nothing (weights of NaN stay NaN).
__device__ __forceinline__ float chunk_result(float O, float L) { return L == 0.0f ? 0.0f : O / L; }

// A job is (sequence, block of rows, kv head, split of its tiles); the device lays them
// out from the lengths.  A wave of every workgroup works it out, a sequence a lane: one
// round trip to the lengths, where a plan of its own would be a launch.
struct ChunkSeq {
  int s0, n, len;      // first query, queries, keys
  int blocks, tiles;   // of rows; of keys (the most that a block of rows attends)
};

struct ChunkJob {
  int b, s0, n, len;
  int blk, kvh, split, splits;
  int slot;            // of its partials
};
constexpr int kJobInts = sizeof(ChunkJob) / sizeof(int);

template <int ROWS, int TK, bool FEW>
__device__ __forceinline__ ChunkSeq chunk_seq(const TileParams& p, int b) {
  ChunkSeq c{0, 0, 0, 0, 0};
  if (b < p.nq) {
    c.s0 = min(max(p.starts[b], 0), p.queries);
    c.n = min(max(p.starts[b + 1], c.s0), p.queries) - c.s0;
    c.len = max(min(p.seq_lens[b], p.n_clamp), 0);
    if ((c.n * p.gqa <= p.few) == FEW) c.blocks = (min(c.n, p.max_new) * p.gqa + ROWS - 1) / ROWS;
    c.tiles = (c.len + TK - 1) / TK;
    if (p.window > 0) {  // sinks, the rows' windows, and a tile that those begin in
      const int64_t keys = static_cast<int64_t>(p.window) + ROWS + 2 * TK;
      c.tiles = static_cast<int>(min(static_cast<int64_t>(c.tiles), keys / TK + p.sinks / TK + 1));
    }
  }
  return c;
}

__device__ __forceinline__ float sum_of_wave(float v) { return group_sum<64>(v); }

// Tiles of a job at most.  With T >= work / cus (workgroups that run at once), splits make
// fewer than cus more jobs of the blocks, and jobs of split blocks are fewer than 2 cus: a
// block of t > T tiles makes ceil(t / T) < 1 + t / T < 2 t / T of them.  Of a few such T,
// and of no splits, the one with the least estimated time, in the units of
// plan_paged_tiles: that of a job or of an even share of all.
constexpr int kMostSplits = 64;
template <bool FEW>
constexpr int kLeastTiles = FEW ? 16 : 4;

// (one function of the lengths for all who ask; one more or less than the quotient rounded
// up would do: a block's tiles are shared out evenly whatever it is)
__device__ __forceinline__ int splits_of(const ChunkSeq& c, int T) {
  return c.tiles <= T ? 1 : min(static_cast<int>(ceilf(c.tiles * __builtin_amdgcn_rcpf(static_cast<float>(T)))), kMostSplits);
}

// f(sequence of this lane) for the sequences of the batch, 64 at a time; `first`: the
// first 64, loaded once.
template <int ROWS, int TK, bool FEW, typename F>
__device__ __forceinline__ void each_seq(const TileParams& p, const ChunkSeq& first, F f) {
  f(first);
#pragma unroll 1
  for (int b0 = 64; b0 < p.nq; b0 += 64) f(chunk_seq<ROWS, TK, FEW>(p, b0 + static_cast<int>(threadIdx.x & 63)));
}

template <int ROWS, int TK, bool FEW>
__device__ __forceinline__ int chunk_tiles(const TileParams& p, const ChunkSeq& first) {
  float work = 0.0f, blocks = 0.0f;
  int most = 0;
  each_seq<ROWS, TK, FEW>(p, first, [&](const ChunkSeq& c) {
    const float n = static_cast<float>(c.blocks) * p.Hkv;
    work += n * c.tiles;
    blocks += n;
    if (c.blocks > 0) most = max(most, c.tiles);
  });
  work = sum_of_wave(work);
  blocks = sum_of_wave(blocks);
  most = max_of_wave(most);
  constexpr float kTile = FEW ? 1.0f : ROWS == 64 ? 8.0f : 13.0f, kFixed = FEW ? 24.0f : ROWS == 64 ? 48.0f : 72.0f;
  const float cus = static_cast<float>(p.cus), share = work / cus;
  const auto time = [&](float jobs, int T) {
    return fmaxf(T * kTile + kFixed, (work * kTile + jobs * kFixed) / cus + (jobs > cus ? 0.5f * T * kTile : 0.0f));
  };
  int best = max(most, 1);
  float least = time(blocks, best);
#pragma unroll 1
  for (int k = 2; k <= 8; k += k < 4 ? 1 : 2) {  // shares of 1, 1.5, 2, 3, 4
    const int T = max(static_cast<int>(fminf(share * (0.5f * k) * 1.0001f, 1e8f)) + 1, kLeastTiles<FEW>);
    if (T >= most) break;
    float jobs = 0.0f;
    each_seq<ROWS, TK, FEW>(p, first, [&](const ChunkSeq& c) { jobs += static_cast<float>(c.blocks) * p.Hkv * splits_of(c, T); });
    const float t = time(sum_of_wave(jobs), T);
    if (t < least) {
      least = t;
      best = T;
    }
  }
  return best;
}

// Inclusive prefix, of counts up to kMostJobs, where it stays: starts that do not ascend may
// add up to anything, and what lies past the grid or the slots is left out.
constexpr int kMostJobs = 1 << 29;

__device__ __forceinline__ int scan_of_wave(int v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(v, d, 64);
    if (lane >= d) v = min(v + y, kMostJobs);
  }
  return v;
}

// Job j (MERGE: the j-th split block of rows and head), or none: splits 0.
template <int ROWS, int TK, bool FEW, bool MERGE>
__device__ __forceinline__ ChunkJob find_chunk_job(const TileParams& p, int j) {
  const int lane = threadIdx.x & 63;
  const ChunkSeq first = chunk_seq<ROWS, TK, FEW>(p, lane);
  const int T = p.slots > 0 ? chunk_tiles<ROWS, TK, FEW>(p, first) : 1 << 30;
  int jobs = 0, slots = 0;  // of the sequences before these
  ChunkJob r{};
#pragma unroll 1
  for (int b0 = 0; b0 < p.nq; b0 += 64) {
    const ChunkSeq c = b0 == 0 ? first : chunk_seq<ROWS, TK, FEW>(p, b0 + lane);
    const int s = splits_of(c, T), mine = c.blocks * p.Hkv;
    const int slot = s > 1 ? min(mine * s, kMostJobs) : 0;
    const int n = MERGE ? (s > 1 ? mine : 0) : s > 1 ? slot : mine;
    const int upto = min(jobs + scan_of_wave(n), kMostJobs), slot_upto = min(slots + scan_of_wave(slot), kMostJobs);
    const uint64_t hit = __ballot(upto > j);
    if (hit != 0) {
      const int l = __builtin_ctzll(hit);
      const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      // (of the lanes before: not past j)
      const int before = l > 0 ? __builtin_amdgcn_readlane(upto, l - 1) : jobs;
      const int slot0 = l > 0 ? __builtin_amdgcn_readlane(slot_upto, l - 1) : slots;
      r.b = b0 + l;
      r.s0 = of(c.s0);
      r.n = of(c.n);
      r.len = of(c.len);
      r.splits = of(s);
      const int blocks = of(c.blocks);
      int at = j - before;
      r.kvh = at % p.Hkv;
      at /= p.Hkv;
      r.split = MERGE ? 0 : at % r.splits;
      if (!MERGE) at /= r.splits;
      r.blk = blocks - 1 - at;  // the longest key ranges (last queries) start first
      r.slot = slot0 + (r.blk * p.Hkv + r.kvh) * r.splits + r.split;
      if (r.splits > 1 && r.slot > p.slots - (MERGE ? r.splits : 1)) r.splits = 0;
      return r;
    }
    jobs = __builtin_amdgcn_readlane(upto, 63);
    slots = __builtin_amdgcn_readlane(slot_upto, 63);
  }
  return r;
}

// The same, found by the first of the waves that ask (tid: a thread's number among theirs)
// and told by way of the LDS.  A barrier of the workgroup.
template <int ROWS, int TK, bool FEW, bool MERGE>
__device__ __forceinline__ ChunkJob chunk_job(const TileParams& p, int j, int tid, int (&told)[kJobInts]) {
  if (tid < 64) {
    const ChunkJob r = find_chunk_job<ROWS, TK, FEW, MERGE>(p, j);
    const int v[kJobInts] = {r.b, r.s0, r.n, r.len, r.blk, r.kvh, r.split, r.splits, r.slot};
    if (tid == 0) {
#pragma unroll
      for (int i = 0; i < kJobInts; ++i) told[i] = v[i];
    }
  }
  __syncthreads();
  int v[kJobInts];
#pragma unroll
  for (int i = 0; i < kJobInts; ++i) v[i] = __builtin_amdgcn_readfirstlane(told[i]);
  return {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8]};
}

}  // namespace
}  // namespace tq
