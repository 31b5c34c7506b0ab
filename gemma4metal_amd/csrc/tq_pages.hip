// Page management of the paged int4 cache: reserving, forking, reordering, freeing,
// evicting, compacting and copying pages, all on the device.
//
// A call is a plan and an application.  The plan is integer work over the
// reference counts and the requests, by one workgroup (scans in order, so that
// the page a request gets does not depend on timing); the application copies
// pages with every CU and rewrites table rows.
#include "tq_internal.h"
#include "tq_page_plan.h"

#include <algorithm>
#include <type_traits>

namespace tq {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
// Free places and movers of a scan tile share one 32-bit count, 16 bits each.
constexpr int kScanPer = 4, kScanTile = kPlanThreads * kScanPer;
static_assert(kScanTile < 65536, "packed counts");

// Workspace of a plan (ints): its counts, per sequence the pages it needs and
// those needed before it, the free pages (compact: destinations), the movers'
// counts, the map of a compaction, and the copy jobs.
struct PlanWs {
  int* n_jobs;
  int* need;
  int* before;
  int* list;
  int* aux;
  int* map;
  int2* jobs;
};

size_t plan_ints(int64_t seqs, int64_t pages) { return 16 + 2 * seqs + 3 * pages + 2 * std::max(seqs, pages) + 4; }

PlanWs plan_ws(void* ws, int64_t seqs, int64_t pages) {
  int* p = static_cast<int*>(ws);
  PlanWs w;
  w.n_jobs = p;
  w.jobs = reinterpret_cast<int2*>(p + 16);
  p += 16 + 2 * std::max(seqs, pages);
  w.need = p;
  w.before = p + seqs;
  w.list = p + 2 * seqs;
  w.aux = w.list + pages;
  w.map = w.aux + pages;
  return w;
}

struct PlanParams {
  int32_t* tables;
  int32_t* refs;
  int32_t* lengths;
  const int32_t* ask;  // reserve: new rows; fork: parents
  int32_t* granted;
  int seqs, max_pages, num_pages, page_size;
  PlanWs w;
};

__device__ __forceinline__ bool is_page(int e, int num_pages) { return static_cast<unsigned>(e) < static_cast<unsigned>(num_pages); }

// The free pages, lowest first, until `want` of them are in list; how many are.
__device__ __forceinline__ int free_pages(const int32_t* refs, int num_pages, int want, int* list, int* lds) {
  int found = 0;
  for (int p0 = 0; p0 < num_pages && found < want; p0 += kScanTile) {  // uniform
    const int p = p0 + kScanPer * threadIdx.x;
    bool f[kScanPer];
    int n = 0;
#pragma unroll
    for (int i = 0; i < kScanPer; ++i) {
      f[i] = p + i < num_pages && refs[p + i] <= 0;
      n += f[i];
    }
    int total;
    int at = found + wg_scan<kPlanThreads>(n, lds, total);
#pragma unroll
    for (int i = 0; i < kScanPer; ++i)
      if (f[i]) list[at++] = p + i;
    found += total;
  }
  return found;
}

// Pages per request, -1 where there is none or it is refused; then the pages needed
// before each, the free pages, and the grants.  Chains of dependent loads bound it
// (request, length, parent, table), so a sequence gets kPlanGroup lanes and 64
// sequences are in flight: a fork of 56 sequences took 12 us with a wave a sequence,
// 6 us so.
constexpr int kPlanGroup = 16;

// Of the lanes of one's group, those with a condition.
__device__ __forceinline__ unsigned group_ballot(bool c) {
  return static_cast<unsigned>(__ballot(c) >> (threadIdx.x & 63 & ~(kPlanGroup - 1))) & ((1u << kPlanGroup) - 1);
}

template <bool FORK>
__global__ __launch_bounds__(kPlanThreads) void pages_plan_kernel(PlanParams p) {
  __shared__ int lds[kPlanWaves];
  using ScanSum = typename std::conditional<FORK, int, PlanSum>::type;  // (a fork needs one page at most)
  __shared__ ScanSum sums[kPlanWaves];
  constexpr int kGroups = kPlanThreads / kPlanGroup;
  const int lane = threadIdx.x % kPlanGroup, group = threadIdx.x / kPlanGroup;
  const int64_t rows = static_cast<int64_t>(p.max_pages) * p.page_size;
  for (int s = group; s < p.seqs; s += kGroups) {
    const int ask = p.ask[s], own = p.lengths[s];
    const int32_t* row = p.tables + static_cast<int64_t>(s) * p.max_pages;
    int need = -1;
    if constexpr (FORK) {
      if (ask >= 0 && ask < p.seqs && ask != s && own == 0) {
        const int grand = p.ask[ask];
        const int n = static_cast<int>(min(static_cast<int64_t>(max(p.lengths[ask], 0)), rows));
        bool page = false;
#pragma unroll 4
        for (int e = lane; e < p.max_pages; e += kPlanGroup) page |= is_page(row[e], p.num_pages);
        if (grand < 0 && group_ballot(page) == 0)
          need = n % p.page_size != 0 && is_page(p.tables[static_cast<int64_t>(ask) * p.max_pages + n / p.page_size], p.num_pages);
      }
    } else {
      const int64_t n = max(own, 0);
      const int64_t e1 = (n + ask + p.page_size - 1) / p.page_size;
      if (ask > 0 && e1 <= p.max_pages) {
        need = 0;
        for (int e = static_cast<int>(n / p.page_size); e < e1; e += kPlanGroup)
          need += __popc(group_ballot(e + lane < e1 && !is_page(row[e + lane], p.num_pages)));
      }
    }
    if (lane == 0) p.w.need[s] = need;
  }
  __syncthreads();
  PlanSum want = 0;
  for (int s0 = 0; s0 < p.seqs; s0 += kPlanThreads) {
    const int s = s0 + threadIdx.x;
    ScanSum total;
    const ScanSum b = wg_scan<kPlanThreads, ScanSum>(s < p.seqs ? max(p.w.need[s], 0) : 0, sums, total);
    if (s < p.seqs) p.w.before[s] = plan_before(want + b, p.num_pages);
    want += total;
  }
  const int found = free_pages(p.refs, p.num_pages, static_cast<int>(min(want, static_cast<PlanSum>(p.num_pages))), p.w.list, lds);
  __syncthreads();
  for (int s = FORK ? threadIdx.x : group; s < p.seqs; s += FORK ? kPlanThreads : kGroups) {
    const int need = p.w.need[s], before = p.w.before[s], ask = p.ask[s];
    const bool ok = plan_grants(need, before, found);
    if (FORK || lane == 0) p.granted[s] = ok;
    if (!ok) continue;
    if constexpr (FORK) {
      if (need > 0) {
        const int full = min(max(p.lengths[ask], 0) / p.page_size, p.max_pages - 1);
        const int dst = p.w.list[before];
        p.w.jobs[before] = int2{p.tables[static_cast<int64_t>(ask) * p.max_pages + full], dst};
        p.refs[dst] = 1;
      }
    } else {
      const int64_t n = max(p.lengths[s], 0);
      const int e1 = static_cast<int>((n + ask + p.page_size - 1) / p.page_size);
      int at = before;
      for (int e = static_cast<int>(n / p.page_size); e < e1; e += kPlanGroup) {
        int32_t* t = p.tables + static_cast<int64_t>(s) * p.max_pages + e + lane;
        const bool lacks = e + lane < e1 && !is_page(*t, p.num_pages);
        const unsigned m = group_ballot(lacks);
        if (lacks) {
          const int page = p.w.list[at + __popc(m & ((1u << lane) - 1))];
          *t = page;
          p.refs[page] = 1;
        }
        at += __popc(m);
      }
    }
  }
  if constexpr (FORK) {
    // granted requests for a page are the first `found` in order, all or none
    if (threadIdx.x == 0) *p.w.n_jobs = static_cast<int>(min(want, static_cast<PlanSum>(found)));
  }
}

// Reordering: every sequence becomes the continuation of its parent, all at once.
enum Role : int { kEnds, kStays, kHeir, kCopy };  // an heir takes its parent's row over

struct RolesParams {
  PlanParams plan;
  int* role;
  int* new_len;
  int32_t* saved;  // rows of parents, by parent, as they were
};

__device__ __forceinline__ int rows_of(const PlanParams& p, int s) {
  return static_cast<int>(min(static_cast<int64_t>(max(p.lengths[s], 0)), static_cast<int64_t>(p.max_pages) * p.page_size));
}

// Roles; rows without a child give up their pages, rows that others need are kept.  A
// workgroup a sequence reads all parents (of at most kReorderSeqs, from L2).
constexpr int kReorderSeqs = 65536;

__global__ __launch_bounds__(256) void pages_roles_kernel(RolesParams r) {
  __shared__ int has_child, has_other, first;
  const PlanParams& p = r.plan;
  for (int s = blockIdx.x; s < p.seqs; s += gridDim.x) {
    if (threadIdx.x == 0) {
      has_child = has_other = 0;
      first = p.seqs;
    }
    __syncthreads();
    const int par = parent_of(p.ask, s, p.seqs);
    for (int t = threadIdx.x; t < p.seqs; t += 256) {
      const int q = p.ask[t];
      if (q == s) {
        has_child = 1;
        if (t != s) has_other = 1;
      }
      if (q == par) atomicMin(&first, t == q ? -1 : t);
    }
    __syncthreads();
    const int32_t* row = p.tables + static_cast<int64_t>(s) * p.max_pages;
    const bool keeps = has_child != 0, kept = has_other != 0;
    for (int e = threadIdx.x; e < p.max_pages; e += 256) {
      const int v = row[e];
      if (!keeps && is_page(v, p.num_pages)) atomicSub(&p.refs[v], 1);  // whole numbers: any order
      if (kept) r.saved[static_cast<int64_t>(s) * p.max_pages + e] = v;
    }
    if (threadIdx.x == 0) r.role[s] = par < 0 ? kEnds : par == s ? kStays : first == s ? kHeir : kCopy;
    __syncthreads();
  }
}

// The same by the plan's workgroup, of few sequences and entries: a launch less.  Replays of
// a graph, without and with: 4 sequences of 4 pages 10.7 us, 9.3, 64 of 20 16.8, 15.3, 64 of
// 64 17.0, 17.1, 64 of 128 16.9, 18.8; calls of 4 beams 19.5, 16.3 (the host's time).
constexpr int kOneSeqs = 256, kOneEntries = 4096;

__device__ __forceinline__ void pages_roles(const RolesParams& r) {
  __shared__ int first[kOneSeqs], child[kOneSeqs];  // child: 1 itself, 2 another
  const PlanParams& p = r.plan;
  const int s = threadIdx.x, entries = p.seqs * p.max_pages;
  const int ahead = s < entries ? p.tables[s] : -1;
  const int q = s < p.seqs ? parent_of(p.ask, s, p.seqs) : -1;
  if (s < p.seqs) {
    first[s] = p.seqs;
    child[s] = 0;
  }
  __syncthreads();
  if (q >= 0) {
    atomicOr(&child[q], s == q ? 1 : 2);
    atomicMin(&first[q], s == q ? -1 : s);
  }
  __syncthreads();
  if (s < p.seqs) r.role[s] = q < 0 ? kEnds : q == s ? kStays : first[q] == s ? kHeir : kCopy;
  for (int i = s; i < entries; i += kPlanThreads) {
    const int v = i == s ? ahead : p.tables[i], c = child[static_cast<unsigned>(i) / static_cast<unsigned>(p.max_pages)];
    if (c == 0 && is_page(v, p.num_pages)) atomicSub(&p.refs[v], 1);  // whole numbers: any order
    if (c >= 2) r.saved[i] = v;
  }
  __syncthreads();  // (references are read)
}

// Copies of last pages to the lowest free ones, in sequence order.  ONE: the roles too.
template <bool ONE>
__global__ __launch_bounds__(kPlanThreads) void pages_reorder_plan_kernel(RolesParams r) {
  __shared__ int lds[kPlanWaves], sums[kPlanWaves];
  if constexpr (ONE) pages_roles(r);
  const PlanParams& p = r.plan;
  int want = 0;  // (at most one page a sequence)
  for (int s0 = 0; s0 < p.seqs; s0 += kPlanThreads) {
    const int s = s0 + threadIdx.x;
    int need = -1;
    if (s < p.seqs) {
      const int role = r.role[s];
      if (role != kEnds) {
        const int par = p.ask[s], n = rows_of(p, par);
        need = role == kCopy && n % p.page_size != 0 &&
               is_page(p.tables[static_cast<int64_t>(par) * p.max_pages + n / p.page_size], p.num_pages);
        r.new_len[s] = n;
      }
      p.w.need[s] = need;
    }
    int total;
    const int b = wg_scan<kPlanThreads>(max(need, 0), sums, total);
    if (s < p.seqs) p.w.before[s] = plan_before(static_cast<PlanSum>(want) + b, p.num_pages);
    want += total;
  }
  const int found = free_pages(p.refs, p.num_pages, min(want, p.num_pages), p.w.list, lds);
  __syncthreads();
  for (int s = threadIdx.x; s < p.seqs; s += kPlanThreads) {
    const int need = p.w.need[s], before = p.w.before[s];
    const bool ok = plan_grants(need, before, found);
    p.granted[s] = ok;
    if (!ok) {
      r.role[s] = kEnds;
    } else if (need > 0) {
      const int par = p.ask[s], dst = p.w.list[before];
      p.w.jobs[before] = int2{p.tables[static_cast<int64_t>(par) * p.max_pages + r.new_len[s] / p.page_size], dst};
      p.refs[dst] = 1;
    }
  }
  if (threadIdx.x == 0) *p.w.n_jobs = min(want, found);
}

struct CompactParams {
  const int32_t* refs;
  int32_t* refs_out;
  int32_t* live_out;
  int num_pages;
  PlanWs w;
};

__global__ __launch_bounds__(kPlanThreads) void pages_compact_plan_kernel(CompactParams p) {
  __shared__ int lds[kPlanWaves];
  int mine = 0, live;
  for (int i = threadIdx.x; i < p.num_pages; i += kPlanThreads) mine += p.refs[i] > 0;
  wg_scan<kPlanThreads>(mine, lds, live);
  int* hole = p.w.list;
  int n_hole = 0, n_move = 0;
  for (int p0 = 0; p0 < p.num_pages; p0 += kScanTile) {  // uniform
    const int q = p0 + kScanPer * threadIdx.x;
    int kind[kScanPer];  // 1: a free place in front, 1 << 16: a page to move, 0: neither
    int n = 0;
#pragma unroll
    for (int i = 0; i < kScanPer; ++i) {
      const bool in = q + i < p.num_pages;
      const bool used = in && p.refs[q + i] > 0;
      kind[i] = !in || used == (q + i < live) ? 0 : (used ? 1 << 16 : 1);
      if (in) p.w.map[q + i] = used ? q + i : -1;
      n += kind[i];
    }
    int total;
    const int b = wg_scan<kPlanThreads>(n, lds, total);
    int h = n_hole + (b & 0xFFFF), m = n_move + (b >> 16);
#pragma unroll
    for (int i = 0; i < kScanPer; ++i) {
      if (kind[i] == 1) hole[h++] = q + i;
      else if (kind[i] != 0) p.w.jobs[m++].x = q + i;
    }
    n_hole += total & 0xFFFF;
    n_move += total >> 16;
  }
  __syncthreads();
  // as many places as movers: live pages in all, `live` places in front
  for (int k = threadIdx.x; k < n_move; k += kPlanThreads) {
    const int src = p.w.jobs[k].x, dst = hole[k];
    p.w.jobs[k].y = dst;
    p.w.map[src] = dst;
    p.w.aux[k] = p.refs[src];
  }
  __syncthreads();  // refs_out may be refs
  for (int i = threadIdx.x; i < p.num_pages; i += kPlanThreads) {
    const int r = p.refs[i];
    p.refs_out[i] = i < live && r > 0 ? r : 0;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < n_move; k += kPlanThreads) p.refs_out[hole[k]] = p.w.aux[k];
  if (threadIdx.x == 0) {
    *p.w.n_jobs = n_move;
    *p.live_out = live;
  }
}

// Page tensors as bytes, and what an application does beside the copies.
struct ApplyParams {
  char* base[6];
  int64_t bytes[6];   // of one page of one layer
  int units[6];       // kCopyUnit parts of it
  int layers, num_pages;
  const int* n_jobs;  // device count of jobs; else n, and the pairs src, dst
  const int2* jobs;
  const int32_t* src;
  const int32_t* dst;
  int n;
  // fork: rows to write; compact: entries to map
  int32_t* tables;
  const int32_t* tables_in;
  int32_t* refs;
  int32_t* lengths;
  const int32_t* parents;
  const int32_t* granted;
  const int* need;
  const int* before;
  const int* list;
  const int* map;
  const int* role;  // reorder
  const int* new_len;
  int seqs, max_pages, page_size;
};

constexpr int kCopyUnit = 16384;  // bytes a workgroup copies at a time

enum class Apply { copy, fork, compact, reorder };

// What bounds it: HBM, as a copy; a workgroup moves 16 KB at a time, four 16-byte
// loads a lane in flight, and takes units at the grid's stride, so that the
// count of jobs may stay on the device.  56 forks' last pages, 8 layers of 16 heads
// of D 256 (264 MB with what free and lookup move): 39 us; 460 MB of a compaction 96
// us, at the rate of a large copy (4.8 TB/s).
template <Apply KIND>
__global__ __launch_bounds__(256) void pages_apply_kernel(ApplyParams p) {
  if constexpr (KIND == Apply::fork) {
    for (int s = blockIdx.x; s < p.seqs; s += gridDim.x) {
      if (p.granted[s] == 0) continue;
      const int par = p.parents[s];
      const int n = static_cast<int>(min(static_cast<int64_t>(max(p.lengths[par], 0)), static_cast<int64_t>(p.max_pages) * p.page_size));
      const int full = n / p.page_size;
      const bool part = p.need[s] > 0;
      const int32_t* from = p.tables + static_cast<int64_t>(par) * p.max_pages;
      int32_t* to = p.tables + static_cast<int64_t>(s) * p.max_pages;
      for (int e = threadIdx.x; e < p.max_pages; e += 256) {
        int v = -1;
        if (e < full) {
          v = from[e];
          if (is_page(v, p.num_pages)) atomicAdd(&p.refs[v], 1);  // whole numbers: any order
        } else if (e == full && part) {
          v = p.list[p.before[s]];
        }
        to[e] = v;
      }
      if (threadIdx.x == 0) p.lengths[s] = n;
    }
  }
  if constexpr (KIND == Apply::reorder) {
    for (int s = blockIdx.x; s < p.seqs; s += gridDim.x) {
      const int role = p.role[s];
      if (role == kStays) continue;
      const int n = role == kEnds ? 0 : p.new_len[s], full = n / p.page_size;
      const bool part = role == kCopy && p.need[s] > 0;
      const int32_t* from = role == kEnds ? nullptr : p.tables_in + static_cast<int64_t>(p.parents[s]) * p.max_pages;
      int32_t* to = p.tables + static_cast<int64_t>(s) * p.max_pages;
      for (int e = threadIdx.x; e < p.max_pages; e += 256) {
        int v = -1;
        if (role == kHeir) {
          v = from[e];
        } else if (role == kCopy && e < full) {
          v = from[e];
          if (is_page(v, p.num_pages)) atomicAdd(&p.refs[v], 1);  // whole numbers: any order
        } else if (part && e == full) {
          v = p.list[p.before[s]];
        }
        to[e] = v;
      }
      if (threadIdx.x == 0) p.lengths[s] = n;
    }
  }
  if constexpr (KIND == Apply::compact) {
    const int64_t n = static_cast<int64_t>(p.seqs) * p.max_pages;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
      const int v = p.tables_in[i];
      p.tables[i] = is_page(v, p.num_pages) ? p.map[v] : v;
    }
  }
  const int n_jobs = KIND == Apply::copy ? p.n : *p.n_jobs;
  int upp = 0;  // units of a page of one layer
#pragma unroll
  for (int a = 0; a < 6; ++a) upp += p.units[a];
  const int64_t total = static_cast<int64_t>(n_jobs) * p.layers * upp;
  for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
    const int64_t jl = w / upp;
    int u = static_cast<int>(w - jl * upp);
    const int job = static_cast<int>(jl / p.layers), layer = static_cast<int>(jl - static_cast<int64_t>(job) * p.layers);
    int src, dst;
    if constexpr (KIND == Apply::copy) {
      src = p.src[job];
      dst = p.dst[job];
      if (!is_page(src, p.num_pages) || !is_page(dst, p.num_pages) || src == dst) continue;
    } else {
      src = p.jobs[job].x;
      dst = p.jobs[job].y;
    }
    char* base = p.base[0];
    int64_t bytes = p.bytes[0];
    int units = p.units[0];
#pragma unroll
    for (int a = 1; a < 6; ++a) {
      if (u >= units) {
        u -= units;
        base = p.base[a];
        bytes = p.bytes[a];
        units = p.units[a];
      } else {
        break;
      }
    }
    const int64_t at = static_cast<int64_t>(u) * kCopyUnit;
    const int n16 = static_cast<int>(min(static_cast<int64_t>(kCopyUnit), bytes - at) / 16);
    const int64_t row = static_cast<int64_t>(layer) * p.num_pages;
    const uint4* from = reinterpret_cast<const uint4*>(base + (row + src) * bytes + at);
    uint4* to = reinterpret_cast<uint4*>(base + (row + dst) * bytes + at);
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (threadIdx.x + 256 * i < static_cast<unsigned>(n16)) v[i] = from[threadIdx.x + 256 * i];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (threadIdx.x + 256 * i < static_cast<unsigned>(n16)) to[threadIdx.x + 256 * i] = v[i];
  }
}

// Frees (EVICT false) or evicts (true) the pages of sequences: one thread an entry.
template <bool EVICT>
__global__ __launch_bounds__(256) void pages_free_kernel(int32_t* tables, int32_t* refs, int32_t* lengths,
                                                         const int32_t* which, int64_t entries, int max_pages,
                                                         int num_pages, int page_size, int window, int sinks) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= entries) return;
  const int s = static_cast<int>(i / max_pages), e = static_cast<int>(i - static_cast<int64_t>(s) * max_pages);
  if (which != nullptr && which[s] == 0) return;
  if constexpr (EVICT) {
    const int64_t r0 = static_cast<int64_t>(e) * page_size;
    if (r0 < sinks || r0 + page_size > static_cast<int64_t>(lengths[s]) - window) return;
  }
  const int v = tables[i];
  if (is_page(v, num_pages)) atomicSub(&refs[v], 1);  // whole numbers: any order
  tables[i] = -1;
  if constexpr (!EVICT) {
    if (e == 0) lengths[s] = 0;
  }
}

// Lengths of sequences whose new rows have pages, a group of lanes a sequence.  One
// chain of loads (length, entry) bounds it.
__global__ __launch_bounds__(256) void pages_advance_kernel(const int32_t* tables, int32_t* lengths, const int32_t* n_new,
                                                            int32_t* advanced, int seqs, int max_pages, int num_pages,
                                                            int page_size) {
  const int lane = threadIdx.x % kPlanGroup;
  const int s = static_cast<int>((static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / kPlanGroup);
  if (s >= seqs) return;  // whole groups
  const int64_t own = lengths[s], k = n_new[s];
  const int64_t n = max(own, int64_t{0}), e1 = (n + k + page_size - 1) / page_size;
  bool ok = k > 0 && e1 <= max_pages;
  if (ok) {
    const int32_t* row = tables + static_cast<int64_t>(s) * max_pages;
    bool lacks = false;
#pragma unroll 4
    for (int64_t e = n / page_size + lane; e < e1; e += kPlanGroup) lacks |= !is_page(row[e], num_pages);
    ok = group_ballot(lacks) == 0;
  }
  if (lane == 0) {
    if (ok) lengths[s] = static_cast<int>(n + k);
    else if (k < 0) lengths[s] = static_cast<int>(max(own + k, int64_t{0}));
    advanced[s] = ok;
  }
}

int check_tables(int num_seqs, int max_pages, int num_pages, int page_size, const char* fn) {
  if (int r = check_paging(page_size, num_pages, max_pages, fn)) return r;
  TQ_CHECK_ARG(num_seqs >= 0 && num_seqs <= (1 << 20), "%s: num_seqs must be 0 to 2^20", fn);
  TQ_CHECK_ARG(static_cast<int64_t>(num_seqs) * max_pages < (int64_t{1} << 38), "%s: block_tables too large", fn);
  return TQ_OK;
}

int check_plan_ws(const void* ws, size_t bytes, int num_seqs, int num_pages, const char* fn) {
  const size_t need = tq_kv_pages_workspace_size(num_seqs, num_pages);
  if (!ws || bytes < need) {
    set_error("%s: workspace of %zu bytes needed (got %zu)", fn, need, ws ? bytes : size_t{0});
    return TQ_ERR_WORKSPACE;
  }
  TQ_CHECK_ARG(reinterpret_cast<uintptr_t>(ws) % 16 == 0, "%s: workspace must be 16-byte aligned", fn);
  return TQ_OK;
}

int set_pages(ApplyParams& a, void* const* pages, int sb_dtype, int num_layers, int num_kv_heads, int head_dim,
              int num_pages, int page_size, const char* fn) {
  TQ_CHECK_ARG(sb_dtype == TQ_F16 || sb_dtype == TQ_F32, "%s: sb_dtype must be f16 or f32", fn);
  TQ_CHECK_ARG(num_layers >= 1 && num_layers <= 65536 && num_kv_heads >= 1 && num_kv_heads <= 65535, "%s: bad num_layers or num_kv_heads", fn);
  TQ_CHECK_ARG(head_dim > 0 && head_dim % 64 == 0 && head_dim <= 4096, "%s: head_dim must be a multiple of 64 <= 4096", fn);
  TQ_CHECK_ARG(pages != nullptr, "%s: null pages", fn);
  const int64_t rows = static_cast<int64_t>(num_kv_heads) * page_size;
  for (int i = 0; i < 6; ++i) {
    TQ_CHECK_ARG(pages[i] != nullptr, "%s: null page tensor", fn);
    TQ_CHECK_ARG(reinterpret_cast<uintptr_t>(pages[i]) % 16 == 0, "%s: page tensors must be 16-byte aligned", fn);
    a.base[i] = static_cast<char*>(pages[i]);
    a.bytes[i] = rows * (i % 3 == 0 ? head_dim / 2 : head_dim / 64 * static_cast<int64_t>(dtype_size(sb_dtype)));
    const int64_t units = (a.bytes[i] + kCopyUnit - 1) / kCopyUnit;
    TQ_CHECK_ARG(units <= (1 << 24), "%s: page too large", fn);
    a.units[i] = static_cast<int>(units);
  }
  a.layers = num_layers;
  a.num_pages = num_pages;
  return TQ_OK;
}

// Workgroups of an application of at most `jobs` copies: eight a CU hold all
// of its waves (units beyond are taken at the grid's stride).
unsigned apply_grid(const ApplyParams& a, int64_t jobs) {
  int64_t upp = 0;
  for (int i = 0; i < 6; ++i) upp += a.units[i];
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(jobs * a.layers * upp, 2048)));
}

}  // namespace
}  // namespace tq

using namespace tq;

extern "C" size_t tq_kv_pages_workspace_size(int num_seqs, int num_pages) {
  if (num_seqs < 0 || num_pages < 1) return 0;
  return sizeof(int) * ((plan_ints(num_seqs, num_pages) + 3) / 4 * 4);
}

extern "C" int tq_kv_pages_reserve(int32_t* block_tables, int32_t* refs, const int32_t* lengths,
                                   const int32_t* n_new, int32_t* granted, int num_seqs, int max_pages,
                                   int num_pages, int page_size, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  clear_error();
  const char* fn = "tq_kv_pages_reserve";
  if (int r = check_tables(num_seqs, max_pages, num_pages, page_size, fn)) return r;
  if (num_seqs == 0) return TQ_OK;
  TQ_CHECK_ARG(block_tables && refs && lengths && n_new && granted, "%s: null pointer", fn);
  if (int r = check_plan_ws(workspace, workspace_bytes, num_seqs, num_pages, fn)) return r;
  PlanParams p{block_tables, refs, const_cast<int32_t*>(lengths), n_new, granted, num_seqs, max_pages, num_pages,
               page_size, plan_ws(workspace, num_seqs, num_pages)};
  pages_plan_kernel<false><<<1, kPlanThreads, 0, static_cast<hipStream_t>(stream)>>>(p);
  TQ_CHECK_LAUNCH("pages_plan_kernel");
  return TQ_OK;
}

extern "C" int tq_kv_pages_fork(void* const* pages, tq_dtype sb_dtype, int num_layers, int num_kv_heads,
                                int head_dim, int32_t* block_tables, int32_t* refs, int32_t* lengths,
                                const int32_t* parents, int32_t* granted, int num_seqs, int max_pages,
                                int num_pages, int page_size, void* workspace, size_t workspace_bytes,
                                void* stream) {
  clear_error();
  const char* fn = "tq_kv_pages_fork";
  if (int r = check_tables(num_seqs, max_pages, num_pages, page_size, fn)) return r;
  ApplyParams a{};
  if (int r = set_pages(a, pages, sb_dtype, num_layers, num_kv_heads, head_dim, num_pages, page_size, fn)) return r;
  if (num_seqs == 0) return TQ_OK;
  TQ_CHECK_ARG(block_tables && refs && lengths && parents && granted, "%s: null pointer", fn);
  if (int r = check_plan_ws(workspace, workspace_bytes, num_seqs, num_pages, fn)) return r;
  hipStream_t s = static_cast<hipStream_t>(stream);
  PlanParams p{block_tables, refs, lengths, parents, granted, num_seqs, max_pages, num_pages, page_size,
               plan_ws(workspace, num_seqs, num_pages)};
  pages_plan_kernel<true><<<1, kPlanThreads, 0, s>>>(p);
  TQ_CHECK_LAUNCH("pages_plan_kernel");
  a.n_jobs = p.w.n_jobs;
  a.jobs = p.w.jobs;
  a.tables = block_tables;
  a.refs = refs;
  a.lengths = lengths;
  a.parents = parents;
  a.granted = granted;
  a.need = p.w.need;
  a.before = p.w.before;
  a.list = p.w.list;
  a.seqs = num_seqs;
  a.max_pages = max_pages;
  a.page_size = page_size;
  pages_apply_kernel<Apply::fork><<<apply_grid(a, std::min(num_seqs, num_pages)), 256, 0, s>>>(a);
  TQ_CHECK_LAUNCH("pages_apply_kernel");
  return TQ_OK;
}

namespace {
// Workspace of a reordering: a plan's, roles and new lengths, and the saved rows.
size_t reorder_ints(int64_t seqs, int64_t pages, int64_t max_pages) {
  return plan_ints(seqs, pages) + 2 * seqs + seqs * max_pages;
}
}  // namespace

extern "C" size_t tq_kv_pages_reorder_workspace_size(int num_seqs, int num_pages, int max_pages) {
  if (num_seqs < 0 || num_pages < 1 || max_pages < 1) return 0;
  return sizeof(int) * ((reorder_ints(num_seqs, num_pages, max_pages) + 3) / 4 * 4);
}

extern "C" int tq_kv_pages_reorder(void* const* pages, tq_dtype sb_dtype, int num_layers, int num_kv_heads,
                                   int head_dim, int32_t* block_tables, int32_t* refs, int32_t* lengths,
                                   const int32_t* parents, int32_t* granted, int num_seqs, int max_pages,
                                   int num_pages, int page_size, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  clear_error();
  const char* fn = "tq_kv_pages_reorder";
  if (int r = check_tables(num_seqs, max_pages, num_pages, page_size, fn)) return r;
  TQ_CHECK_ARG(num_seqs <= kReorderSeqs, "%s: num_seqs must be 0 to %d", fn, kReorderSeqs);
  ApplyParams a{};
  if (int r = set_pages(a, pages, sb_dtype, num_layers, num_kv_heads, head_dim, num_pages, page_size, fn)) return r;
  if (num_seqs == 0) return TQ_OK;
  TQ_CHECK_ARG(block_tables && refs && lengths && parents && granted, "%s: null pointer", fn);
  const size_t bytes = tq_kv_pages_reorder_workspace_size(num_seqs, num_pages, max_pages);
  if (!workspace || workspace_bytes < bytes) {
    set_error("%s: workspace of %zu bytes needed (got %zu)", fn, bytes, workspace ? workspace_bytes : size_t{0});
    return TQ_ERR_WORKSPACE;
  }
  TQ_CHECK_ARG(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "%s: workspace must be 16-byte aligned", fn);
  hipStream_t s = static_cast<hipStream_t>(stream);
  RolesParams r{};
  r.plan = PlanParams{block_tables, refs, lengths, parents, granted, num_seqs, max_pages, num_pages, page_size,
                      plan_ws(workspace, num_seqs, num_pages)};
  r.role = static_cast<int*>(workspace) + plan_ints(num_seqs, num_pages);
  r.new_len = r.role + num_seqs;
  r.saved = r.new_len + num_seqs;
  if (num_seqs <= kOneSeqs && static_cast<int64_t>(num_seqs) * max_pages <= kOneEntries) {
    pages_reorder_plan_kernel<true><<<1, kPlanThreads, 0, s>>>(r);
  } else {
    pages_roles_kernel<<<static_cast<unsigned>(std::min(num_seqs, 2048)), 256, 0, s>>>(r);
    TQ_CHECK_LAUNCH("pages_roles_kernel");
    pages_reorder_plan_kernel<false><<<1, kPlanThreads, 0, s>>>(r);
  }
  TQ_CHECK_LAUNCH("pages_reorder_plan_kernel");
  a.n_jobs = r.plan.w.n_jobs;
  a.jobs = r.plan.w.jobs;
  a.tables = block_tables;
  a.tables_in = r.saved;
  a.refs = refs;
  a.lengths = lengths;
  a.parents = parents;
  a.need = r.plan.w.need;
  a.before = r.plan.w.before;
  a.list = r.plan.w.list;
  a.role = r.role;
  a.new_len = r.new_len;
  a.seqs = num_seqs;
  a.max_pages = max_pages;
  a.page_size = page_size;
  pages_apply_kernel<Apply::reorder><<<apply_grid(a, std::min(num_seqs, num_pages)), 256, 0, s>>>(a);
  TQ_CHECK_LAUNCH("pages_apply_kernel");
  return TQ_OK;
}

extern "C" int tq_kv_pages_free(int32_t* block_tables, int32_t* refs, int32_t* lengths, const int32_t* which,
                                int num_seqs, int max_pages, int num_pages, void* stream) {
  clear_error();
  const char* fn = "tq_kv_pages_free";
  if (int r = check_tables(num_seqs, max_pages, num_pages, 32, fn)) return r;
  if (num_seqs == 0) return TQ_OK;
  TQ_CHECK_ARG(block_tables && refs && lengths && which, "%s: null pointer", fn);
  const int64_t n = static_cast<int64_t>(num_seqs) * max_pages;
  pages_free_kernel<false><<<static_cast<unsigned>((n + 255) / 256), 256, 0, static_cast<hipStream_t>(stream)>>>(
      block_tables, refs, lengths, which, n, max_pages, num_pages, 32, 0, 0);
  TQ_CHECK_LAUNCH("pages_free_kernel");
  return TQ_OK;
}

extern "C" int tq_kv_pages_evict(int32_t* block_tables, int32_t* refs, const int32_t* lengths,
                                 const int32_t* which, int num_seqs, int max_pages, int num_pages,
                                 int page_size, int sliding_window, int num_sinks, void* stream) {
  clear_error();
  const char* fn = "tq_kv_pages_evict";
  if (int r = check_tables(num_seqs, max_pages, num_pages, page_size, fn)) return r;
  TQ_CHECK_ARG(sliding_window > 0, "%s: sliding_window must be > 0", fn);
  TQ_CHECK_ARG(num_sinks >= 0, "%s: num_sinks must be >= 0", fn);
  if (num_seqs == 0) return TQ_OK;
  TQ_CHECK_ARG(block_tables && refs && lengths, "%s: null pointer", fn);
  const int64_t n = static_cast<int64_t>(num_seqs) * max_pages;
  pages_free_kernel<true><<<static_cast<unsigned>((n + 255) / 256), 256, 0, static_cast<hipStream_t>(stream)>>>(
      block_tables, refs, const_cast<int32_t*>(lengths), which, n, max_pages, num_pages, page_size, sliding_window,
      num_sinks);
  TQ_CHECK_LAUNCH("pages_free_kernel");
  return TQ_OK;
}

extern "C" int tq_kv_pages_advance(const int32_t* block_tables, int32_t* lengths, const int32_t* n_new,
                                   int32_t* advanced, int num_seqs, int max_pages, int num_pages, int page_size,
                                   void* stream) {
  clear_error();
  const char* fn = "tq_kv_pages_advance";
  if (int r = check_tables(num_seqs, max_pages, num_pages, page_size, fn)) return r;
  if (num_seqs == 0) return TQ_OK;
  TQ_CHECK_ARG(block_tables && lengths && n_new && advanced, "%s: null pointer", fn);
  constexpr int kSeqs = 256 / kPlanGroup;
  pages_advance_kernel<<<static_cast<unsigned>((num_seqs + kSeqs - 1) / kSeqs), 256, 0, static_cast<hipStream_t>(stream)>>>(
      block_tables, lengths, n_new, advanced, num_seqs, max_pages, num_pages, page_size);
  TQ_CHECK_LAUNCH("pages_advance_kernel");
  return TQ_OK;
}

extern "C" int tq_kv_pages_compact(void* const* pages, tq_dtype sb_dtype, int num_layers, int num_kv_heads,
                                   int head_dim, const int32_t* block_tables, const int32_t* refs,
                                   int32_t* tables_out, int32_t* refs_out, int32_t* live_out, int num_seqs,
                                   int max_pages, int num_pages, int page_size, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  clear_error();
  const char* fn = "tq_kv_pages_compact";
  if (int r = check_tables(num_seqs, max_pages, num_pages, page_size, fn)) return r;
  ApplyParams a{};
  if (int r = set_pages(a, pages, sb_dtype, num_layers, num_kv_heads, head_dim, num_pages, page_size, fn)) return r;
  TQ_CHECK_ARG((num_seqs == 0 || (block_tables && tables_out)) && refs && refs_out && live_out, "%s: null pointer", fn);
  if (int r = check_plan_ws(workspace, workspace_bytes, num_seqs, num_pages, fn)) return r;
  hipStream_t s = static_cast<hipStream_t>(stream);
  CompactParams p{refs, refs_out, live_out, num_pages, plan_ws(workspace, num_seqs, num_pages)};
  pages_compact_plan_kernel<<<1, kPlanThreads, 0, s>>>(p);
  TQ_CHECK_LAUNCH("pages_compact_plan_kernel");
  a.n_jobs = p.w.n_jobs;
  a.jobs = p.w.jobs;
  a.tables = tables_out;
  a.tables_in = block_tables;
  a.map = p.w.map;
  a.seqs = num_seqs;
  a.max_pages = max_pages;
  pages_apply_kernel<Apply::compact><<<apply_grid(a, num_pages / 2 + 1), 256, 0, s>>>(a);
  TQ_CHECK_LAUNCH("pages_apply_kernel");
  return TQ_OK;
}

extern "C" int tq_kv_pages_copy(void* const* pages, tq_dtype sb_dtype, int num_layers, int num_kv_heads,
                                int head_dim, int num_pages, int page_size, const int32_t* src,
                                const int32_t* dst, int n, void* stream) {
  clear_error();
  const char* fn = "tq_kv_pages_copy";
  if (int r = check_tables(0, 1, num_pages, page_size, fn)) return r;
  ApplyParams a{};
  if (int r = set_pages(a, pages, sb_dtype, num_layers, num_kv_heads, head_dim, num_pages, page_size, fn)) return r;
  TQ_CHECK_ARG(n >= 0, "%s: n must be >= 0", fn);
  if (n == 0) return TQ_OK;
  TQ_CHECK_ARG(src && dst, "%s: null pointer", fn);
  a.src = src;
  a.dst = dst;
  a.n = n;
  pages_apply_kernel<Apply::copy><<<apply_grid(a, n), 256, 0, static_cast<hipStream_t>(stream)>>>(a);
  TQ_CHECK_LAUNCH("pages_apply_kernel");
  return TQ_OK;
}
