// Beam search: choosing the next beams from the logits, and reordering a contiguous
// int4 cache by the beams chosen (paged caches: tq_pages.hip).
#include "tq_internal.h"

#include <math.h>

#include <algorithm>
#include <cfloat>

namespace tq {
namespace {

// ---- choosing the next beams ------------------------------------------------
// total(w, t) = score[w] + x[w][t] - log sum_t' exp x[w][t'], and of a group's W V
// totals the K largest, the lowest (w, t) first among equals.
//
// One pass over the logits leaves the largest of every segment of kSeg tokens and the sum
// of exponentials of every kScanWaves segments.  An element of the K best lies in one of
// the K segments whose largest totals come first in the same order (the largest of K
// segments before its own would all come before it), so that the second kernel reads K
// segments again and nothing else: the work does not depend on the values, and no
// candidate list is kept while streaming.  Totals are compared in 64 bits: beams are told
// apart by scores of any distance, and equal ones have to be equal.
constexpr int kSeg = 1024;
constexpr int kScanWaves = 4;  // segments of a workgroup
constexpr int kMaxBeams = 64;

// Of kScanWaves segments: their largest logit, and their exponentials as sum exp(ref).
struct ScanSum {
  float most, ref;
  double sum;
};

// v's exponentials less a logit m, which none of the row's is above.
__device__ __forceinline__ double exp_from(const ScanSum& v, float m) {
  return v.sum == 0.0 ? 0.0 : v.sum * (v.ref == m ? 1.0 : exp(static_cast<double>(v.ref) - static_cast<double>(m)));
}

struct SelectParams {
  const void* x;
  int64_t group_stride, beam_stride;  // elements
  const float* scores;
  const uint8_t* finished;
  int groups, beams, vocab, num_out, pad;
  int nseg, nsum;  // segments of a row, and sums
  ScanSum* sum;    // [groups * beams][nsum]
  float* seg;      // [groups * beams][nseg]: largest
  float* scores_out;
  int32_t* parents_out;
  int32_t* tokens_out;
};

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<_Float16>(_Float16 v) { return static_cast<float>(v); }
template <>
__device__ __forceinline__ float to_f32<uint16_t>(uint16_t v) { return bf16_to_f32(v); }

// Whether a beam has candidates of its own (a score of -inf or NaN has none), and
// whether it is finished: one candidate, the beam itself.
__device__ __forceinline__ bool beam_alive(float score) { return score > -INFINITY; }

// log2(e) in two parts, 2^-49 of it apart.
constexpr float kLog2eHi = 1.4426950216293335f, kLog2eLo = 1.925963033500011e-8f;

template <int CTRL>
__device__ __forceinline__ double dpp_add(double v) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v));
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, 0xF, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, 0xF, 0xF, false);
  return v + __longlong_as_double(static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo));
}
// group_sum<64> in 64 bits.
__device__ __forceinline__ double sum_of_wave(double v) {
  v = dpp_add<0xB1>(v);
  v = dpp_add<0x4E>(v);
  v = dpp_add<0x141>(v);
  v = dpp_add<0x140>(v);
  const auto pair = [](uint32_t hi, uint32_t lo) { return __longlong_as_double(static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo)); };
  uint64_t u = static_cast<uint64_t>(__double_as_longlong(v));
  const auto l16 = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(u), static_cast<uint32_t>(u), false, false);
  const auto h16 = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(u >> 32), static_cast<uint32_t>(u >> 32), false, false);
  v = pair(h16[0], l16[0]) + pair(h16[1], l16[1]);
  u = static_cast<uint64_t>(__double_as_longlong(v));
  const auto l32 = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(u), static_cast<uint32_t>(u), false, false);
  const auto h32 = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(u >> 32), static_cast<uint32_t>(u >> 32), false, false);
  return pair(h32[0], l32[0]) + pair(h32[1], l32[1]);
}

// The sum of N exponentials: exp x = 2^a (1 + r ln 2), a = x log2 e rounded, r what is left of
// it, which two fmas find; the corrections are summed by themselves.  (With a alone all equal
// logits err alike, by 2^-21 or 2^-20: sums were off by up to 0.9e-6.)  Terms are added in
// pairs, so that equal ones add up exactly.  Off by 2^-23 (the power, an ulp) + 4 2^-24 =
// 3.6e-7 of itself at most.
template <int N>
__device__ __forceinline__ double sum_of_exps(const float (&x)[N]) {
  float e[N], c = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float a = x[i] * kLog2eHi, r = fmaf(x[i], kLog2eLo, fmaf(x[i], kLog2eHi, -a));
    e[i] = fast_exp2(a);
    c = fmaf(e[i], r, c);
  }
#pragma unroll
  for (int d = 1; d < N; d *= 2)
#pragma unroll
    for (int i = 0; i < N; i += 2 * d) e[i] += e[i + d];
  return fma(static_cast<double>(c), 0.69314718055994531, static_cast<double>(e[0]));
}

// A wave a segment (behind the row's end: an empty one).  16-byte loads at the alignment
// of an element: what a lane sums goes by the place in the row alone, so that equal rows
// give equal sums.  Logits of ordinary size are taken as they are (ref 0), so that segments
// add up without a common reference.  More than a lane's 16 terms are added in 64 bits.
//
// What bounds it: VALU (87%) beside HBM (248 rows of 262,144 bf16 tokens 30 us, 4.3 TB/s, where
// a large copy reaches 5.1; 28 without the corrections, 35 with the exponent split off by
// adding 1.5 2^23 and one reference for four segments).
template <typename T>
__global__ __launch_bounds__(64 * kScanWaves) void beam_scan_kernel(SelectParams p) {
  constexpr int E = 16 / sizeof(T), NV = kSeg / (64 * E);
  __shared__ ScanSum part[kScanWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = static_cast<int>(blockIdx.x / static_cast<uint32_t>(p.nsum));
  const int js = static_cast<int>(blockIdx.x) - row * p.nsum, j = js * kScanWaves + wave;
  if (!beam_alive(p.scores[row]) || (p.finished && p.finished[row])) return;  // (nobody reads its segments)
  const int b = row / p.beams, w = row - b * p.beams;
  const T* x = static_cast<const T*>(p.x) + b * p.group_stride + w * p.beam_stride + static_cast<int64_t>(j) * kSeg;
  const int n = min(p.vocab - j * kSeg, kSeg);
  float v[NV * E];
  if (n == kSeg) {
    T raw[NV][E];
#pragma unroll
    for (int i = 0; i < NV; ++i) __builtin_memcpy(raw[i], x + (64 * i + lane) * E, 16);
#pragma unroll
    for (int i = 0; i < NV * E; ++i) v[i] = to_f32(raw[i / E][i % E]);
  } else {
#pragma unroll
    for (int i = 0; i < NV * E; ++i) {
      const int at = (64 * (i / E) + lane) * E + i % E;
      v[i] = at < n ? to_f32(x[at]) : -INFINITY;
    }
  }
  float m = -INFINITY;  // (fmaxf passes NaN over)
#pragma unroll
  for (int i = 0; i < NV * E; ++i) m = fmaxf(m, v[i]);
  m = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(wave_max_dpp(m))));
  const bool plain = m > -40.0f && m < 80.0f;
  double s = 0.0;
  if (plain) s = sum_of_exps(v);
  if (!plain || __any(!(s < INFINITY))) {  // -inf, the lowest values and NaN leave NaN
    // from the largest (exact where it counts: no logit within 40 of it is nearer to 0 than
    // to it), what is lower by 85 and NaN as 85 lower: nothing; infinities are 0 apart
    const float from = plain ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < NV * E; ++i) v[i] = fmaxf(v[i] == from ? 0.0f : v[i] - from, -85.0f);
    s = m > -INFINITY ? sum_of_exps(v) : 0.0;
  }
  s = sum_of_wave(s);
  if (lane == 0) {
    if (j < p.nseg) p.seg[static_cast<int64_t>(row) * p.nseg + j] = m;
    part[wave] = ScanSum{m, plain || s == 0.0 ? 0.0f : m, s};
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    ScanSum all = part[0];
    bool alike = all.ref == 0.0f;
#pragma unroll
    for (int i = 1; i < kScanWaves; ++i) {
      all.most = fmaxf(all.most, part[i].most);
      all.sum += part[i].sum;
      alike &= part[i].ref == 0.0f;
    }
    if (!alike) {
      all.ref = all.most;
      all.sum = 0.0;
#pragma unroll 1
      for (int i = 0; i < kScanWaves; ++i) all.sum += exp_from(part[i], all.most);
    }
    p.sum[static_cast<int64_t>(row) * p.nsum + js] = all;
  }
}

// A candidate: its total in an order of whole numbers (0: none), and its place.
struct Cand {
  uint64_t k;
  uint32_t i;
};
__device__ __forceinline__ bool before(const Cand& a, const Cand& b) { return a.k > b.k || (a.k == b.k && a.i < b.i); }
__device__ __forceinline__ Cand cand(double total, uint32_t i) {
  const int64_t u = __double_as_longlong(total + 0.0);  // (-0 is 0)
  const uint64_t k = static_cast<uint64_t>(u) ^ (u < 0 ? ~uint64_t{0} : uint64_t{1} << 63);
  return total > -INFINITY ? Cand{k, i} : Cand{0, ~0u};
}
__device__ __forceinline__ double total_of(uint64_t k) {
  return __longlong_as_double(static_cast<int64_t>(k >> 63 ? k ^ (uint64_t{1} << 63) : ~k));
}
__device__ __forceinline__ Cand shfl_xor_c(const Cand& c, int d) {
  const uint32_t lo = shfl_xor_u(static_cast<uint32_t>(c.k), d), hi = shfl_xor_u(static_cast<uint32_t>(c.k >> 32), d);
  return {static_cast<uint64_t>(hi) << 32 | lo, shfl_xor_u(c.i, d)};
}
constexpr int kPick = 1024;         // threads of the choice, and tokens of a segment
constexpr int kGroup = 8;           // threads that offer one total as a bound
constexpr int kGroups = kPick / kGroup;
constexpr int kSurvivors = 2048;
static_assert(kPick == kSeg && kGroups >= kMaxBeams, "choice");

struct PickLds {
  float group[kGroups];
  float bound;
  int count;
  Cand first[kPick / 64];
  Cand kept[kSurvivors];
  Cand out[kMaxBeams];
};

__device__ __forceinline__ float max_of_8(float v) {
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, false)));
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, false)));
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, false)));
}

// The K first of n items into L.out, in order; how many there are.  about(i): an item's
// total in 32 bits, -inf where it is none; exact(i): the candidate.  The K-th largest of
// the groups' largest bounds the K-th of all from below; the few items that reach it,
// less what 32 bits can be off, are compared exactly: each counts those before it.
//
// 32 bits: a total is base + d, d <= 0, each rounded and the sum too, so off by at most
// 2^-24 (|base| + |d| + |total|) <= 2^-23 (|base| + |total|), and |total| is at most the
// larger of |bound| and |base| where it reaches the bound: 2^-22 (2 most + |bound|) for two
// of them, `most` the largest |base|.  Four times that is allowed for.
// A thread's first HELD items are looked at once: about(i, number).
template <int HELD, typename F, typename G>
__device__ __forceinline__ int pick(PickLds& L, int n, int K, float most, F about, G exact) {
  const int tid = threadIdx.x;
  float held[HELD], best = -INFINITY;
#pragma unroll
  for (int i = 0; i < HELD; ++i) held[i] = tid + i * kPick < n ? about(tid + i * kPick, i) : -INFINITY;
#pragma unroll
  for (int i = 0; i < HELD; ++i) best = fmaxf(best, held[i]);
#pragma unroll 4
  for (int i = tid + HELD * kPick; i < n; i += kPick) best = fmaxf(best, about(i, HELD));
  best = max_of_8(best);
  if (tid % kGroup == 0) L.group[tid / kGroup] = best;
  if (tid == 0) {
    L.bound = -INFINITY;
    L.count = 0;
  }
  __syncthreads();
  int r = 0;  // groups above this one's, and (high half) not below it
#pragma unroll
  for (int j = 0; j < kGroups / kGroup; ++j) {
    const float o = L.group[tid % kGroup + kGroup * j];
    r += (o > best ? 1 : 0) + (o >= best ? 1 << 16 : 0);
  }
  r = group_sum_i<kGroup>(r);
  if (tid % kGroup == 0 && (r & 0xFFFF) < K && K <= r >> 16) L.bound = best;  // (one value)
  __syncthreads();
  const float bound = L.bound, cut = bound - 0x1p-20f * (2.0f * most + fabsf(bound));
  const float least = cut == cut ? cut : -INFINITY;
  const auto keep = [&](int i) {
    const Cand c = exact(i);
    if (c.k != 0) {
      const int at = atomicAdd(&L.count, 1);  // (any order: each one's place is counted below)
      if (at < kSurvivors) L.kept[at] = c;
    }
  };
  // (few of them: code that runs once is bound by its fetching, so there is one copy)
  unsigned these = 0;
#pragma unroll
  for (int i = 0; i < HELD; ++i) these |= held[i] > -INFINITY && held[i] >= least ? 1u << i : 0u;
#pragma unroll 1
  for (; these != 0; these &= these - 1) keep(tid + __builtin_ctz(these) * kPick);
#pragma unroll 1
  for (int i = tid + HELD * kPick; i < n; i += kPick) {
    const float v = about(i, HELD);
    if (v > -INFINITY && v >= least) keep(i);
  }
  __syncthreads();
  const int kept = L.count;
  if (kept <= kSurvivors) {
    for (int s = tid; s < kept; s += kPick) {
      const Cand c = L.kept[s];
      int at = 0;
      for (int j = 0; j < kept; ++j) at += before(L.kept[j], c);
      if (at < K) L.out[at] = c;
    }
    __syncthreads();
    return min(kept, K);
  }
  // many equal ones, or all in a few groups: one after the other
  Cand last{~uint64_t{0}, 0};
  for (int k = 0; k < K; ++k) {
    Cand c{0, ~0u};
    for (int i = tid; i < n; i += kPick) {
      const Cand x = exact(i);
      if (before(last, x) && before(x, c)) c = x;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const Cand o = shfl_xor_c(c, d);
      if (before(o, c)) c = o;
    }
    if ((tid & 63) == 0) L.first[tid >> 6] = c;
    __syncthreads();
    for (int j = 0; j < kPick / 64; ++j)
      if (before(L.first[j], c)) c = L.first[j];
    if (tid == 0) L.out[k] = c;
    last = c;
    __syncthreads();
  }
  return K;
}

// The choice of one group.  What bounds it: latency (a round trip to the segments'
// statistics, one to the chosen segments, and the barriers of two choices): 8 us of 4
// beams of 32,000 tokens, 10.7 of 32 groups of 8 beams of 262,144, 13.7 with 10 places.
// HELD: chosen segments that a thread holds its tokens of.
template <typename T, int HELD>
__global__ __launch_bounds__(kPick) void beam_pick_kernel(SelectParams p) {
  __shared__ PickLds L;
  __shared__ double base[kMaxBeams];  // score - log of the sum of exp(x - most)
  __shared__ float most[kMaxBeams];   // the beam's largest logit (finished: 0)
  __shared__ int state[kMaxBeams];    // 0: no candidates, 1: alive, 2: finished
  __shared__ int2 chosen[kMaxBeams];  // segments: beam, first token
  const int b = blockIdx.x, W = p.beams, V = p.vocab, K = p.num_out, nseg = p.nseg;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float* seg = p.seg + static_cast<int64_t>(b) * W * nseg;
  // (what the first choice looks at, on its way from the start)
  constexpr int kSegs = 2;
  float ahead[kSegs];
#pragma unroll
  for (int i = 0; i < kSegs; ++i) ahead[i] = seg[min(static_cast<int>(threadIdx.x) + i * kPick, W * nseg - 1)];
#pragma unroll 1
  for (int w = wave; w < W; w += kPick / 64) {
    const ScanSum* sum = p.sum + static_cast<int64_t>(b * W + w) * p.nsum;
    const ScanSum mine = lane < p.nsum ? sum[lane] : ScanSum{-INFINITY, 0.0f, 0.0};  // (unwritten where nobody needs it)
    const float score = p.scores[b * W + w];
    const bool done = p.finished && p.finished[b * W + w];
    const int st = !beam_alive(score) ? 0 : done ? 2 : 1;
    double c = score;
    float m = -INFINITY;
    if (st == 1) {
      m = mine.most;
#pragma unroll 1
      for (int j = lane + 64; j < p.nsum; j += 64) m = fmaxf(m, sum[j].most);
      m = wave_max_dpp(m);
      double s = 0.0;
#pragma unroll 1
      for (int j = lane; j < p.nsum; j += 64) s += exp_from(j == lane ? mine : sum[j], m);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d, 64);
      c -= log(s);
    }
    if (lane == 0) {
      base[w] = c;
      most[w] = st == 2 ? 0.0f : m;
      state[w] = st == 1 && !(m > -INFINITY) ? 0 : st;
    }
  }
  __syncthreads();
  const auto total = [&](int w, float x) {
    return base[w] + (x == most[w] ? 0.0 : static_cast<double>(x) - static_cast<double>(most[w]));
  };
  // (what 32 bits cannot hold is not lost: it counts as their lowest value)
  const auto about = [&](int w, float x) {
    const float d = x == most[w] ? 0.0f : fmaxf(x - most[w], -FLT_MAX);
    return x > -INFINITY ? fmaxf(static_cast<float>(base[w]) + d, -FLT_MAX) : -INFINITY;
  };
  // the largest |base| (of at most 64 beams)
  const float far = wave_max_dpp(lane < W && state[lane] != 0 ? fabsf(static_cast<float>(base[lane])) : 0.0f);
  // i / nseg: below 64, off by 64 2^-22 at most, and a half is 2^-15 of it at least
  const float inv = 1.0f / static_cast<float>(nseg);
  const auto beam_of = [&](int i) { return static_cast<int>((static_cast<float>(i) + 0.5f) * inv); };
  // a segment's total is its largest token's; a finished beam is the first of its segments
  const int n1 = pick<kSegs>(
      L, W * nseg, K, far,
      [&](int i, int r) {
        const int w = beam_of(i);
        const float m = r < kSegs ? ahead[r < kSegs ? r : 0] : seg[i];  // (unwritten where nobody needs it)
        return state[w] == 1 ? about(w, m) : state[w] == 2 && i == w * nseg ? static_cast<float>(base[w]) : -INFINITY;
      },
      [&](int i) {
        const int w = beam_of(i);
        return cand(state[w] == 1 ? total(w, seg[i]) : state[w] == 2 && i == w * nseg ? base[w] : -INFINITY, i);
      });
  if (threadIdx.x < static_cast<unsigned>(n1)) {
    const int i = L.out[threadIdx.x].i, w = beam_of(i);
    chosen[threadIdx.x] = int2{w, (i - w * nseg) * kSeg};
  }
  __syncthreads();
  const T* x = static_cast<const T*>(p.x) + b * p.group_stride;
  const auto logit = [&](int2 c) {  // this thread's of a chosen segment (behind the row's end: the last one)
    return to_f32(x[c.x * p.beam_stride + min(c.y + static_cast<int>(threadIdx.x), V - 1)]);
  };
  const auto value = [&](int2 c, float v) {  // a finished beam is its first token; NaN is none
    const bool in = state[c.x] == 2 ? threadIdx.x == 0 : c.y + static_cast<int>(threadIdx.x) < V && v == v;
    return !in ? -INFINITY : state[c.x] == 2 ? most[c.x] : v;
  };
  // The first HELD chosen segments: what concerns segment r in lane r, the loads all on
  // their way before the first is looked at.
  float held[HELD];
  if (n1 > 0) {
    const int2 c = chosen[min(lane, n1 - 1)];
    const int64_t off = c.x * p.beam_stride + c.y;
    const int lo = static_cast<int>(off), hi = static_cast<int>(off >> 32), left = V - 1 - c.y, fin = state[c.x] == 2;
    const int top = __float_as_int(most[c.x]), from = __float_as_int(static_cast<float>(base[c.x]));
    const auto of = [](int v, int r) { return __builtin_amdgcn_readlane(v, r); };
#pragma unroll
    for (int r = 0; r < HELD; ++r) {
      const int64_t o = static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(of(hi, r))) << 32 | static_cast<uint32_t>(of(lo, r)));
      held[r] = to_f32(x[o + min(static_cast<int>(threadIdx.x), of(left, r))]);
    }
#pragma unroll
    for (int r = 0; r < HELD; ++r) {
      const float m = __int_as_float(of(top, r));
      const bool in = of(fin, r) ? threadIdx.x == 0 : static_cast<int>(threadIdx.x) <= of(left, r);
      const float v = of(fin, r) ? m : held[r];
      const float d = v == m ? 0.0f : fmaxf(v - m, -FLT_MAX);
      held[r] = in && v > -INFINITY ? fmaxf(__int_as_float(of(from, r)) + d, -FLT_MAX) : -INFINITY;
    }
  }
  const int n2 = pick<HELD>(
      L, n1 * kSeg, K, far,
      [&](int i, int r) {
        if (r < HELD) return held[r < HELD ? r : 0];
        const int2 c = chosen[i / kSeg];
        return about(c.x, value(c, logit(c)));
      },
      [&](int i) {
        const int2 c = chosen[i / kSeg];
        const float v = value(c, logit(c));
        return cand(v > -INFINITY ? total(c.x, v) : -INFINITY, c.x * V + (state[c.x] == 2 ? p.pad : c.y + static_cast<int>(threadIdx.x)));
      });
  for (int k = threadIdx.x; k < K; k += kPick) {
    const int64_t at = static_cast<int64_t>(b) * K + k;
    const Cand c = k < n2 ? L.out[k] : Cand{0, 0};
    const int w = static_cast<int>(c.i) / V;
    p.scores_out[at] = k < n2 ? static_cast<float>(total_of(c.k)) : -INFINITY;
    p.parents_out[at] = k < n2 ? b * W + w : -1;
    p.tokens_out[at] = k < n2 ? static_cast<int>(c.i) - w * V : -1;
  }
}

template <typename T>
int launch_select(const SelectParams& p, hipStream_t s) {
  const int64_t sums = static_cast<int64_t>(p.groups) * p.beams * p.nsum;
  beam_scan_kernel<T><<<static_cast<unsigned>(sums), 64 * kScanWaves, 0, s>>>(p);
  TQ_CHECK_LAUNCH("beam_scan_kernel");
  const unsigned groups = static_cast<unsigned>(p.groups);
  if (p.num_out <= 4) beam_pick_kernel<T, 4><<<groups, kPick, 0, s>>>(p);
  else if (p.num_out <= 8) beam_pick_kernel<T, 8><<<groups, kPick, 0, s>>>(p);
  else beam_pick_kernel<T, 16><<<groups, kPick, 0, s>>>(p);
  TQ_CHECK_LAUNCH("beam_pick_kernel");
  return TQ_OK;
}

int segments(int vocab) { return (vocab + kSeg - 1) / kSeg; }
int sums(int vocab) { return (segments(vocab) + kScanWaves - 1) / kScanWaves; }

// ---- reordering a contiguous cache ------------------------------------------
// Rows of sequence b become those of parents[b], in place.  Sequences that are joined by
// the map (a group's beams) are a component; a workgroup takes the same bytes of all
// sequences of one, loads those of every parent before it stores any, and no other
// workgroup touches them, so that any map (swaps, cycles, one parent of many) comes out as
// if all moved at once.  A plan by one workgroup finds the components and the rows each
// moves, so that nothing behind the lengths is visited.
constexpr int kMaxSeqs = 1024;
constexpr int kHeldParents = 8;  // of a component, in a thread's registers; else by way of LDS
constexpr int kUnits = 4;        // 16-byte units of a thread
constexpr int kTileUnits = 256 * kUnits;
constexpr int kLdsUnits = 1024;

struct ReorderComp {
  int from, nf, rows, tiles;  // parents [from, from + nf), the most rows of one, tiles of the components before
};
struct ReorderParent {
  int seq, rows, to, nd;      // its children [to, to + nd)
};

struct ReorderParams {
  char* base[6];
  int row_bytes[6];
  int heads, cap, seqs;
  int32_t* lengths;
  const int32_t* parents;
  int* head;             // components, tiles in all
  ReorderComp* comps;
  ReorderParent* from;
  int* to;
};

// Tiles of one head of n rows, tensor by tensor.
__device__ __forceinline__ int tiles_of(const ReorderParams& p, int a, int n) {
  return static_cast<int>((static_cast<int64_t>(n) * p.row_bytes[a] + 16 * kTileUnits - 1) / (16 * kTileUnits));
}

// One thread a sequence, of N at most; lengths become the parents'.  What bounds it: a
// chain of loads, shared counts and scans; 4 sequences 3.9 us with a wave, 5.7 with sixteen,
// 32 sequences 5.0 and 7.1.
template <int N>
__global__ __launch_bounds__(N) void kv_reorder_plan_kernel(ReorderParams p) {
  __shared__ int label[N], kids[N], nf[N], most[N], at[N], first[N];
  __shared__ int lds[N / 64], changed;
  const int s = threadIdx.x;
  const bool in = s < p.seqs;
  const int q = in ? parent_of(p.parents, s, p.seqs) : -1;
  const int len = in ? p.lengths[s] : 0;
  const int length = q < 0 ? 0 : p.lengths[q];
  const int rows = max(min(len, p.cap), 0);
  label[s] = s;
  kids[s] = nf[s] = most[s] = at[s] = 0;
  __syncthreads();  // (lengths are read)
  if (in) p.lengths[s] = length;
  const bool moves = q >= 0 && q != s;
  if (moves) atomicAdd(&kids[q], 1);
  __syncthreads();
  const bool gives = kids[s] > 0 && rows > 0;
  // components: the lowest number that the map reaches either way
  for (;;) {
    if (s == 0) changed = 0;
    __syncthreads();
    if (moves) {
      const int a = label[s], b = label[q];
      if (a != b) {
        atomicMin(&label[max(a, b)], min(a, b));
        atomicMin(&label[s], min(a, b));
        atomicMin(&label[q], min(a, b));
        changed = 1;
      }
    }
    __syncthreads();
    const int l = label[label[s]];
    __syncthreads();
    atomicMin(&label[s], l);
    const bool done = changed == 0;
    __syncthreads();
    if (done) break;
  }
  const int root = label[s];
  if (gives) {
    atomicAdd(&nf[root], 1);
    atomicMax(&most[root], rows);
  }
  __syncthreads();
  const bool comp = nf[s] > 0;  // of the component's lowest sequence
  int comps, parents, children, tiles;
  const int c = wg_scan<N, int>(comp, lds, comps);
  const int from0 = wg_scan<N>(nf[s], lds, parents);
  const int to0 = wg_scan<N>(gives ? kids[s] : 0, lds, children);
  int n = 0;
#pragma unroll
  for (int a = 0; a < 6; ++a) n += comp ? tiles_of(p, a, most[s]) : 0;
  const int tile0 = wg_scan<N>(n * p.heads, lds, tiles);
  first[s] = from0;
  if (comp) p.comps[c] = ReorderComp{from0, nf[s], most[s], tile0};
  if (s == 0) {
    p.head[0] = comps;
    p.head[1] = tiles;
  }
  __syncthreads();
  // (the order of a component's parents is only that of their loads)
  if (gives) p.from[first[root] + atomicAdd(&at[root], 1)] = ReorderParent{s, rows, to0, kids[s]};
  kids[s] = gives ? to0 : -1;
  __syncthreads();
  if (moves && kids[q] >= 0) p.to[atomicAdd(&kids[q], 1)] = s;
}

__device__ __forceinline__ uint4 load_unit(const char* src, int64_t left) {
  uint4 v{};
  if (left >= 16) {
    __builtin_memcpy(&v, src, 16);
  } else if (left > 0) {  // the last rows end inside: whole elements of two bytes
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (2 * e < left) w[e / 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(src + 2 * e)) << (16 * (e & 1));
    v = uint4{w[0], w[1], w[2], w[3]};
  }
  return v;
}
__device__ __forceinline__ void store_unit(char* dst, const uint4& v, int64_t left) {
  if (left >= 16) {
    __builtin_memcpy(dst, &v, 16);
  } else if (left > 0) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (2 * e < left) *reinterpret_cast<uint16_t*>(dst + 2 * e) = static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)));
  }
}

// What bounds it: HBM.  Up to kHeldParents parents a component a thread holds its units of
// all of them, with no barrier; 16-byte accesses at the alignment of an element.  32
// sequences (8 groups) of 700 to 4,000 rows, 16 heads of D 256, calls: 151 us with one
// unit a thread, 113 with two, 105 with four (this kernel 99, 4.6 TB/s read and written);
// tiles of all sequences through the LDS, shorter chunks by the number of groups, 150.
__global__ __launch_bounds__(256) void kv_reorder_kernel(ReorderParams p) {
  __shared__ uint4 unit[kLdsUnits];
  __shared__ int start[kMaxSeqs / 2];  // tiles of the components before (each has two sequences at least)
  const int comps = p.head[0], total = p.head[1];
  if (static_cast<int>(blockIdx.x) >= total) return;
  for (int i = threadIdx.x; i < comps; i += 256) start[i] = p.comps[i].tiles;
  __syncthreads();
  for (int g = blockIdx.x; g < total; g += gridDim.x) {
    int c = 0;
    for (int end = comps; end - c > 1;) {
      const int mid = (c + end) / 2;
      (start[mid] <= g ? c : end) = mid;
    }
    c = __builtin_amdgcn_readfirstlane(c);
    const ReorderComp k = p.comps[c];
    int tiles[6], per_head = 0;
#pragma unroll
    for (int a = 0; a < 6; ++a) per_head += tiles[a] = tiles_of(p, a, k.rows);
    const int h = (g - k.tiles) / per_head;
    int u = g - k.tiles - h * per_head, a = 0;
#pragma unroll
    for (int i = 0; i < 5; ++i)
      if (a == i && u >= tiles[i]) {
        u -= tiles[i];
        a = i + 1;
      }
    char* base = p.base[0];
    int rb = p.row_bytes[0];
#pragma unroll
    for (int i = 1; i < 6; ++i)
      if (a == i) {
        base = p.base[i];
        rb = p.row_bytes[i];
      }
    const int64_t first = static_cast<int64_t>(u) * (16 * kTileUnits);  // bytes into the head's rows
    const int64_t head = static_cast<int64_t>(p.cap) * rb, stride = p.heads * head;
    base += h * head + first;
    const ReorderParent* from = p.from + k.from;
    const auto left = [&](int rows, int at) { return static_cast<int64_t>(rows) * rb - first - at; };
    if (k.nf <= kHeldParents) {
      uint4 v[kHeldParents][kUnits];
#pragma unroll
      for (int i = 0; i < kHeldParents; ++i)
        if (i < k.nf) {
          const ReorderParent f = from[i];
#pragma unroll
          for (int j = 0; j < kUnits; ++j) {
            const int at = 16 * (threadIdx.x + 256 * j);
            v[i][j] = load_unit(base + f.seq * stride + at, left(f.rows, at));
          }
        }
#pragma unroll
      for (int i = 0; i < kHeldParents; ++i)
        if (i < k.nf) {
          const ReorderParent f = from[i];
          for (int d = 0; d < f.nd; ++d) {
            char* dst = base + p.to[f.to + d] * stride;
#pragma unroll
            for (int j = 0; j < kUnits; ++j) {
              const int at = 16 * (threadIdx.x + 256 * j);
              store_unit(dst + at, v[i][j], left(f.rows, at));
            }
          }
        }
      continue;
    }
    // as many units at a time as the LDS holds of every parent
    const int T = max(kLdsUnits / k.nf, 1);
    for (int u0 = 0; u0 < kTileUnits; u0 += T) {
      for (int i = threadIdx.x; i < T * k.nf; i += 256) {
        const ReorderParent f = from[i / T];
        const int at = 16 * (u0 + i % T);
        if (u0 + i % T < kTileUnits) unit[i] = load_unit(base + f.seq * stride + at, left(f.rows, at));
      }
      __syncthreads();
      for (int i = threadIdx.x; i < T * k.nf; i += 256) {
        const ReorderParent f = from[i / T];
        const int at = 16 * (u0 + i % T);
        if (u0 + i % T < kTileUnits)
          for (int d = 0; d < f.nd; ++d) store_unit(base + p.to[f.to + d] * stride + at, unit[i], left(f.rows, at));
      }
      __syncthreads();
    }
  }
}

}  // namespace
}  // namespace tq

using namespace tq;

extern "C" size_t tq_beam_select_workspace_size(int groups, int beams, int vocab) {
  if (groups < 1 || beams < 1 || vocab < 1) return 0;
  return static_cast<size_t>(groups) * beams * (sizeof(ScanSum) * sums(vocab) + sizeof(float) * segments(vocab));
}

extern "C" int tq_beam_select(const void* logits, tq_dtype x_dtype, int64_t group_stride, int64_t beam_stride,
                              const float* scores, const uint8_t* finished, int groups, int beams, int vocab,
                              int num_out, int pad_token, float* scores_out, int32_t* parents_out,
                              int32_t* tokens_out, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  const char* fn = "tq_beam_select";
  TQ_CHECK_ARG(valid_dtype(x_dtype), "%s: bad x_dtype %d", fn, x_dtype);
  TQ_CHECK_ARG(groups >= 0 && groups <= (1 << 20), "%s: groups must be 0 to 2^20", fn);
  TQ_CHECK_ARG(beams >= 1 && beams <= kMaxBeams, "%s: beams must be 1 to %d (got %d)", fn, kMaxBeams, beams);
  TQ_CHECK_ARG(num_out >= 1 && num_out <= kMaxBeams, "%s: num_out must be 1 to %d (got %d)", fn, kMaxBeams, num_out);
  TQ_CHECK_ARG(vocab >= 1 && vocab <= (1 << 24), "%s: vocab must be 1 to 2^24 (got %d)", fn, vocab);
  TQ_CHECK_ARG(pad_token >= 0 && pad_token < vocab, "%s: pad_token must be a token (got %d)", fn, pad_token);
  if (groups == 0) return TQ_OK;
  TQ_CHECK_ARG(group_stride >= 0 && beam_stride >= 0 && group_stride < (int64_t{1} << 40) && beam_stride < (int64_t{1} << 40), "%s: bad strides", fn);
  TQ_CHECK_ARG(logits && scores && scores_out && parents_out && tokens_out, "%s: null pointer", fn);
  TQ_CHECK_ARG(reinterpret_cast<uintptr_t>(logits) % dtype_size(x_dtype) == 0, "%s: logits must be aligned to their type", fn);
  const size_t need = tq_beam_select_workspace_size(groups, beams, vocab);
  if (!workspace || workspace_bytes < need) {
    set_error("%s: workspace of %zu bytes needed (got %zu)", fn, need, workspace ? workspace_bytes : size_t{0});
    return TQ_ERR_WORKSPACE;
  }
  TQ_CHECK_ARG(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "%s: workspace must be 16-byte aligned", fn);
  const int nseg = segments(vocab);
  // (a launch has fewer than 2^32 threads)
  TQ_CHECK_ARG(static_cast<int64_t>(groups) * beams * sums(vocab) < (int64_t{1} << 32) / (64 * kScanWaves), "%s: logits too large", fn);
  ScanSum* sum = static_cast<ScanSum*>(workspace);
  SelectParams p{logits, group_stride, beam_stride, scores, finished, groups, beams, vocab, num_out, pad_token, nseg,
                 sums(vocab), sum, reinterpret_cast<float*>(sum + static_cast<size_t>(groups) * beams * sums(vocab)),
                 scores_out, parents_out, tokens_out};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (x_dtype == TQ_F32) return launch_select<float>(p, s);
  if (x_dtype == TQ_F16) return launch_select<_Float16>(p, s);
  return launch_select<uint16_t>(p, s);
}

extern "C" size_t tq_kv_reorder_int4_workspace_size(int batch) {
  if (batch < 1 || batch > kMaxSeqs) return 0;
  return 16 + static_cast<size_t>(batch) * (sizeof(ReorderComp) + sizeof(ReorderParent) + sizeof(int));
}

extern "C" int tq_kv_reorder_int4(uint32_t* k_quant, void* k_scales, void* k_biases, uint32_t* v_quant,
                                  void* v_scales, void* v_biases, tq_dtype sb_dtype, int batch, int num_kv_heads,
                                  int head_dim, int kv_capacity, int32_t* lengths, const int32_t* parents,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  const char* fn = "tq_kv_reorder_int4";
  TQ_CHECK_ARG(sb_dtype == TQ_F16 || sb_dtype == TQ_F32, "%s: sb_dtype must be f16 or f32", fn);
  TQ_CHECK_ARG(batch >= 0 && batch <= kMaxSeqs, "%s: batch must be 0 to %d (got %d)", fn, kMaxSeqs, batch);
  TQ_CHECK_ARG(num_kv_heads >= 1 && num_kv_heads <= 65535, "%s: bad num_kv_heads", fn);
  TQ_CHECK_ARG(head_dim > 0 && head_dim % 64 == 0 && head_dim <= 4096, "%s: head_dim must be a multiple of 64 <= 4096", fn);
  TQ_CHECK_ARG(kv_capacity >= 1 && kv_capacity <= (1 << 24), "%s: kv_capacity must be 1 to 2^24", fn);
  if (batch == 0) return TQ_OK;
  ReorderParams p{};
  void* const t[6] = {k_quant, k_scales, k_biases, v_quant, v_scales, v_biases};
  int64_t tiles = 0;
  for (int i = 0; i < 6; ++i) {
    TQ_CHECK_ARG(t[i] != nullptr, "%s: null tensor pointer", fn);
    TQ_CHECK_ARG(reinterpret_cast<uintptr_t>(t[i]) % 4 == 0, "%s: cache tensors must be 4-byte aligned", fn);
    p.base[i] = static_cast<char*>(t[i]);
    p.row_bytes[i] = i % 3 == 0 ? head_dim / 2 : head_dim / 64 * static_cast<int>(dtype_size(sb_dtype));
    tiles += (static_cast<int64_t>(kv_capacity) * p.row_bytes[i] + 16 * kTileUnits - 1) / (16 * kTileUnits);
  }
  tiles *= static_cast<int64_t>(num_kv_heads) * ((batch + 1) / 2);  // (a component has two sequences at least)
  TQ_CHECK_ARG(tiles < (int64_t{1} << 30), "%s: cache too large", fn);
  TQ_CHECK_ARG(lengths && parents, "%s: null pointer", fn);
  const size_t need = tq_kv_reorder_int4_workspace_size(batch);
  if (!workspace || workspace_bytes < need) {
    set_error("%s: workspace of %zu bytes needed (got %zu)", fn, need, workspace ? workspace_bytes : size_t{0});
    return TQ_ERR_WORKSPACE;
  }
  TQ_CHECK_ARG(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "%s: workspace must be 16-byte aligned", fn);
  p.heads = num_kv_heads;
  p.cap = kv_capacity;
  p.seqs = batch;
  p.lengths = lengths;
  p.parents = parents;
  p.head = static_cast<int*>(workspace);
  p.comps = reinterpret_cast<ReorderComp*>(p.head + 4);
  p.from = reinterpret_cast<ReorderParent*>(p.comps + batch);
  p.to = reinterpret_cast<int*>(p.from + batch);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (batch <= 64) kv_reorder_plan_kernel<64><<<1, 64, 0, s>>>(p);
  else kv_reorder_plan_kernel<kMaxSeqs><<<1, kMaxSeqs, 0, s>>>(p);
  TQ_CHECK_LAUNCH("kv_reorder_plan_kernel");
  kv_reorder_kernel<<<static_cast<unsigned>(std::min<int64_t>(tiles, 8192)), 256, 0, s>>>(p);
  TQ_CHECK_LAUNCH("kv_reorder_kernel");
  return TQ_OK;
}
