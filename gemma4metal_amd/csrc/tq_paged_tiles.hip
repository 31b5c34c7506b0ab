// Multi-query attention over pages with K/V tiles shared by a workgroup's 64 or
// 128 (query, head) rows of one kv head: prompts (rows of consecutive queries of one
// sequence), and the shared prefix of a batch (rows of all its sequences).
//
// The mathematics, operand layouts and staging are those of tq_prefill.hip, and
// so is what bounds it (VALU).  What differs:
// - A tile is TK keys at a multiple of TK, one or two 32-row parts of pages;
//   the pool rows of the next 64 parts are held in a wave's lanes.  Tiles
//   between the sinks and the window that no row attends are left out.
// - Rows have limits of their own, [lo, hi) or below the sinks.  In a part of a
//   tile that some row does not attend wholly, V scales and biases of weight 0
//   are taken as 0 (a key that other rows attend may be infinite or NaN); rows
//   that nobody attends are staged with scales and biases of 0.
// - The tiles of a workgroup's rows may be split over workgroups (grid y), which
//   then leave partials (m, l, O).
// - fp32 queries are two fp16 parts, 22 bits, and take two products a k-step.
//   fp32 biases are applied in fp32.
#include "tq_prefill_tile.h"

#include <cfloat>

namespace tq {
namespace {

constexpr int kRs = 4;  // 16-row sets of a tile's geometry (PfGeom): 8 waves

// Pool rows at which the 32-row parts of a run of tiles begin: part h of the run's
// tile i in lane KH i + h, and whether its page exists in that bit of has.
struct PgRun {
  int lo, hi;
  uint64_t has;
};

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

// Raw loads behind a uniform address: a 32-bit lane offset beside the scalar base,
// where global loads of this kernel took 64-bit addresses in vector registers.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t pg_rsrc(const void* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0x7FFFFFFF, 0x00020000);
}

// The tensors a wave stages from: of its words (K or V) per unit, and of its
// scales or biases.
template <class Gm>
struct PgSource {
  const char* w[Gm::NU];
  const char* s[Gm::NSD];
};

template <class Gm>
__device__ __forceinline__ PgSource<Gm> pg_source(const PagedParams& p) {
  PgSource<Gm> r;
#pragma unroll
  for (int i = 0; i < Gm::NU; ++i)
    r.w[i] = reinterpret_cast<const char*>(
        __builtin_amdgcn_readfirstlane((threadIdx.x + i * Gm::NT) / Gm::UNITS) == 0 ? p.kq : p.vq);
#pragma unroll
  for (int i = 0; i < Gm::NSD; ++i) {
    const int a = __builtin_amdgcn_readfirstlane((threadIdx.x + i * Gm::NT) / Gm::SDW);
    r.s[i] = static_cast<const char*>(a == 0 ? p.ks : a == 1 ? p.kb : a == 2 ? p.vs : p.vb);
  }
  return r;
}

// A tile's words and scales into registers.  No load is conditional (the wait for
// one would drain all of them).
template <class Gm>
__device__ __forceinline__ void pg_load(PfRaw<Gm>& R, const PgSource<Gm>& from, const PgRun& run, int i0) {
  constexpr int KH = Gm::KH;
  // (i0: lane of the tile's first part)
  const auto lane_row = [&](int i) {
    return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(run.hi, i))) << 32 |
                                static_cast<uint32_t>(__builtin_amdgcn_readlane(run.lo, i)));
  };
  const int64_t only = KH == 1 ? lane_row(i0) : 0;  // (once, not on every branch)
  const auto base_of = [&](int part) { return KH == 1 ? only : lane_row(i0 + part); };
  // the part of a tile row; the same for a wave's 64 units where those span at
  // most one part
  const auto part = [](int r) { return KH == 1 ? 0 : __builtin_amdgcn_readfirstlane(r >> 5); };
#pragma unroll
  for (int i = 0; i < Gm::NU; ++i) {
    const int e = threadIdx.x + i * Gm::NT;
    const int role = __builtin_amdgcn_readfirstlane(e / Gm::UNITS);
    const int u = e % Gm::UNITS;
    if (role == 0) {
      const int r = u / Gm::NG;
      const int64_t base = base_of(part(r));
      const uint32_t off = (r & 31) * (4 * Gm::W) + 32 * (u % Gm::NG);
      const auto src = pg_rsrc(from.w[i] + base * (4 * Gm::W));
      const u32x4 a = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(src, off, 0, 0));
      const u32x4 b = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(src, off, 16, 0));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        R.w[i][k] = a[k];
        R.w[i][4 + k] = b[k];
      }
    } else {  // (threads past the units load one again and do not store it)
      const int w = u % Gm::W, kc = u / Gm::W;  // kc = 4 part + c
      const int64_t base = base_of(part(8 * kc));
      const uint32_t off = 4 * (kc & 3) * (4 * Gm::W) + 4 * w;
      const auto src = pg_rsrc(from.w[i] + base * (4 * Gm::W));
#pragma unroll
      for (int j = 0; j < 8; ++j)
        R.w[i][j] = __builtin_amdgcn_raw_buffer_load_b32(src, off, (16 * (j >> 2) + (j & 3)) * (4 * Gm::W), 0);
    }
  }
#pragma unroll
  for (int i = 0; i < Gm::NSD; ++i) {
    const int e = threadIdx.x + i * Gm::NT;
    // (threads past the tensors load one again and do not store it)
    const int d = e % Gm::SDW;
    constexpr int DPR = Gm::SDW / Gm::TK;  // dwords a row
    const int r = d / DPR;
    const uint32_t off = (r & 31) * (4 * DPR) + 4 * (d % DPR);
    if constexpr (KH == 2 && DPR == 1) {  // a wave spans both parts
      const int64_t base = r >= 32 ? base_of(KH - 1) : base_of(0);
      R.s[i] = *reinterpret_cast<const uint32_t*>(from.s[i] + base * (4 * DPR) + off);
    } else {
      const int64_t base = base_of(part(r));
      R.s[i] = __builtin_amdgcn_raw_buffer_load_b32(pg_rsrc(from.s[i] + base * (4 * DPR)), off, 0, 0);
    }
  }
}

// Zeroes the scales and biases of rows past every limit and of missing pages,
// which may hold anything.
template <class Gm>
__device__ __forceinline__ void pg_mask(PfRaw<Gm>& R, int key, int has, int hi) {
  if (key <= hi - Gm::TK && has == (1 << Gm::KH) - 1) return;  // uniform, most tiles
#pragma unroll
  for (int i = 0; i < Gm::NSD; ++i) {
    constexpr int DPR = Gm::SDW / Gm::TK;
    const int r = (threadIdx.x + i * Gm::NT) % Gm::SDW / DPR;
    R.s[i] = (has >> (r >> 5) & 1) && key + r < hi ? R.s[i] : 0u;
  }
}

// LDS of a workgroup: the operand images of PfGeom, K scales and biases by key,
// and what the V products take by group: scales and biases (fp32 caches), and the
// rows of the bias products' A operand in fp16 -- bias and scale of a group (fp16
// caches), or high and low parts of both, over 2^e0 (fp32).
template <int D, bool F32>
struct PgStage {
  using Gm = PfGeom<D, F32, kRs>;
  using SB = typename Gm::SB;
  static constexpr int NP = F32 ? 4 : 2;       // fp16 rows of a group
  static constexpr int TKP = Gm::TK + 8;       // (rows apart in the banks)
  u32x4 k[2][2 * Gm::KH * Gm::KU];
  u32x4 v[2][Gm::KH * Gm::VU];
  SB ksb[2][2][Gm::TK * Gm::NG];               // k scale, k bias: [key][group]
  _Float16 vp[2][NP][Gm::NG][TKP];
  float vsb[F32 ? 2 : 1][2][F32 ? Gm::NG : 1][F32 ? Gm::TK + 4 : 4];  // fp32 scale, bias
  _Float16 one[TKP], zero[TKP];
  float zero32[F32 ? Gm::TK : 1];
  v4f xch[Gm::DH == 2 ? Gm::NW : 1][2][64];    // score parts of a row set's waves
};

// Scales and biases from registers into LDS buffer b.
template <int D, bool F32>
__device__ __forceinline__ void pg_store_sb(PgStage<D, F32>& S, const PfRaw<PfGeom<D, F32, kRs>>& R, int b, int e0) {
  using St = PgStage<D, F32>;
  using Gm = typename St::Gm;
  constexpr int DPR = Gm::SDW / Gm::TK;
#pragma unroll
  for (int i = 0; i < Gm::NSD; ++i) {
    const int e = threadIdx.x + i * Gm::NT;
    const int t = __builtin_amdgcn_readfirstlane(e / Gm::SDW), d = e % Gm::SDW;
    const uint32_t a = R.s[i];
    if (t < 2) {
      reinterpret_cast<uint32_t*>(S.ksb[b][t])[d] = a;
    } else if (t < 4) {
      const int key = d / DPR;
      if constexpr (F32) {
        const int g = d % DPR;
        const float x = ldexpf(__uint_as_float(a), -e0);
        uint32_t hb = __builtin_bit_cast(uint16_t, static_cast<_Float16>(x));
        asm("" : "+v"(hb));  // one rounding: the remainder is of the stored part
        const _Float16 h = __builtin_bit_cast(_Float16, static_cast<uint16_t>(hb));
        const int part = t == 2 ? 2 : 0;
        S.vp[b][part][g][key] = h;
        S.vp[b][part + 1][g][key] = static_cast<_Float16>(x - static_cast<float>(h));
        S.vsb[b][t - 2][g][key] = __uint_as_float(a);
      } else {
        const int g = 2 * (d % DPR);
        const v2h h = __builtin_bit_cast(v2h, a);
        S.vp[b][t == 2 ? 1 : 0][g][key] = h[0];
        S.vp[b][t == 2 ? 1 : 0][g + 1][key] = h[1];
      }
    }
  }
}

// Whether a tile's V scales are alike (0, or within 2^-kPfDown .. 2^kPfUp of 2^e0) and
// its V biases of fp16's range (fp32: over 2^e0), per wave that stages some, into
// ok[2 NSW].
template <class Gm>
__device__ __forceinline__ void pg_alike(const PfRaw<Gm>& R, int e0, int* ok) {
  constexpr bool kHalf = sizeof(typename Gm::SB) == 2;
  // the bounds' bit patterns (magnitudes order as these do), of 2^k
  const auto bits = [](int k) -> uint32_t {
    if constexpr (kHalf) return k > 15 ? 0x7C00u : k >= -14 ? (k + 15) << 10 : k >= -24 ? 1u << (k + 24) : 0u;
    else return (k + 127) << 23;
  };
  const uint32_t lo = bits(e0 - kPfDown), n = bits(e0 + kPfUp) - lo;
  const uint32_t big = kHalf ? 0x7C00u : bits(e0 + 15);
#pragma unroll
  for (int i = 0; i < Gm::NSD; ++i) {
    const int e = threadIdx.x + i * Gm::NT;
    const int t = __builtin_amdgcn_readfirstlane(e / Gm::SDW);
    if (t != 2 && t != 3) continue;
    const auto fine = [&](uint32_t a) { return t == 2 ? a - lo < n || a == 0 : a < big; };
    const uint32_t a = R.s[i];
    bool in;
    if constexpr (kHalf) in = fine(a & 0x7FFFu) && fine(a >> 16 & 0x7FFFu);
    else in = fine(a & 0x7FFFFFFFu);
    ok[(t - 2) * Gm::NSW + e % Gm::SDW / 64] = __all(in);  // (one value from every lane)
  }
}

struct TileParams : PagedParams {
  int splits;  // workgroups along the tiles (grid y); 1: write p.out
};

// RS: 16-row sets of a workgroup.  4: a wave takes 32 keys of a tile (of 64 keys, D
// 512 of 32); 8 (D < 512): all 64, one half after the other, so that twice as many
// rows share the staging of a tile (64 sequences with 2 query heads a kv head over
// 32,768 shared keys, D 256: 233 us with 4, 212 with 8, 199 with the steps after).
// Two waves fill a SIMD (registers).  VALU takes 54% of its cycles and the matrix
// cores 27% there, 49% and 23% at D 512 (2,048 queries after 6,144 keys: 2.75 ms, 350
// TFLOP/s); a wave runs the two one after the other.
template <int D, bool F32, bool Q32, int RS>
__global__ __launch_bounds__(128 * kRs) __attribute__((amdgpu_waves_per_eu(2, 2)))
void paged_tiles_kernel(TileParams p) {
  using Gm = PfGeom<D, F32, kRs>;
  using SB = typename Gm::SB;
  constexpr int NG = Gm::NG, NWG = Gm::NW_, TK = Gm::TK, KH = Gm::KH, DH = Gm::DH;
  constexpr int KW = Gm::NW / (RS * DH), HB = KH / KW;  // waves that share a row set's keys; parts of each
  constexpr int kRows = 16 * RS;
  static_assert(KW >= 1 && HB >= 1, "waves");
  using St = PgStage<D, F32>;
  __shared__ __attribute__((aligned(16))) union Lds {
    St st;
    float o[Gm::NW][16 * Gm::OSTR];
    __device__ Lds() {}
  } L;
  __shared__ uint32_t vmx;                  // bits of the first tile's largest |V scale|
  __shared__ int alike[2][2 * Gm::NSW];     // see pg_alike (all of them set)
  __shared__ float ml[Gm::NW][16], ll[Gm::NW][16];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int rs = wave % RS, kw = wave / RS % KW, dh = wave / (RS * KW);
  const int m = lane & 15, c = lane >> 4;
  // heads vary fastest, the longest key ranges (last queries) start first
  const int nblk = gridDim.x / p.Hkv;
  const int kvh = blockIdx.x % p.Hkv, blk = nblk - 1 - static_cast<int>(blockIdx.x / p.Hkv);
  const int total = p.nq * p.gqa;           // rows of this kv head
  const int r0 = blk * kRows;               // first row of this workgroup

  // ---- the rows' limits, and the workgroup's tiles ----------------------------
  // row r attends key t iff t < hi and (t >= lo or t < sinks)
  const auto limits = [&](int r, int& hi, int& lo) {
    const int q = r / p.gqa;
    if (p.prefill) {
      hi = p.n + q + 1;
      lo = p.window > 0 ? max(0, hi - p.window) : 0;
    } else {
      const int n = max(min(p.seq_lens[q], p.n_clamp), 0);
      const int W = p.windows ? p.windows[q] : p.window;
      hi = min(n, p.shared);
      lo = W > 0 ? max(0, n - W) : 0;
    }
  };
  int hi_w, lo_w;
  {
    int h, l;
    limits(min(r0 + lane, total - 1), h, l);
    if constexpr (kRows > 64) {
      int h1, l1;
      limits(min(r0 + 64 + lane, total - 1), h1, l1);
      h = max(h, h1);
      l = min(l, l1);
    }
    hi_w = max_of_wave(h);
    lo_w = min_of_wave(l);
  }
  const int end = (hi_w + TK - 1) / TK;
  const int ns = min(p.sinks / TK + (p.sinks % TK != 0), end);  // tiles that hold sinks
  const int skip = max(0, min(lo_w / TK, end) - ns);            // tiles between those and the window's
  const int nt = end - skip;
  const int per = (nt + p.splits - 1) / p.splits;
  const int it0 = min(static_cast<int>(blockIdx.y) * per, nt), it1 = min(it0 + per, nt);
  PgRun run;
  const auto load_run = [&](int it) {  // of tiles it ...
    const int v = min(it + lane / KH, nt - 1);
    const int key = max(TK * (v + (v < ns ? 0 : skip)) + 32 * (lane % KH), 0);
    const int e = nt > 0 ? p.tables[min(key >> p.page_shift, p.max_pages - 1)] : -1;
    const bool has = static_cast<unsigned>(e) < static_cast<unsigned>(p.num_pages);
    const int64_t row = ((static_cast<int64_t>(has ? e : 0) * p.Hkv + kvh) << p.page_shift) + (key & ((1 << p.page_shift) - 1));
    run.lo = static_cast<int>(row);
    run.hi = static_cast<int>(row >> 32);
    run.has = __ballot(has);
  };
  // Tile it: its lane in the run, first key, and bits of the parts that exist.
  const auto tile_at = [&](int it, int& key, int& has) {
    const int i = (it - it0) & (64 / KH - 1);
    if (it != it0 && i == 0) {  // waited for in here: the steady loop waits for nothing
      load_run(it);
      asm volatile("" : "+v"(run.lo), "+v"(run.hi));
    }
    key = TK * (it + (it < ns ? 0 : skip));
    has = static_cast<int>(run.has >> (i * KH)) & ((1 << KH) - 1);
    return i * KH;
  };
  load_run(it0);

  const int rw = r0 + 16 * rs;              // the wave's first row
  const int R = min(rw + m, total - 1);     // this lane's row (column m)
  const int qi = R / p.gqa;
  int hi, lo;
  limits(R, hi, lo);
  // over the wave's rows
  const int hi_max = max_of_wave(hi), hi_min = min_of_wave(hi);
  const int lo_max = max_of_wave(lo), lo_min = min_of_wave(lo);

  int key, has;  // of the tile in LDS
  const int i0 = tile_at(it0, key, has);
  const PgSource<Gm> from = pg_source<Gm>(p);
  PfRaw<Gm> raw;
  pg_load<Gm>(raw, from, run, i0);

  // ---- q: B operands of k-step s of group g are dims 64 g + 16 c + 8 s + {0, 4,
  // 1, 5, 2, 6, 3, 7}, times 2^(6 - ex) (the row's largest below 2^6, so that group
  // sums fit fp16; what is below fp16's 2^-24 is 2^-26 of it and less), the odd
  // ones over 16; fp32 queries in two fp16 parts.  The sign of a negative scale
  // goes into q.
  v8h qf[2 * NWG], ql[Q32 ? 2 * NWG : 1], qb;
  const int64_t qrow = static_cast<int64_t>(qi) * p.Hq + kvh * p.gqa + (R - qi * p.gqa);
  float f[2 * NWG][8];
  float mx = 0.0f;
#pragma unroll
  for (int j = 0; j < 2 * NWG; ++j) {
    const int64_t e0 = qrow * D + Gm::OW * dh + 64 * (j >> 1) + 16 * c + 8 * (j & 1);
    if constexpr (Q32) {
      const v4f* src = reinterpret_cast<const v4f*>(static_cast<const float*>(p.q) + e0);
      const v4f a = src[0], b = src[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[j][i] = a[i];
        f[j][4 + i] = b[i];
      }
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + e0);
      const uint32_t wd[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (p.q_dtype == TQ_F16) {
          const v2h h = __builtin_bit_cast(v2h, wd[i]);
          f[j][2 * i] = static_cast<float>(h[0]);
          f[j][2 * i + 1] = static_cast<float>(h[1]);
        } else {
          f[j][2 * i] = __uint_as_float(wd[i] << 16);
          f[j][2 * i + 1] = __uint_as_float(wd[i] & 0xFFFF0000u);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(f[j][i]));
  }
  mx = xor32_max(xor16_max(mx));
  const int ex = __builtin_amdgcn_frexp_expf(mx);
  // score = rf * products (of a scale of 0 not 0: -inf stays one)
  const float rf0 = ldexpf(fabsf(p.scale_log2), ex - 6);
  const float rf = rf0 < FLT_MIN ? FLT_MIN : rf0 > FLT_MAX ? FLT_MAX : rf0;
  const bool neg = p.scale_log2 < 0.0f;
  float qs[NWG];
#pragma unroll
  for (int g = 0; g < NWG; ++g) qs[g] = 0.0f;
#pragma unroll
  for (int j = 0; j < 2 * NWG; ++j) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float x = ldexpf(f[j][i], 6 - ex);
      x = neg ? -x : x;
      qs[j >> 1] += x;
      const int slot = (i & 2) ? 4 + 2 * (i & 1) + (i >> 2) : 2 * (i & 1) + (i >> 2);
      const float y = (i & 1) ? x * 0.0625f : x;
      if constexpr (Q32) {
        // one rounding for both parts: the remainder is of the part that is stored
        uint32_t hb = __builtin_bit_cast(uint16_t, static_cast<_Float16>(y));
        asm("" : "+v"(hb));
        const _Float16 h = __builtin_bit_cast(_Float16, static_cast<uint16_t>(hb));
        qf[j][slot] = h;
        ql[j][slot] = static_cast<_Float16>(y - static_cast<float>(h));
      } else {
        qf[j][slot] = static_cast<_Float16>(y);
      }
    }
  }
  // group sums (|.| < 2^12).  fp16 scale/bias: part c of three fp16
  // parts in lane group c for the biases, 8 times it for the scales; fp32: kept
  // in fp32.
#pragma unroll
  for (int g = 0; g < NWG; ++g) qs[g] = xor32_sum(xor16_sum(qs[g]));
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    _Float16 pt = static_cast<_Float16>(0.0f);
    if (!F32 && g < NWG) {
      float x = qs[g < NWG ? g : 0];
      const _Float16 h0 = static_cast<_Float16>(x);
      x -= static_cast<float>(h0);
      const _Float16 h1 = static_cast<_Float16>(x);
      x -= static_cast<float>(h1);
      const _Float16 h2 = static_cast<_Float16>(x);
      pt = c == 0 ? h0 : c == 1 ? h1 : c == 2 ? h2 : pt;
    }
    qb[g] = pt;
    qb[4 + g] = pt * static_cast<_Float16>(8.0f);
  }

  if (threadIdx.x == 0) vmx = 0;
  if (threadIdx.x < St::TKP) {
    L.st.one[threadIdx.x] = static_cast<_Float16>(1.0f);
    L.st.zero[threadIdx.x] = static_cast<_Float16>(0.0f);
  }
  if (F32 && threadIdx.x < Gm::TK) L.st.zero32[threadIdx.x] = 0.0f;
  __syncthreads();
  pg_mask<Gm>(raw, key, has, hi_w);
  const float wm = pf_vmax<Gm>(raw);
  if (lane == 0) atomicMax(&vmx, __float_as_uint(wm));
  __syncthreads();
  // (a first tile outside these bounds, like an infinity, is not alike)
  const int e0 = min(max(__builtin_amdgcn_frexp_expf(__uint_as_float(__builtin_amdgcn_readfirstlane(vmx))), -20), 24);
  const auto stage = [&](int b) {
    pf_store_words<Gm>(L.st, raw, b);
    pg_store_sb<D, F32>(L.st, raw, b, e0);
    pg_alike<Gm>(raw, e0, alike[b]);
  };
  stage(0);
  __syncthreads();

  // Rows of the bias products' A operand: lane group c's keys of row m = 4 part +
  // group of this wave's groups; row 8 is 1 (fp16 caches: the sum of the weights).
  // Weights go in times 2^(e0 + 2), below 2^14; sums come out times 1 / bun.
  const _Float16* brow = L.st.zero;
  int bstep = 0;
  if (m / 4 < St::NP && m % 4 < NWG) {
    brow = &L.st.vp[0][m / 4][NWG * dh + m % 4][0];
    bstep = sizeof(L.st.vp[0]) / sizeof(_Float16);
  } else if (!F32 && m == 8) {
    brow = L.st.one;
  }
  brow += 4 * c;
  const float pscale = __uint_as_float((e0 + 2 + 127) << 23);
  const float bun = F32 ? 0.25f : __uint_as_float((127 - e0 - 2) << 23), bup = F32 ? 4.0f : pscale;

  // p = 2^(x - m_ref), m_ref = a score of the row + e0 - kPfHead, the largest so
  // far up to kPfLazy
  float m_ref = -INFINITY, l_run = 0.0f;
  const v4f z = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  v4f o[4 * NWG], ob = z;
#pragma unroll
  for (int b = 0; b < 4 * NWG; ++b) o[b] = z;

#pragma unroll 1
  for (int it = it0; it < it1; ++it) {
    const int buf = (it - it0) & 1;
    int nkey = key, nhas = has;
    if (it + 1 < it1) {
      const int i = tile_at(it + 1, nkey, nhas);
      pg_load<Gm>(raw, from, run, i);
    }
#pragma unroll 1
    for (int part = 0; part < HB; ++part) {
      const int kh = KW == 1 ? part : kw;
      const int t0 = key + 32 * kh;  // this wave's keys t0 .. t0 + 31
      const bool any = (has >> kh & 1) && rw < total && t0 < hi_max && (t0 + 31 >= lo_min || t0 < p.sinks);  // wave-uniform
      // this wave's groups
      const u32x4* ku = L.st.k[buf] + 2 * kh * Gm::KU + 128 * NWG * dh + 16 * c;
      const u32x4* vu = L.st.v[buf] + kh * Gm::VU + 256 * NWG * dh + 16 * c;
      const SB* sks = L.st.ksb[buf][0] + 32 * kh * NG + NWG * dh;
      const SB* skb = L.st.ksb[buf][1] + 32 * kh * NG + NWG * dh;
      // V operands of group g, and its scales of this lane's 8 keys
      const auto v_read = [&](int g, u32x4 (&a)[4]) {
#pragma unroll
        for (int x = 0; x < 4; ++x) a[x] = vu[(4 * g + x) * 64 + (m ^ Gm::vswz(g))];
      };
      typedef typename std::conditional<F32, v4f, v4h>::type s4;
      // (from, by bytes a group: the staged scales, or zeros)
      const auto s_read = [&](const char* from, int step, int g, s4 (&s)[2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) s[h] = *reinterpret_cast<const s4*>(from + g * step + 16 * h * (F32 ? 4 : 2));
      };

      u32x2 b0{}, b1{};  // the bias products' operand
      int al = 1;
      float sc[8];
      if (any) {
        // ---- S^T: two 16-key halves.  The operands of GB groups are read at once,
        // the next ones under the products and scores of these.
        constexpr int GB = Q32 && NWG > 1 ? NWG / 2 : NWG;
        u32x4 ka[2 * GB];
        const auto k_read = [&](int h, int g0) {
#pragma unroll
          for (int g = 0; g < GB; ++g) {
            const u32x4* kr = ku + h * Gm::KU + 128 * (g0 + g) + (m ^ Gm::kswz(NWG * dh + g0 + g));
            ka[2 * g] = kr[0];
            ka[2 * g + 1] = kr[64];
          }
          __builtin_amdgcn_sched_barrier(0);
        };
        k_read(0, 0);
        // and the scales and biases: of key m for the bias product, of this lane's
        // scores (keys 4 c + i); of both halves, or (fp32: registers) of one
        typedef SB row_t __attribute__((ext_vector_type(NWG)));
        constexpr int HA = F32 ? 1 : 2;
        row_t kbr[HA], ksr[HA], sk[HA][4], bk[4];
        const auto sb_read = [&](int h) {
          if constexpr (!F32) {
            kbr[h % HA] = *reinterpret_cast<const row_t*>(skb + (16 * h + m) * NG);
            ksr[h % HA] = *reinterpret_cast<const row_t*>(sks + (16 * h + m) * NG);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sk[h % HA][i] = *reinterpret_cast<const row_t*>(sks + (16 * h + 4 * c + i) * NG);
            if constexpr (F32) bk[i] = *reinterpret_cast<const row_t*>(skb + (16 * h + 4 * c + i) * NG);
          }
        };
#pragma unroll
        for (int h = 0; h < HA; ++h) sb_read(h);
        b0 = *reinterpret_cast<const u32x2*>(brow + buf * bstep + 32 * kh);
        b1 = *reinterpret_cast<const u32x2*>(brow + buf * bstep + 32 * kh + 16);
#pragma unroll
        for (int i = 0; i < 2 * Gm::NSW; ++i) al &= alike[buf][i];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          v4f bt = z;
          if constexpr (!F32) {
            v8h kb;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const _Float16 zero = static_cast<_Float16>(0.0f);
              kb[g] = g < NWG ? kbr[h % HA][g < NWG ? g : 0] : zero;
              kb[4 + g] = g < NWG ? ksr[h % HA][g < NWG ? g : 0] : zero;
            }
            bt = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, qb, z, 0, 0, 0);
          }
          v4f acc[NWG];
#pragma unroll
          for (int g0 = 0; g0 < NWG; g0 += GB) {
#pragma unroll
            for (int gi = 0; gi < GB; ++gi) {
              const int g = g0 + gi;
              const v8h a0 = __builtin_bit_cast(v8h, ka[2 * gi]), a1 = __builtin_bit_cast(v8h, ka[2 * gi + 1]);
              v4f a = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, qf[2 * g], z, 0, 0, 0);
              a = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, qf[2 * g + 1], a, 0, 0, 0);
              if constexpr (Q32) {
                a = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, ql[2 * g], a, 0, 0, 0);
                a = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, ql[2 * g + 1], a, 0, 0, 0);
              }
              acc[g] = a;
            }
            __builtin_amdgcn_sched_barrier(0);
            if (g0 + GB < NWG) k_read(h, g0 + GB);
            else if (h == 0) k_read(1, 0);
          }
          if (F32 && h == 1) sb_read(1);
          // (four sums side by side: one after the other, each step waits for the last)
          float s[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) s[i] = bt[i];
#pragma unroll
          for (int g = 0; g < NWG; ++g) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if constexpr (F32) {
                // s (. + 8 sum q) + b sum q
                s[i] = fmaf(bk[i][g], qs[g], s[i]);
                s[i] = fmaf(sk[h % HA][i][g], fmaf(qs[g], 8.0f, acc[g][i]), s[i]);
              } else {
                s[i] = fmaf(static_cast<float>(sk[h % HA][i][g]), acc[g][i], s[i]);
              }
            }
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[4 * h + i] = DH == 2 ? s[i] * rf : s[i];  // (a wave's dims have an rf of their own)
        }
      }
      if constexpr (DH == 2) {
        // the other wave's groups: its parts of the same scores
        if (any) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            L.st.xch[wave][h][lane] = v4f{sc[4 * h], sc[4 * h + 1], sc[4 * h + 2], sc[4 * h + 3]};
        }
        __syncthreads();
        if (any) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const v4f x = L.st.xch[wave ^ RS][h][lane];
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[4 * h + i] += x[i];
          }
        }
      }
      if (any) {
        // whether all of these keys are attended by all rows; wave-uniform
        const bool inside = t0 <= hi_min - 32 && (t0 >= lo_max || t0 <= p.sinks - 32);
        if (!inside) {
          const int at = t0 + 4 * c;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int k = 16 * (j >> 2) + (j & 3);
            sc[j] = k < hi - at && (k >= lo - at || k < p.sinks - at) ? sc[j] : -INFINITY;
          }
        }

        // ---- online softmax (log2 domain) of rows m ------------------------------
        const float up = static_cast<float>(e0 - kPfHead);
        float mt = sc[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) mt = fmaxf(mt, sc[j]);
        const float need = fmaf(xor32_max(xor16_max(mt)), DH == 2 ? 1.0f : rf, up);
        // (a row with nothing attended yet and nothing here keeps -inf)
        if (__any(need > m_ref + kPfLazy)) {
          const float m_new = need > m_ref ? need : m_ref;
          const float fr = m_new == m_ref ? 1.0f : merge_factor(m_ref, m_new);
          l_run *= fr;
          ob *= fr;
#pragma unroll
          for (int b = 0; b < 4 * NWG; ++b) o[b] *= fr;
          m_ref = m_new;
        }
        // In a tile that is not plain the products below take weights and biases of 0
        // (a branch around them would cost a second set of accumulators).
        const bool plain = __builtin_amdgcn_readfirstlane(al) != 0;
        const char* sfrom;
        int sstep = 0;
        if constexpr (F32) {
          sfrom = reinterpret_cast<const char*>(plain ? &L.st.vsb[buf][0][NWG * dh][32 * kh] : &L.st.zero32[0]);
          if (plain) sstep = sizeof(L.st.vsb[0][0][0]);
          sfrom += 16 * c;
        } else {
          sfrom = reinterpret_cast<const char*>(plain ? &L.st.vp[buf][1][NWG * dh][32 * kh] : &L.st.zero[0]);
          if (plain) sstep = sizeof(L.st.vp[0][0][0]);
          sfrom += 8 * c;
        }
        u32x4 va[4];
        s4 vs[2][2];
        v_read(0, va);
        s_read(sfrom, sstep, 0, vs[0]);
        const uint32_t bm = plain ? ~0u : 0u;
        const v8h ba = __builtin_bit_cast(v8h, u32x4{b0[0] & bm, b0[1] & bm, b1[0] & bm, b1[1] & bm});
        __builtin_amdgcn_sched_barrier(0);
        float pw[8];
        // (with nothing attended so far, -inf - -inf would be NaN)
        const float ms = m_ref == -INFINITY ? 0.0f : m_ref;
#pragma unroll
        for (int j = 0; j < 8; ++j) pw[j] = fast_exp2(DH == 2 ? sc[j] - ms : fmaf(sc[j], rf, -ms));
        if constexpr (F32) {
#pragma unroll
          for (int j = 0; j < 8; ++j) l_run += pw[j];
        }

        // ---- O^T += V^T P^T ----------------------------------------------------
        // B operands of eight weights
        const auto split = [&](const float (&y)[8], v8h& bh, v8h& bl) {
          u32x4 hw, lw;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            hw[q] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(y[2 * q], y[2 * q + 1]));
            lw[q] = pf_rem_pair(hw[q], y[2 * q], y[2 * q + 1]);
          }
          bh = __builtin_bit_cast(v8h, hw);
          bl = __builtin_bit_cast(v8h, lw);
        };
        if (!plain) {
          // V scales apart, or scales and biases out of range or not finite: the
          // largest weight of every row and group to 2^13 .. 2^14 (an infinity, of
          // exponent 0, stays one), the products on their own, added in fp32, and
          // bias terms in fp32 -- without those of weight 0, whose keys the row may
          // not attend at all
          const auto times = [](float w, float x) { return w > 0.0f || w != w ? w * x : 0.0f; };
          float add[4] = {0.0f, 0.0f, 0.0f, 0.0f}, lw = 0.0f;
#pragma unroll 1
          for (int g = 0; g < NWG; ++g) {
            float y[8], big = 0.0f, sb = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int at = 32 * kh + 16 * (j >> 2) + 4 * c + (j & 3);
              float s, b;
              if constexpr (F32) {
                s = L.st.vsb[buf][0][NWG * dh + g][at];
                b = L.st.vsb[buf][1][NWG * dh + g][at];
              } else {
                s = static_cast<float>(L.st.vp[buf][1][NWG * dh + g][at]);
                b = static_cast<float>(L.st.vp[buf][0][NWG * dh + g][at]);
              }
              y[j] = times(pw[j], s);
              sb += times(pw[j], fmaf(s, 8.0f, b));
              big = fmaxf(big, fabsf(y[j]));
            }
            sb = xor32_sum(xor16_sum(sb)) * bup;
#pragma unroll
            for (int i = 0; i < 4; ++i) add[i] = i == g ? sb : add[i];
            const int k = min(14 - __builtin_amdgcn_frexp_expf(xor32_max(xor16_max(big))), 120);
            const float un = ldexpf(1.0f, -k);
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = ldexpf(y[j], k);
            v8h bh, bl;
            split(y, bh, bl);
#pragma unroll
            for (int gg = 0; gg < NWG; ++gg) {
              if (gg != g) continue;
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const v8h a = __builtin_bit_cast(v8h, vu[(4 * gg + x) * 64 + (m ^ Gm::vswz(gg))]);
                v4f t = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bh, z, 0, 0, 0);
                t = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bl, t, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[4 * gg + x][i] = fmaf(t[i], un, o[4 * gg + x][i]);
              }
            }
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) lw += pw[j];
          lw = xor32_sum(xor16_sum(lw)) * bup;
          // into the rows that hold biases and, for fp16 caches, the weights' sum
#pragma unroll
          for (int i = 0; i < 4; ++i) ob[i] += c == 0 ? add[i] : 0.0f;
          if (!F32 && c == 2) ob[0] += lw;
#pragma unroll
          for (int j = 0; j < 8; ++j) pw[j] = 0.0f;
        }
        {
          v8h bh, bl;
          float y[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = pw[j] * pscale;
          split(y, bh, bl);
          ob = __builtin_amdgcn_mfma_f32_16x16x32_f16(ba, bh, ob, 0, 0, 0);
          ob = __builtin_amdgcn_mfma_f32_16x16x32_f16(ba, bl, ob, 0, 0, 0);
        }
#pragma unroll
        for (int g = 0; g < NWG; ++g) {
          if (g + 1 < NWG) s_read(sfrom, sstep, g + 1, vs[(g + 1) & 1]);
          __builtin_amdgcn_sched_barrier(0);
          v8h bh, bl;
          float y[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = fmaf(static_cast<float>(vs[g & 1][j >> 2][j & 3]), pw[j], 0.0f);
          split(y, bh, bl);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const v8h a = __builtin_bit_cast(v8h, va[x]);
            v4f& acc = o[4 * g + x];
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bh, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bl, acc, 0, 0, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
          if (g + 1 < NWG) v_read(g + 1, va);  // under the next group's weights
        }
      }
    }
    if (it + 1 < it1) {
      pg_mask<Gm>(raw, nkey, nhas, hi_w);
      stage(buf ^ 1);
    }
    key = nkey;
    has = nhas;
    __syncthreads();
  }

  // ---- merge of the KW partials of every row, and the output ------------------
  const float un = c < 2 ? 1.0f : 0.0625f;  // odd nibbles (rows 8-15) were 16 times as large
  const float lt = F32 ? xor32_sum(xor16_sum(l_run)) : xor32_sum(xor16_sum(c == 2 ? ob[0] : 0.0f)) * bun;
  if (c == 0) {
    ml[wave][m] = m_ref;
    ll[wave][m] = lt;
  }
  float* orow = L.o[wave] + m * Gm::OSTR;
#pragma unroll
  for (int g = 0; g < NWG; ++g) {
    // b' = b + 8 s: biases in the rows of lane group 0 (fp32 caches: and 1), scales
    // in those of 1 (2 and 3)
    const float bs = c < (F32 ? 2 : 1) ? ob[g] : c < (F32 ? 4 : 2) ? 8.0f * ob[g] : 0.0f;
    const float bg = xor32_sum(xor16_sum(bs)) * bun;
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        orow[64 * g + 8 * (4 * (c & 1) + i) + 2 * x + (c >> 1)] = fmaf(o[4 * g + x][i], un, bg);
  }
  __syncthreads();
  for (int u = threadIdx.x; u < kRows * (D / 2); u += Gm::NT) {
    // a wave's 64 units lie in one row and in one wave's dims
    const int r = __builtin_amdgcn_readfirstlane(u / (D / 2)), d = 2 * (u % (D / 2));
    const int Ro = r0 + r;
    if (Ro >= total) break;
    const int rm = r % 16, w0 = r / 16 + RS * KW * (d / Gm::OW);
    float M = -INFINITY;
#pragma unroll
    for (int k = 0; k < KW; ++k) M = fmaxf(M, ml[w0 + RS * k][rm]);
    float l = 0.0f, x0 = 0.0f, x1 = 0.0f;
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      const int wv = w0 + RS * k;
      const float fk = merge_factor(ml[wv][rm], M);
      const float2 v = *reinterpret_cast<const float2*>(&L.o[wv][rm * Gm::OSTR + d % Gm::OW]);
      l = fmaf(ll[wv][rm], fk, l);
      x0 = fmaf(v.x, fk, x0);
      x1 = fmaf(v.y, fk, x1);
    }
    const int qo = Ro / p.gqa;
    const int64_t row = static_cast<int64_t>(qo) * p.Hq + kvh * p.gqa + (Ro - qo * p.gqa);
    if (p.ext_merge == 0) {
      *reinterpret_cast<float2*>(p.out + row * D + d) = make_float2(normalise(x0, l, 0.0f), normalise(x1, l, 0.0f));
    } else {
      const int64_t slot = row * p.max_splits + blockIdx.y;
      *reinterpret_cast<float2*>(p.ws_o + slot * D + d) = make_float2(x0, x1);
      if (d == 0) *reinterpret_cast<float2*>(p.ws_ml + slot * 2) = make_float2(M, l);
    }
  }
}

// The output of a row from its S partials: a thread takes four dims.
__global__ __launch_bounds__(256) void merge_tiles_kernel(const float* ws_ml, const float* ws_o, float* out,
                                                          int64_t rows, int S, int stride, int D4) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= rows * D4) return;
  const int64_t row = i / D4;
  const int d4 = static_cast<int>(i - row * D4);
  const float2* ml = reinterpret_cast<const float2*>(ws_ml) + row * stride;
  const v4f* po = reinterpret_cast<const v4f*>(ws_o) + row * stride * D4 + d4;
  float M = -INFINITY, L = 0.0f;
  for (int k = 0; k < S; ++k) M = fmaxf(M, ml[k].x);
  v4f O = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int k = 0; k < S; ++k) {
    const float fk = merge_factor(ml[k].x, M);
    L = fmaf(ml[k].y, fk, L);
    O += fk * po[static_cast<int64_t>(k) * D4];
  }
  v4f r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = normalise(O[e], L, 0.0f);
  reinterpret_cast<v4f*>(out)[i] = r;
}

template <int D, bool F32, int RS>
void launch_q(const TileParams& p, dim3 grid, hipStream_t s) {
  if constexpr (!(D == 256 && F32 && RS == 8)) {  // (never planned for fp32 queries)
    if (p.q_dtype == TQ_F32) {
      paged_tiles_kernel<D, F32, true, RS><<<grid, 128 * kRs, 0, s>>>(p);
      return;
    }
  }
  paged_tiles_kernel<D, F32, false, RS><<<grid, 128 * kRs, 0, s>>>(p);
}

template <bool F32>
void launch_dim(const TileParams& p, int D, int rs, dim3 grid, hipStream_t s) {
  if (D == 512) launch_q<512, F32, 4>(p, grid, s);
  else if (D == 256) rs == 8 ? launch_q<256, F32, 8>(p, grid, s) : launch_q<256, F32, 4>(p, grid, s);
  else rs == 8 ? launch_q<128, F32, 8>(p, grid, s) : launch_q<128, F32, 4>(p, grid, s);
}

int tile_keys(int D) { return D == 512 ? 32 : 64; }
int64_t tile_wgs(int64_t rows, int Hkv, int rs) { return (rows + 16 * rs - 1) / (16 * rs) * Hkv; }

// Splits of a grid of wgs workgroups that could be of use.
int most_splits(int64_t wgs, int64_t tiles) {
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({64, tiles / 2, (target_wgs() + wgs - 1) / wgs})));
}

}  // namespace

int paged_tiles_max_splits(int64_t rows, int Hkv, int D, int64_t keys) {
  return most_splits(tile_wgs(rows, Hkv, D == 512 ? 4 : 8), (keys + tile_keys(D) - 1) / tile_keys(D));
}

TilesPlan plan_paged_tiles(int64_t rows, int Hkv, int D, int64_t keys, int64_t longest, bool all32) {
  const int64_t tiles = (keys + tile_keys(D) - 1) / tile_keys(D), most = (longest + tile_keys(D) - 1) / tile_keys(D);
  const int64_t cus = target_wgs();
  // A workgroup fills a CU, and costs its prologue, epilogue and part of the merge
  // beside its tiles; in eighths of a tile of 64 rows, a tile of 128 rows costs
  // kTile[1], and the rest kFixed.  The plan of least estimated time: of the rounds of
  // average workgroups, or of the longest one (a causal prompt's last rows).  64
  // against 128 rows in us, bf16 queries and fp16 scales, D 128 (Hq 16 Hkv 8) and D 256
  // (Hq 32 Hkv 16):
  //   64 sequences over 32,768 shared keys    74 : 68     209 : 184   128 taken
  //   prompt of 2,048 after 4,096            302 : 280    936 : 758   128
  //   prompt of 512 after 4,096               78 : 73     211 : 191   128
  //   prompt of 512 after 4,000, W 1,024      32 : 36      62 : 71     64
  //   prompt of 1,024                         38 : 45      75 : 91     64
  //   prompt of 67 after 4,001, W 1,024       19 : 24      34 : 42     64
  // Of 180 such pairs (other heads, fp32 queries or scales) four take the slower one:
  // by 3 to 4%, 6% and 10%, the last three of fp32 scales at D 256.
  constexpr int64_t kTile[2] = {8, 13}, kFixed[2] = {48, 72};
  TilesPlan best{4, 1};
  int64_t least = INT64_MAX;
  // (D 256 with fp32 queries and scales: 100 registers spilled with 128 rows, 331
  // against 240 us over 32,768 shared keys; with one of them in 16 bits, none to 13
  // and 202 to 216 against 226 to 229)
  for (int rs = 4; rs <= (D == 512 || (D == 256 && all32) ? 4 : 8); rs += 4) {
    const int64_t wgs = tile_wgs(rows, Hkv, rs), tile = kTile[rs / 8], fixed = kFixed[rs / 8];
    for (int s = 1; s <= most_splits(wgs, tiles); ++s) {
      const int64_t cost = std::max((wgs * s + cus - 1) / cus * ((tiles + s - 1) / s * tile + fixed),
                                    (most + s - 1) / s * tile + fixed);
      if (cost < least) {
        least = cost;
        best = {rs, s};
      }
    }
  }
  return best;
}

int launch_paged_tiles(const PagedParams& p0, int D, int sb_dtype, TilesPlan plan, bool partials, hipStream_t s) {
  TileParams p;
  static_cast<PagedParams&>(p) = p0;
  p.splits = plan.splits;
  p.ext_merge = partials || plan.splits > 1;
  const int64_t rows = static_cast<int64_t>(p.nq) * p.gqa;
  const dim3 grid(static_cast<unsigned>(tile_wgs(rows, p.Hkv, plan.rs)), plan.splits);
  if (sb_dtype == TQ_F32) launch_dim<true>(p, D, plan.rs, grid, s);
  else launch_dim<false>(p, D, plan.rs, grid, s);
  TQ_CHECK_LAUNCH("paged_tiles_kernel");
  if (partials || plan.splits == 1) return TQ_OK;
  const int64_t out_rows = static_cast<int64_t>(p.nq) * p.Hq;
  merge_tiles_kernel<<<static_cast<unsigned>((out_rows * (D / 4) + 255) / 256), 256, 0, s>>>(
      p.ws_ml, p.ws_o, p.out, out_rows, plan.splits, p.max_splits, D / 4);
  TQ_CHECK_LAUNCH("merge_tiles_kernel");
  return TQ_OK;
}

}  // namespace tq
