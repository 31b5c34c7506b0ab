// Chunks of a batch: a job of few rows (queries x heads of a kv head) over pages.
//
// Four waves take 16 rows of one kv head and split their keys, where tiles staged for 64
// or 128 rows would leave most of a workgroup idle: each wave streams 32-key blocks of its
// own, with no barrier until the end.  The mathematics is that of tq_paged_tiles.hip
// (centred fp16 nibbles; S^T = K q^T by quant group, P V as fp16 high part and remainder),
// with one difference: the weights p s_v of a (row, group) go in times a power of two that
// its sums carry too.  It falls where a weight would pass fp16 and rises where a row with a
// p of about 1 (its largest is that or more) has no weight of 1 or more, so that no range of
// V scales needs a path beside this one: fp16's last step is 2^-24, and what is rounded off a
// weight is 2^-25 of the row's sums at most.  (5 tokens as below: 49.4 us without the rise,
// 50.2 with it in a branch of the other's, 54 with a rise at every new reference.)
// What bounds it: VALU (about 700 instructions a wave and block at D 256, 61% of a SIMD's
// cycles with two waves) and the start and end of a job (about 9 us).  5 new tokens
// of 32 sequences behind a window of 1,024 (Hq 32 Hkv 16 D 256): 52 us, 2.9 TB/s of what
// has to be read, where the tile kernel takes 114.  Measured, not kept: workgroups of eight
// waves, one a CU, 69; V's operands read ahead of the softmax 60 (spills); nibbles as fp16
// subnormals, uncentred, for K 51 against 55, but errors of 3e-6 to 5e-6 in place of 0.5e-6.
#pragma once

#include "tq_chunk_jobs.h"
#include "tq_prefill_tile.h"

#include <cfloat>

namespace tq {
namespace {

constexpr int kFewBlock = 16;  // rows of a workgroup

template <int D, bool F32>
struct FewGeom {
  using SB = typename std::conditional<F32, float, _Float16>::type;
  // Four waves a job; two jobs a CU (one streams under the other's start and
  // end), at D 512 one, for its 128 accumulators and as many words in flight.
  static constexpr int NW = 4, NT = 64 * NW;
  static constexpr int W = D / 8, NG = D / 64;
  static constexpr int WP = W + 4;              // row stride in LDS: operand reads reach distinct banks
  static constexpr int NK = W / 8;              // 16-byte pieces of 32 keys' words, per lane
  static constexpr int SCB = 2 * NG * static_cast<int>(sizeof(SB));  // bytes of two keys' scales
  static constexpr int NS = SCB / 8;            // 8-byte pieces of them
  static constexpr int OSTR = D + 2;
  struct Stage {
    uint32_t k[32][WP], v[32][WP];
    uint64_t s[4][32 * NG * sizeof(SB) / 8];    // k scale, k bias, v scale, v bias: [key][group]
  };
  union Shared {
    Stage st[NW];
    float o[NW][16 * OSTR];
    __device__ Shared() {}
  };
  struct Lds {
    Shared u;
    float ml[NW][16], ll[NW][16];
    int told[kJobInts];
    __device__ Lds() {}
  };
};

// A block's words and scales in flight: pieces of 16 bytes in a row, lane after lane;
// lane l: the scales of keys 2 (l % 16) and the next of array l / 16.
template <int D, bool F32>
struct FewRaw {
  u32x4 k[FewGeom<D, F32>::NK], v[FewGeom<D, F32>::NK];
  uint64_t s[FewGeom<D, F32>::NS];
};

template <int D, bool F32>
__device__ __forceinline__ void few_load(FewRaw<D, F32>& R, const TileParams& p, const char* scales, int64_t row) {
  using Gm = FewGeom<D, F32>;
  const uint32_t lane = threadIdx.x & 63;
  const char* k = reinterpret_cast<const char*>(p.kq) + row * (4 * Gm::W);
  const char* v = reinterpret_cast<const char*>(p.vq) + row * (4 * Gm::W);
  const char* s = scales + row * (Gm::SCB / 2);
#pragma unroll
  for (int i = 0; i < Gm::NS; i += 2) {
    if constexpr (Gm::NS == 1) {
      R.s[0] = *reinterpret_cast<const uint64_t*>(s);
    } else {
      const u32x4 u = *reinterpret_cast<const u32x4*>(s + 8 * i);
      R.s[i] = static_cast<uint64_t>(u[1]) << 32 | u[0];
      R.s[i + 1] = static_cast<uint64_t>(u[3]) << 32 | u[2];
    }
  }
#pragma unroll
  for (int i = 0; i < Gm::NK; ++i) R.k[i] = *reinterpret_cast<const u32x4*>(k + 16 * lane + 1024 * i);
#pragma unroll
  for (int i = 0; i < Gm::NK; ++i) R.v[i] = *reinterpret_cast<const u32x4*>(v + 16 * lane + 1024 * i);
}

template <int D, bool F32>
__device__ __forceinline__ void few_store(typename FewGeom<D, F32>::Stage& S, const FewRaw<D, F32>& R) {
  using Gm = FewGeom<D, F32>;
  const int lane = threadIdx.x & 63;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // (behind the last block's reads)
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < Gm::NS; ++i) S.s[lane >> 4][(lane & 15) * Gm::NS + i] = R.s[i];
#pragma unroll
  for (int i = 0; i < Gm::NK; ++i) {
    const int w = 4 * lane + 256 * i;
    *reinterpret_cast<u32x4*>(&S.k[w / Gm::W][w % Gm::W]) = R.k[i];
    *reinterpret_cast<u32x4*>(&S.v[w / Gm::W][w % Gm::W]) = R.v[i];
  }
  // (other lanes of this wave read it)
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// pf_centre with the nibble, and so the offset, chosen by the lane.
__device__ __forceinline__ uint32_t few_centre(uint32_t t, uint32_t mask, v2h off) {
  uint32_t b;
  asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(b) : "v"(t), "v"(mask), "s"(0x64006400u));
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, b) + off);
}

// y0 f, y1 f as a packed fp16 pair, and what that pair leaves of them: mixed-precision
// fmas, each rounded once (the remainder is of the pair that is stored).
__device__ __forceinline__ uint32_t few_high(float y0, float y1, float f) {
  uint32_t r;
  asm("v_fma_mixlo_f16 %0, %1, %3, 0 op_sel_hi:[0,0,0]\n\t"
      "v_fma_mixhi_f16 %0, %2, %3, 0 op_sel_hi:[0,0,0]"
      : "=&v"(r)
      : "v"(y0), "v"(y1), "v"(f));
  return r;
}
__device__ __forceinline__ uint32_t few_low(uint32_t h, float y0, float y1, float f) {
  uint32_t r;
  asm("v_fma_mixlo_f16 %0, %1, %3, -%4 op_sel_hi:[0,0,1]\n\t"
      "v_fma_mixhi_f16 %0, %2, %3, -%4 op_sel:[0,0,1] op_sel_hi:[0,0,1]"
      : "=&v"(r)
      : "v"(y0), "v"(y1), "v"(f), "v"(h));
  return r;
}

// Job j, by NT threads of a workgroup (tid: a thread's number among them); three barriers
// of the workgroup, also where there is no such job.
template <int D, bool F32, bool Q32>
__device__ __forceinline__ void few_job(const TileParams& p, int j, int tid, typename FewGeom<D, F32>::Lds& lds) {
  using Gm = FewGeom<D, F32>;
  using SB = typename Gm::SB;
  constexpr int NG = Gm::NG, NW = Gm::NW, G4 = NG < 4 ? NG : 4;
  auto& L = lds.u;
  auto &ml = lds.ml, &ll = lds.ll;

  const ChunkJob job = chunk_job<kFewBlock, 32, true, false>(p, j, tid, lds.told);
  if (job.splits == 0) {  // (all of these threads; others of the workgroup may have a job)
    __syncthreads();
    __syncthreads();
    return;
  }
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, c = lane >> 4;
  const int total = job.n * p.gqa, r0 = job.blk * kFewBlock;
  const int* table = p.tables + static_cast<int64_t>(job.b) * p.max_pages;

  // ---- the rows' limits (row r attends key t iff t < hi and (t >= lo or t < sinks)),
  // and the workgroup's blocks of keys
  const auto hi_of = [&](int q) { return max(job.len - job.n + q + 1, 0); };
  const auto lo_of = [&](int hi) { return p.window > 0 ? max(0, hi - p.window) : 0; };
  const int hi_min = hi_of(r0 / p.gqa), hi_max = hi_of(min(r0 + kFewBlock - 1, total - 1) / p.gqa);
  const int lo_min = lo_of(hi_min), lo_max = lo_of(hi_max);
  const int end = (hi_max + 31) / 32;
  const int ns = min(p.sinks / 32 + (p.sinks % 32 != 0), end);
  const int skip = max(0, min(lo_min / 32, end) - ns);
  const int nt = end - skip;
  const int per = (nt + job.splits - 1) / job.splits;
  const int it0 = min(job.split * per, nt), it1 = min(it0 + per, nt);
  const int mine = max(0, (it1 - it0 - wave + NW - 1) / NW);  // this wave's: it0 + wave + NW i
  int run_lo = 0, run_hi = 0;  // first pool row of blocks i .. i + 63, in the lanes
  uint64_t run_has = 0;
  const auto key_of = [&](int i) {
    const int v = it0 + wave + NW * i;
    return 32 * (v + (v < ns ? 0 : skip));
  };
  const auto load_run = [&](int i) {
    const int key = key_of(min(i + lane, max(mine - 1, 0)));
    const int e = mine > 0 ? table[min(key >> p.page_shift, p.max_pages - 1)] : -1;
    const bool has = static_cast<unsigned>(e) < static_cast<unsigned>(p.num_pages);
    const int64_t row = ((static_cast<int64_t>(has ? e : 0) * p.Hkv + job.kvh) << p.page_shift) + (key & ((1 << p.page_shift) - 1));
    run_lo = static_cast<int>(row);
    run_hi = static_cast<int>(row >> 32);
    run_has = __ballot(has);
  };
  const auto row_of = [&](int i) {
    return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(run_hi, i & 63))) << 32 |
                                static_cast<uint32_t>(__builtin_amdgcn_readlane(run_lo, i & 63)));
  };
  load_run(0);

  const int R = min(r0 + m, total - 1);  // this lane's row (column m)
  const int qi = R / p.gqa;
  const int hi = hi_of(qi), lo = lo_of(hi);
  const int64_t qrow = static_cast<int64_t>(qi + job.s0) * p.Hq + job.kvh * p.gqa + (R - qi * p.gqa);

  // ---- q: B operands as in paged_tiles_kernel ------------------------------------
  float f[2 * NG][8];
#pragma unroll
  for (int j = 0; j < 2 * NG; ++j) {
    const int64_t e0 = qrow * D + 64 * (j >> 1) + 16 * c + 8 * (j & 1);
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
  }
  // the first block's loads go out behind q's
  const int arr = lane >> 4;
  const void* sc_base = arr == 0 ? p.ks : arr == 1 ? p.kb : arr == 2 ? p.vs : p.vb;
  const char* scales = static_cast<const char*>(sc_base) + (lane & 15) * Gm::SCB;
  FewRaw<D, F32> raw;
  few_load<D, F32>(raw, p, scales, row_of(0));  // (a wave without blocks: row 0 of the pool)

  float mx = 0.0f;
#pragma unroll
  for (int j = 0; j < 2 * NG; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(f[j][i]));
  mx = xor32_max(xor16_max(mx));
  const int ex = __builtin_amdgcn_frexp_expf(mx);
  const float rf0 = ldexpf(fabsf(p.scale_log2), ex - 6);
  const float rf = rf0 < FLT_MIN ? FLT_MIN : rf0 > FLT_MAX ? FLT_MAX : rf0;
  const bool neg = p.scale_log2 < 0.0f;
  v8h qf[2 * NG], ql[Q32 ? 2 * NG : 1], qb[NG / G4];
  float qs[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) qs[g] = 0.0f;
#pragma unroll
  for (int j = 0; j < 2 * NG; ++j) {
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
#pragma unroll
  for (int g = 0; g < NG; ++g) qs[g] = xor32_sum(xor16_sum(qs[g]));
  if constexpr (!F32) {
#pragma unroll
    for (int b = 0; b < NG / G4; ++b) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        _Float16 pt = static_cast<_Float16>(0.0f);
        if (g < G4) {
          float x = qs[G4 * b + (g < G4 ? g : 0)];
          const _Float16 h0 = static_cast<_Float16>(x);
          x -= static_cast<float>(h0);
          const _Float16 h1 = static_cast<_Float16>(x);
          x -= static_cast<float>(h1);
          const _Float16 h2 = static_cast<_Float16>(x);
          pt = c == 0 ? h0 : c == 1 ? h1 : c == 2 ? h2 : pt;
        }
        qb[b][g] = pt;
        qb[b][4 + g] = pt * static_cast<_Float16>(8.0f);
      }
    }
  }

  const v4f z = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  v4f o[4 * NG];
#pragma unroll
  for (int b = 0; b < 4 * NG; ++b) o[b] = z;
  float bs[NG];  // sums of p (b_v + 8 s_v)
  float ef[NG];  // a power of two: what the weights p s_v of a row and group go in times
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    bs[g] = 0.0f;
    ef[g] = 0x1p120f;
  }
  float m_ref = -INFINITY, l_run = 0.0f;
  // rows m < 8 of a V operand are the low nibbles of a byte of word m, the others the
  // high ones (16 times as large) of word m - 8
  const uint32_t vmask = m < 8 ? 0x000F000Fu : 0x00F000F0u;
  const _Float16 off1 = static_cast<_Float16>(m < 8 ? -1032.0f : -1152.0f);
  const v2h voff = v2h{off1, off1};
  typename Gm::Stage& S = L.st[wave];
  typedef SB row4 __attribute__((ext_vector_type(G4)));
  const auto scale_row = [&](int a, int key, int b) {
    return *reinterpret_cast<const row4*>(reinterpret_cast<const SB*>(S.s[a]) + key * NG + G4 * b);
  };

#pragma unroll 1
  for (int i = 0; i < mine; ++i) {
    const int t0 = key_of(i);
    const bool has = run_has >> (i & 63) & 1;
    few_store<D, F32>(S, raw);
    if (i + 1 < mine) {
      if (((i + 1) & 63) == 0) {
        load_run(i + 1);
        asm volatile("" : "+v"(run_lo), "+v"(run_hi));  // waited for in here
      }
      few_load<D, F32>(raw, p, scales, row_of(i + 1));
    }
    if (!(has && (t0 + 31 >= lo_min || t0 < p.sinks))) continue;  // wave-uniform

    // ---- S^T: two 16-key halves -----------------------------------------------------
    float sc[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      v4f s4 = z;
      if constexpr (!F32) {
#pragma unroll
        for (int b = 0; b < NG / G4; ++b) {
          const row4 kr = scale_row(0, 16 * h + m, b), br = scale_row(1, 16 * h + m, b);
          v8h kb;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const _Float16 zero = static_cast<_Float16>(0.0f);
            kb[g] = g < G4 ? static_cast<_Float16>(br[g < G4 ? g : 0]) : zero;
            kb[4 + g] = g < G4 ? static_cast<_Float16>(kr[g < G4 ? g : 0]) : zero;
          }
          s4 = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, qb[b], s4, 0, 0, 0);
        }
      }
      float s[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] = s4[e];
#pragma unroll
      for (int b = 0; b < NG / G4; ++b) {
        row4 kr[4], br[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          kr[e] = scale_row(0, 16 * h + 4 * c + e, b);
          if constexpr (F32) br[e] = scale_row(1, 16 * h + 4 * c + e, b);
        }
#pragma unroll
        for (int gi = 0; gi < G4; ++gi) {
          const int g = G4 * b + gi;
          const u32x2 w = *reinterpret_cast<const u32x2*>(&S.k[16 * h + m][8 * g + 2 * c]);
          v8h a[2];
#pragma unroll
          for (int x = 0; x < 2; ++x)
            a[x] = __builtin_bit_cast(v8h, u32x4{pf_centre<false>(w[x], 0x000F000Fu), pf_centre<true>(w[x], 0x00F000F0u),
                                                 pf_centre<false>(w[x] >> 8, 0x000F000Fu), pf_centre<true>(w[x] >> 8, 0x00F000F0u)});
          v4f acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0], qf[2 * g], z, 0, 0, 0);
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[1], qf[2 * g + 1], acc, 0, 0, 0);
          if constexpr (Q32) {
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0], ql[2 * g], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[1], ql[2 * g + 1], acc, 0, 0, 0);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (F32) {
              // s (. + 8 sum q) + b sum q
              s[e] = fmaf(br[e][gi], qs[g], s[e]);
              s[e] = fmaf(kr[e][gi], fmaf(qs[g], 8.0f, acc[e]), s[e]);
            } else {
              s[e] = fmaf(static_cast<float>(kr[e][gi]), acc[e], s[e]);
            }
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[4 * h + e] = s[e];
    }
    row4 vs[8], vb[8];
    uint32_t w[8];
    const auto v_rows = [&](int b) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = 16 * (j >> 2) + 4 * c + (j & 3);
        vs[j] = scale_row(2, key, b);
        vb[j] = scale_row(3, key, b);
      }
    };
    const auto v_words = [&](int g, uint32_t (&to)[8]) {
#pragma unroll
      for (int j = 0; j < 8; ++j) to[j] = S.v[16 * (j >> 2) + 4 * c + (j & 3)][8 * g + (m & 7)];
    };
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

    // ---- online softmax (log2 domain) of rows m ---------------------------------------
    float mt = sc[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) mt = fmaxf(mt, sc[j]);
    const float need = xor32_max(xor16_max(mt)) * rf;
    if (__any(need > m_ref + kPfLazy)) {
      const float m_new = need > m_ref ? need : m_ref;
      const float fr = m_new == m_ref ? 1.0f : merge_factor(m_ref, m_new);
      l_run *= fr;
#pragma unroll
      for (int g = 0; g < NG; ++g) bs[g] *= fr;
#pragma unroll
      for (int b = 0; b < 4 * NG; ++b) o[b] *= fr;
      m_ref = m_new;
    }
    float pw[8];
    // (with nothing attended so far, -inf - -inf would be NaN)
    const float ms = m_ref == -INFINITY ? 0.0f : m_ref;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      pw[j] = fast_exp2(fmaf(sc[j], rf, -ms));
      l_run += pw[j];
    }

    // ---- O^T += V^T P^T -----------------------------------------------------------------
    float pm = pw[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) pm = fmaxf(pm, pw[j]);
    const uint64_t heavy = __ballot(pm >= 0.5f);
#pragma unroll
    for (int b = 0; b < NG / G4; ++b) {
      v_rows(b);
      if (!inside) {  // a key that this row does not attend may hold anything
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool keep = pw[j] > 0.0f || pw[j] != pw[j];
#pragma unroll
          for (int g = 0; g < G4; ++g) {
            vs[j][g] = keep ? vs[j][g] : static_cast<SB>(0.0f);
            vb[j][g] = keep ? vb[j][g] : static_cast<SB>(0.0f);
          }
        }
      }
#pragma unroll
      for (int gi = 0; gi < G4; ++gi) {
        const int g = G4 * b + gi;
        v_words(g, w);
        float y[8], big = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float s = static_cast<float>(vs[j][gi]);
          y[j] = pw[j] * s;
          bs[g] = fmaf(pw[j], fmaf(s, 8.0f, static_cast<float>(vb[j][gi])), bs[g]);
          big = fmaxf(big, fabsf(y[j]));
        }
        const float in = big * ef[g];
        const uint64_t under = __ballot(in < 1.0f) & heavy;
        if ((__ballot(in > 0x1p15f) | under) != 0) {
          // the row's largest to 2^13 .. 2^14 (an infinity, of exponent 0, stays one)
          const float top = xor32_max(xor16_max(big));
          const float row = top * ef[g];
          const int want = min(14 - __builtin_amdgcn_frexp_expf(top), 120) + 1 - __builtin_amdgcn_frexp_expf(ef[g]);
          int by = row > 0x1p15f ? min(want, 0) : 0;
          if (under != 0) {
            // up as far as the sums stay below 2^100 (weights that much smaller are nothing)
            float most = 0.0f;
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
              for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(o[4 * g + x][e]));
            most = xor32_max(xor16_max(most));
            const int room = most > 0.0f ? 100 - __builtin_amdgcn_frexp_expf(most) : want;
            if (top > 0.0f && row < 1.0f) by = max(min(want, room), 0);
          }
          ef[g] = ldexpf(ef[g], by);
#pragma unroll
          for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[4 * g + x][e] = ldexpf(o[4 * g + x][e], by);
        }
        u32x4 hw, lw;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          hw[q] = few_high(y[2 * q], y[2 * q + 1], ef[g]);
          lw[q] = few_low(hw[q], y[2 * q], y[2 * q + 1], ef[g]);
        }
        pf_settle(hw, lw);
        const v8h bh = __builtin_bit_cast(v8h, hw), bl = __builtin_bit_cast(v8h, lw);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          u32x4 a;
#pragma unroll
          for (int q = 0; q < 4; ++q)  // byte x of two keys' words into the low bytes of the halves
            a[q] = few_centre(__builtin_amdgcn_perm(w[2 * q + 1], w[2 * q], 0x0C040C00u + 0x00010001u * x), vmask, voff);
          v4f& acc = o[4 * g + x];
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), bh, acc, 0, 0, 0);
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), bl, acc, 0, 0, 0);
        }
      }
    }
  }

  // ---- merge of the waves' partials of every row, and the output --------------------
  const float lt = xor32_sum(xor16_sum(l_run));
  if (c == 0) {
    ml[wave][m] = m_ref;
    ll[wave][m] = lt;
  }
  __syncthreads();  // (the stages are behind the partials)
  float* orow = L.o[wave] + m * Gm::OSTR;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const float bg = xor32_sum(xor16_sum(bs[g]));
    const float un = ldexpf(c < 2 ? 1.0f : 0.0625f, 1 - __builtin_amdgcn_frexp_expf(ef[g]));  // high nibbles were 16 times as large
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        orow[64 * g + 8 * (4 * (c & 1) + e) + 2 * x + (c >> 1)] = fmaf(o[4 * g + x][e], un, bg);
  }
  __syncthreads();
  for (int u = tid; u < kFewBlock * (D / 2); u += Gm::NT) {
    const int r = __builtin_amdgcn_readfirstlane(u / (D / 2)), d = 2 * (u % (D / 2));  // a wave's 64 units lie in one row
    const int Ro = r0 + r;
    if (Ro >= total) break;
    float M = -INFINITY;
#pragma unroll
    for (int k = 0; k < NW; ++k) M = fmaxf(M, ml[k][r]);
    float l = 0.0f, x0 = 0.0f, x1 = 0.0f;
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      const float fk = merge_factor(ml[k][r], M);
      const float2 v = *reinterpret_cast<const float2*>(&L.o[k][r * Gm::OSTR + d]);
      l = fmaf(ll[k][r], fk, l);
      x0 = fmaf(v.x, fk, x0);
      x1 = fmaf(v.y, fk, x1);
    }
    if (job.splits == 1) {
      const int qo = Ro / p.gqa;
      const int64_t row = static_cast<int64_t>(qo + job.s0) * p.Hq + job.kvh * p.gqa + (Ro - qo * p.gqa);
      *reinterpret_cast<float2*>(p.out + row * D + d) = make_float2(chunk_result(x0, l), chunk_result(x1, l));
    } else {
      const int64_t slot = static_cast<int64_t>(job.slot) * kFewBlock + r;
      *reinterpret_cast<float2*>(p.ws_o + slot * D + d) = make_float2(x0, x1);
      if (d == 0) *reinterpret_cast<float2*>(p.ws_ml + slot * 2) = make_float2(M, l);
    }
  }
}

}  // namespace
}  // namespace tq
