// K/V tiles of the multi-query kernels (tq_prefill.hip over one cache,
// tq_paged_tiles.hip over pages) in LDS: their geometry, the staging of a tile
// from registers, and the range of its V scales.  tq_prefill.hip has the
// mathematics.
#pragma once

#include "tq_sdpa_common.h"

#include <type_traits>

namespace tq {
namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// A running reference moves only when a score passes it by this much (log2).
constexpr float kPfLazy = 8.0f;
// With 2^e0 above every V scale of a workgroup's first tile: p s_v is below
// 2^kPfHead for the row's largest weight and a scale of 2^e0, and below 2^15 (fp16
// overflows at 2^16) for scales up to 2^(e0 + kPfUp).  Scales down to
// 2^(e0 - kPfDown) leave such a weight 19 bits above fp16's step (3 more than bf16
// parts would).  A tile outside these bounds costs half as much again: with every
// tile so (one group of 64 dims at 2^-12), 512 queries after 3,584 keys, 85
// instead of 63 us (Hq 32 Hkv 16 D 256, window 1,024) and 578 instead of 387
// (Hq 32 Hkv 4 D 512).
constexpr int kPfHead = 4, kPfUp = 3, kPfDown = 9;

template <int D, bool F32, int RS>
struct PfGeom {
  using SB = typename std::conditional<F32, float, _Float16>::type;
  static constexpr int W = D / 8;        // packed words per row
  static constexpr int NG = D / 64;      // quant groups per row
  static constexpr int DH = D == 512 ? 2 : 1;  // waves that share a row set's dims
  static constexpr int KH = 2 / DH;            // 32-key parts of a tile
  static constexpr int NW_ = NG / DH;          // groups of a wave
  static constexpr int OW = D / DH;            // dims of a wave
  static constexpr int TK = 32 * KH, NW = RS * KH * DH, NT = 64 * NW;
  // 16-byte units of a 16-key slice of K (8 NG operands) and of V^T per 32 keys
  // (4 NG operands).  An operand is 64 units [c][m]; unit m sits at m ^ swizzle(g),
  // so that the 16 lanes of a store (of several groups) reach distinct banks, as
  // those of a read do.
  static constexpr int KU = 64 * 2 * NG, VU = 64 * 4 * NG;
  static __device__ __forceinline__ constexpr int kswz(int g) { return (16 / NG) * g; }
  static __device__ __forceinline__ constexpr int vswz(int g) { return 8 * (g & 1); }
  static constexpr int UNITS = TK * W / 8;                      // 8-word staging units of K; as many of V
  static constexpr int NU = (2 * UNITS + NT - 1) / NT;
  static constexpr int SDW = TK * NG * static_cast<int>(sizeof(SB)) / 4;  // dwords of one scale tensor a tile
  static constexpr int NSD = (4 * SDW + NT - 1) / NT;
  static constexpr int NSW = SDW / 64;   // waves that stage one of them
  static constexpr int OSTR = OW + 2;    // partial output rows (floats): conflict-free 4-byte stores
  struct Stage {
    u32x4 k[2][2 * KH * KU];             // [16-key slice][g][s][c][key]: word 8 g + 2 c + s
    u32x4 v[2][KH * VU];                 // [kh][g][x][c][dim row]: slots 0-7 of lane group c
    SB sb[2][4][TK * NG];                // k scale, k bias, v scale, v bias
    v4f xch[DH == 2 ? NW : 1][2][64];    // score parts of a row set's waves
  };
  union Lds {
    Stage st;
    float o[NW][16 * OSTR];
  };
  static_assert(SDW % 64 == 0 && UNITS % 64 == 0, "wave-uniform staging roles");
};

// One tile's words and scales, in this thread's registers: a unit is 8 words
// of a key (K), or one word of the 8 keys of a lane group's slots (V).
template <class Gm>
struct PfRaw {
  uint32_t w[Gm::NU][8];
  uint32_t s[Gm::NSD];
};

// Nibbles in bits 0-3 (HI: 4-7) of both halves of t as fp16 n - 8 (16 (n - 8)).
// mask: 0x000F000F (0x00F000F0) in a vector register -- as a literal beside the
// other one, the AND and the OR are two instructions.
template <bool HI>
__device__ __forceinline__ uint32_t pf_centre(uint32_t t, uint32_t mask) {
  uint32_t b;  // 1024 + n, 1024 + 16 n
  asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(b) : "v"(t), "v"(mask), "s"(0x64006400u));
  const _Float16 off = static_cast<_Float16>(HI ? -1152.0f : -1032.0f);
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, b) + v2h{off, off});
}

// Whether this thread's V scales are all within [2^(e0 - kPfDown), 2^(e0 + kPfUp)),
// per wave that stages some, into ok[NSW].
template <class Gm>
__device__ __forceinline__ void pf_alike(const PfRaw<Gm>& R, int e0, int* ok) {
  constexpr bool kHalf = sizeof(typename Gm::SB) == 2;
  // the bounds' bit patterns: magnitudes order as these do
  const auto bits = [](float x) -> uint32_t {
    if constexpr (kHalf) return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x));
    else return __float_as_uint(x);
  };
  const uint32_t lo = bits(ldexpf(1.0f, e0 - kPfDown)), n = bits(ldexpf(1.0f, e0 + kPfUp)) - lo;
#pragma unroll
  for (int i = 0; i < Gm::NSD; ++i) {
    const int e = threadIdx.x + i * Gm::NT;
    if (__builtin_amdgcn_readfirstlane(e / Gm::SDW) != 2) continue;
    const uint32_t a = R.s[i];
    bool in;
    if constexpr (kHalf) in = (a & 0x7FFFu) - lo < n && (a >> 16 & 0x7FFFu) - lo < n;
    else in = (a & 0x7FFFFFFFu) - lo < n;
    ok[e % Gm::SDW / 64] = __all(in);  // (one value from every lane)
  }
}

// Words into LDS buffer b.
template <class Gm, class Stage>
__device__ __forceinline__ void pf_store_words(Stage& S, const PfRaw<Gm>& R, int b) {
  const uint32_t mlo = 0x000F000Fu, mhi = 0x00F000F0u;
#pragma unroll
  for (int i = 0; i < Gm::NU; ++i) {
    const int e = threadIdx.x + i * Gm::NT;
    const int role = __builtin_amdgcn_readfirstlane(e / Gm::UNITS);
    const int u = e % Gm::UNITS;
    if (role == 0) {
      // word 8 g + 2 c + s: nibbles 0, 4, 1, 5, 2, 6, 3, 7
      const int r = u / Gm::NG, g = u % Gm::NG;
      u32x4* d = &S.k[b][(r >> 4) * Gm::KU + 128 * g + ((r & 15) ^ Gm::kswz(g))];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t w = R.w[i][k], h = w >> 8;
        d[64 * (k & 1) + 16 * (k >> 1)] =
            u32x4{pf_centre<false>(w, mlo), pf_centre<true>(w, mhi), pf_centre<false>(h, mlo), pf_centre<true>(h, mhi)};
      }
    } else if (role == 1) {
      const int w = u % Gm::W, kc = u / Gm::W;
      const int g = w >> 3;
      u32x4* d = &S.v[b][(kc >> 2) * Gm::VU + 256 * g + (kc & 3) * 16 + (w & 7)];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        u32x4 lo, hi;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          // byte x of two keys' words into the low bytes of the halves
          const uint32_t t = __builtin_amdgcn_perm(R.w[i][2 * q + 1], R.w[i][2 * q], 0x0C040C00u + 0x00010001u * x);
          lo[q] = pf_centre<false>(t, mlo);
          hi[q] = pf_centre<true>(t, mhi);
        }
        d[64 * x + Gm::vswz(g)] = lo;
        d[64 * x + (8 ^ Gm::vswz(g))] = hi;
      }
    }
  }
}

// Words, scales and biases into LDS buffer b.
template <class Gm>
__device__ __forceinline__ void pf_store(typename Gm::Stage& S, const PfRaw<Gm>& R, int b) {
  pf_store_words<Gm>(S, R, b);
#pragma unroll
  for (int i = 0; i < Gm::NSD; ++i) {
    const int e = threadIdx.x + i * Gm::NT;
    const int t = __builtin_amdgcn_readfirstlane(e / Gm::SDW);
    if ((4 * Gm::SDW) % Gm::NT != 0 && t >= 4) continue;
    reinterpret_cast<uint32_t*>(S.sb[b][0])[e] = R.s[i];
  }
}

// The largest |V scale| of the wave's part of a tile, 0 where it has none.
template <class Gm>
__device__ __forceinline__ float pf_vmax(const PfRaw<Gm>& R) {
  float mx = 0.0f;
#pragma unroll
  for (int i = 0; i < Gm::NSD; ++i) {
    const int e = threadIdx.x + i * Gm::NT;
    if (__builtin_amdgcn_readfirstlane(e / Gm::SDW) != 2) continue;
    if constexpr (sizeof(typename Gm::SB) == 2) {
      const v2h h = __builtin_bit_cast(v2h, R.s[i]);
      mx = fmaxf(mx, fmaxf(fabsf(static_cast<float>(h[0])), fabsf(static_cast<float>(h[1]))));
    } else {
      mx = fmaxf(mx, fabsf(__uint_as_float(R.s[i])));
    }
  }
  return wave_max_dpp(mx);
}

// The fp16 remainders x0 - h0, x1 - h1 of a pair whose fp16 high parts are
// packed in hp, as a packed fp16 pair: one mixed-precision fma each.  The
// difference is exact in fp32 and rounded once, to fp16.
__device__ __forceinline__ uint32_t pf_rem_pair(uint32_t hp, float x0, float x1) {
  uint32_t r;
  asm("v_fma_mixlo_f16 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]\n\t"
      "v_fma_mixhi_f16 %0, %1, -1.0, %3 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
      : "=&v"(r)
      : "v"(hp), "v"(x0), "v"(x1));
  return r;
}

// Operands of matrix instructions that inline assembly has written go through this.  A
// matrix instruction may read what a vector instruction writes two wait states later at
// the earliest; the compiler sees to that for its own instructions and does not look into
// assembly.  (With one state less a kernel of D 512 multiplied V by what half of a
// register had held before.)
__device__ __forceinline__ void pf_settle(u32x4& a) { asm("s_nop 1" : "+v"(a)); }
__device__ __forceinline__ void pf_settle(u32x4& a, u32x4& b) { asm("s_nop 1" : "+v"(a), "+v"(b)); }

}  // namespace
}  // namespace tq
