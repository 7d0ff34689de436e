// What the kernels of windowed attention and of the 4-bit cache share (gfx950):
// matrix operands, the 4-bit cache's layout and conversion, the planes in which
// probabilities enter a product, and what a query sees.
#pragma once

#include <type_traits>

#include "pl_common.h"

namespace pl {
namespace window {

constexpr int kWave = 64;
constexpr int kMaxLen = 1 << 30;   // tokens of a sequence
constexpr int64_t kMaxGroups = 1 << 23;  // workgroups of a launch: under 2^32 threads, 256 each

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// ------------------------------------------------------------ products ---
template <typename T> __device__ __forceinline__ f32x4 mfma32(u32x4 a, u32x4 b, f32x4 c);
template <> __device__ __forceinline__ f32x4 mfma32<bf16_t>(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                 0, 0);
}
template <> __device__ __forceinline__ f32x4 mfma32<f16_t>(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                0);
}

// The largest of the four lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float column_max(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Two floats as fp16, by the packed conversion (to nearest, as pack2's).
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), half2_t));
}

// Probabilities are p = kScale 2^(sc (s - m)), m the running maximum of the products
// q . k themselves that the row's sums are held at, which follows only scores more than
// kLag above it.  The differences s - m come out of the matrix products, whose
// accumulators begin at -m: from a maximum that is scaled and rounded, products of
// millions are whole powers of two away, and a subtraction per score costs 3 % of a
// prompt over 16 bits (256 us, not 250) and, with its registers, a fifth over 4 (212,
// not 173).
// They enter the product with V in planes of its type, each what the one before left:
// three of bf16, cut, hold the 24 bits of fp32, two of fp16, rounded to nearest, 22 of
// them, as in decode and tree attention.  Two planes of bf16 leave 2^-16, which is past
// an output's rounding where the terms cancel to 2^-8 of themselves.
// bf16: p <= 2^-24, so that the sums over 2^24 tokens of the largest V are finite;
// the planes end at 2^-126, 2^-94 of the row's largest weight or less.  fp16: p <= 2^15,
// near the range's top; the planes end at 2^-25, 2^-36 of the largest weight or less.
template <typename MT> struct Planes;
template <> struct Planes<bf16_t> {
  static constexpr int kPlanes = 3;
  static constexpr float kLag = 8.f, kShift = -32.f, kScale = 0x1p-32f;
  // (the factor is a product of its own: in the exponent, 32 would take 5 of the bits)
  __device__ static __forceinline__ float weight(float s, float sc) { return fast_exp2(s * sc) * kScale; }
  __device__ static __forceinline__ void split(float a, float b, uint32_t (&w)[kPlanes]) {
#pragma unroll
    for (int i = 0; i < kPlanes; ++i) {
      const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
      w[i] = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
      a -= __uint_as_float(ua & 0xffff0000u);
      b -= __uint_as_float(ub & 0xffff0000u);
    }
  }
};
template <> struct Planes<f16_t> {
  static constexpr int kPlanes = 2;
  static constexpr float kLag = 4.f, kShift = 11.f, kScale = 0x1p11f;
  // (in the exponent, which 11 leaves off by 2^-21 at most, no more than the planes are)
  __device__ static __forceinline__ float weight(float s, float sc) { return fast_exp2(__builtin_fmaf(s, sc, kShift)); }
  __device__ static __forceinline__ void split(float a, float b, uint32_t (&w)[kPlanes]) {
    const half2_t h = __builtin_convertvector((f32x2{a, b}), half2_t);
    w[0] = __builtin_bit_cast(uint32_t, h);
    w[1] = pack_half(__builtin_fmaf((float)h.x, -1.f, a), __builtin_fmaf((float)h.y, -1.f, b));
  }
};

// What sums held at the maximum m count for at the maximum `top` >= m: nothing where
// nothing was seen (m of -inf, which `top` may be too).
__device__ __forceinline__ float weight(float m, float top, float sc) {
  return m == -INFINITY ? 0.f : fast_exp2((m - top) * sc);
}

// A row's maximum follows the differences of its scores from it, whose largest is
// `top`: they go down by `up` (so that the largest is 0, whatever m + up rounds to),
// sums by alpha.
struct Rise {
  float up, alpha;
};
__device__ __forceinline__ Rise rise_to(float top, float& m, float sc) {
  const bool first = m == -INFINITY;  // nothing was seen yet: the differences are from 0
  const float up = first ? (top == -INFINITY ? 0.f : top) : fmaxf(top, 0.f);
  const Rise r{up, first ? 0.f : fast_exp2(-up * sc)};
  m = first ? top : m + up;
  return r;
}

// ---------------------------------------------------------- 4-bit cache ---
// Of a page and kv head: the codes of `page` tokens, then their scales.  K goes by
// tokens: codes [token][D / 2 bytes], scales [token][D / 32].  V goes by four
// tokens, as the lanes of a V^T operand hold them: codes [token / 4][d / 8]
// [token % 4][4 bytes], scales [token / 4][d / 32][token % 4].
constexpr int kGroup = 32;                     // values that share a scale
constexpr int kScaleMin = 2, kScaleMax = 252;  // 2^(s - 127): every value is a normal bf16
constexpr int kScaleZero = 127;                // every value is 0: a scale that any product's type holds
constexpr int kScaleNan = 255;                 // the group held a NaN or an infinity

// A scale byte as the conversions take it.
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// Codes 2 S, 2 S + 1 of a word as two bf16: exact, and NaN where the scale is kScaleNan.
template <int S> __device__ __forceinline__ uint32_t codes2(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, S));
}
// The eight codes of a word.
__device__ __forceinline__ u32x4 codes8(uint32_t w, float scale) {
  return u32x4{codes2<0>(w, scale), codes2<1>(w, scale), codes2<2>(w, scale), codes2<3>(w, scale)};
}

// And as fp16: exact where 2^-14 <= 0.5 scale and 6 scale is in its range.
template <int S> __device__ __forceinline__ uint32_t halves2(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, S));
}
__device__ __forceinline__ u32x4 halves8(uint32_t w, float scale) {
  return u32x4{halves2<0>(w, scale), halves2<1>(w, scale), halves2<2>(w, scale), halves2<3>(w, scale)};
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pk_min(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ uint32_t pk_max(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

// --------------------------------------------------------------- window ---
// What the queries at positions p0 .. see: positions from `lo` on (the window of
// p0), and those before `se` (sinks).  Tiles of `tile` positions are counted by
// what is seen: `ns` of sinks, then on from tile `fw`.
struct Seen {
  int lo, se, ns, fw;
};
__host__ __device__ __forceinline__ Seen seen_from(int p0, int window, int sinks, int tile) {
  Seen s;
  s.lo = window > 0 && p0 >= window ? p0 - window + 1 : 0;
  s.se = sinks < s.lo ? sinks : s.lo;
  s.fw = s.lo / tile;
  const int t = (s.se + tile - 1) / tile;
  s.ns = t < s.fw ? t : s.fw;
  return s;
}
// The place of seen tile i among all tiles.
__host__ __device__ __forceinline__ int seen_tile(const Seen& s, int i) { return i < s.ns ? i : i - s.ns + s.fw; }

// A sum of a part that counts with weight w >= 0: an infinity stays one however
// small its weight.
__device__ __forceinline__ float weighted(float v, float w) {
  return w == 0.f && fabsf(v) == INFINITY ? v : v * w;
}

__device__ __forceinline__ bool finite16(uint32_t half, bool bf16) {
  const uint32_t mask = bf16 ? 0x7f80u : 0x7c00u;
  return (half & mask) != mask;
}

}  // namespace window
}  // namespace pl
