// Rotation of the elements of a head by the angles of its token's position, after a root-mean-square norm of the head, four elements to a lane.
//
// Element pairs (a, b) of the first 2 half elements, (x[j], x[j + half]) or (x[2j], x[2j + 1]), become
//   (a cos_j - b sin_j, b cos_j + a sin_j),  cos_j and sin_j from the position's rows of two tables;
// the elements behind them stay.  A lane needs the partners of its four elements too.  Where it does not hold them, they come from the lane that does, if that is a
// bit of the lane's number away (wdh_rope alone); else they are loaded again, from cache, so that pairs may lie anywhere in the head.
#pragma once
#include "fp8.h"

namespace wdh {
namespace rope {

using namespace wdh::fp8;

struct Rotation {
  const float *cos, *sin;  // [rows][half]
  int half, rows;
};
// Which pairs there are: (x[2j], x[2j + 1]), in a lane's four elements both; (x[j], x[j + half]) of a whole head, where a lane has four elements of the lower half
// and their partners; the same with partners in a lane that differs in one bit of its number; or anywhere in the head.
enum Pairs { NEIGHBOURS, FACING, EXCHANGED, ANYWHERE };
typedef float f32x2_any __attribute__((ext_vector_type(2), aligned(4)));

// The partners, ANYWHERE, of elements d0 .. d0+3 of `from` (a head, or what it is multiplied with), 0 where there are none.
__device__ __forceinline__ f32x4 partners(const Rotation &r, const float *from, int d0, int d) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (d0 >= 2 * r.half) return v;
  if (r.half % 4 == 0) return load4(from, d0 < r.half ? d0 + r.half : d0 - r.half, d);
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (d0 + e < 2 * r.half) v[e] = from[d0 + e < r.half ? d0 + e + r.half : d0 + e - r.half];
  return v;
}

// What elements d0 .. d0+3 (FACING: of the lower half) and their partners are multiplied with; a position outside the tables makes the rotated ones NaN.
struct Angles {
  f32x4 c, s;
};
template <int PAIRS>
__device__ __forceinline__ Angles angles(const Rotation &r, int position, int d0) {
  Angles a = {{1.f, 1.f, 1.f, 1.f}, {0.f, 0.f, 0.f, 0.f}};
  if (PAIRS != FACING && d0 >= 2 * r.half) return a;
  if (position < 0 || position >= r.rows) {
#pragma unroll
    for (int e = 0; e < 4; e++) a.c[e] = a.s[e] = NAN;
    return a;
  }
  const float *cos = r.cos + (long long)position * r.half, *sin = r.sin + (long long)position * r.half;
  if constexpr (PAIRS == FACING) {
    a.c = *reinterpret_cast<const f32x4_any *>(cos + d0);
    a.s = -*reinterpret_cast<const f32x4_any *>(sin + d0);
  } else if constexpr (PAIRS == NEIGHBOURS) {
    const int j = d0 / 2;
    const bool two = j + 1 < r.half;
    const f32x2_any c = two ? *reinterpret_cast<const f32x2_any *>(cos + j) : f32x2_any{cos[j], 1.0f}, s = two ? *reinterpret_cast<const f32x2_any *>(sin + j) : f32x2_any{sin[j], 0.0f};
    a.c = f32x4{c[0], c[0], c[1], c[1]};
    a.s = f32x4{-s[0], s[0], -s[1], s[1]};
  } else if (r.half % 4 == 0) {
    const int j = d0 < r.half ? d0 : d0 - r.half;
    a.c = load4(cos, j, r.half);
    a.s = load4(sin, j, r.half);
    if (d0 < r.half) a.s = -a.s;
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (d0 + e < 2 * r.half) {
        const int j = d0 + e < r.half ? d0 + e : d0 + e - r.half;
        a.c[e] = cos[j];
        a.s[e] = d0 + e < r.half ? -sin[j] : sin[j];
      }
  }
  return a;
}

// The elements turned: two products, the second rounded before it is added.
__device__ __forceinline__ f32x4 turn(const Rotation &r, int d0, f32x4 own, f32x4 other, Angles a) {
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (d0 + e < 2 * r.half) own[e] = __builtin_fmaf(own[e], a.c[e], other[e] * a.s[e]);
  return own;
}
__device__ __forceinline__ f32x4 turn_neighbours(const Rotation &r, int d0, f32x4 v, Angles a) { return turn(r, d0, v, f32x4{v[1], v[0], v[3], v[2]}, a); }
__device__ __forceinline__ void turn_facing(f32x4 &low, f32x4 &high, Angles a) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const float x = low[e];
    low[e] = __builtin_fmaf(x, a.c[e], high[e] * a.s[e]);
    high[e] = __builtin_fmaf(high[e], a.c[e], x * -a.s[e]);
  }
}

constexpr int DPP_ROTATE8 = 0x128;  // lanes of a row of 16 that are 8 apart

// Sums over groups of LANES neighbouring lanes, in all of them.
template <int CTRL>
__device__ __forceinline__ double dpp_add_d(double v) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (unsigned)b, CTRL, 0xf, 0xf, false);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (unsigned)(b >> 32), CTRL, 0xf, 0xf, false);
  return v + __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
template <int LANES>
__device__ __forceinline__ double group_sum(double v) {
  v = dpp_add_d<rowmath::DPP_XOR1>(v);
  v = dpp_add_d<rowmath::DPP_XOR2>(v);
  if constexpr (LANES >= 8) v = dpp_add_d<rowmath::DPP_HALF_MIRROR>(v);
  if constexpr (LANES >= 16) v = dpp_add_d<rowmath::DPP_MIRROR>(v);
  if constexpr (LANES >= 32) v += __shfl_xor(v, 16, 64);
  if constexpr (LANES >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}
__device__ __forceinline__ double squares(f32x4 v) {
  double sum = 0.0;
#pragma unroll
  for (int e = 0; e < 4; e++) sum = fma((double)v[e], (double)v[e], sum);
  return sum;
}
// A head's sum of squares in the order in which wdh_rope adds it, whose lanes have the pieces of both halves of a head of 64 or 128 (of 32: one of eight pieces), for
// lanes that have one of its pieces each, and for those that have two which face each other: the factor's bits, and with them those of the
// cache, may hang on it.
template <int D>
__device__ __forceinline__ double head_squares(f32x4 own) {
  const double v = squares(own);
  if constexpr (D == 32) return group_sum<8>(v);
  else if constexpr (D == 64) return group_sum<8>(dpp_add_d<DPP_ROTATE8>(v));
  else return group_sum<16>(v + __shfl_xor(v, 16, 64));
}
template <int D>
__device__ __forceinline__ double head_squares(f32x4 low, f32x4 high) {
  if constexpr (D == 32) return group_sum<4>(squares(low)) + group_sum<4>(squares(high));
  else return group_sum<D / 8>(squares(low) + squares(high));
}
// What a head's elements are multiplied with, from the mean of their squares.  Division and root of 64 bits are some 40 instructions for a number that is
// rounded to 32; instead the instruction's root, good to 2^-26 or so, and one step of Newton's, y + y (1 - m y^2) / 2, which leaves 1.5 of that
// squared (0 and infinity are their own).  Six prompts' keys on their way into a cache: 48.5 us with division and root, 44.2 without.
__device__ __forceinline__ rowmath::RowFactor head_factor(double mean, float eps) {
  const double m = mean + (double)eps, y = __builtin_amdgcn_rsq(m);
  double t = __builtin_fma(__builtin_fma(-m * y, y, 1.0), 0.5 * y, y);
  t = m > 0.0 && m <= DBL_MAX ? t : y;
  if (t > 0x1p100) return rowmath::RowFactor{0x1p60f, (float)(t * 0x1p-60)};
  if (t < 0x1p-100) return rowmath::RowFactor{0x1p-40f, (float)(t * 0x1p40)};
  return rowmath::RowFactor{1.0f, (float)t};
}
// Elements by their head's factor and weights, rounded as wdh_rmsnorm rounds them.
__device__ __forceinline__ f32x4 normed(f32x4 v, rowmath::RowFactor f, f32x4 gamma) {
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = v[e] * f.power * f.t * gamma[e];
  return v;
}

}  // namespace rope
}  // namespace wdh
