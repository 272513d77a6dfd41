// Rotation of the elements of a head by the angles of its token's position, after a root-mean-square norm of the head, four elements to a lane.
//
// Element pairs (a, b) of the first 2 half elements, (x[j], x[j + half]) or (x[2j], x[2j + 1]), become
//   (a cos_j - b sin_j, b cos_j + a sin_j),  cos_j and sin_j from the position's rows of two tables;
// the elements behind them stay.  A lane needs the partners of its four elements too: they are loaded again, from cache, rather than
// exchanged, so that pairs may lie anywhere in the head.
#pragma once
#include "fp8.h"

namespace wdh {
namespace rope {

using namespace wdh::fp8;

struct Rotation {
  const float *cos, *sin;  // [rows][half]
  int half, rows;
  int interleaved;
};

// The partners of elements d0 .. d0+3 of `from` (a head, or what it is multiplied with), 0 where there are none.
__device__ __forceinline__ f32x4 partners(const Rotation &r, const float *from, int d0, int d) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (d0 >= 2 * r.half) return v;
  if (r.interleaved) {
    const f32x4 x = load4(from, d0, d);
    return f32x4{x[1], x[0], x[3], x[2]};
  }
  if (r.half % 4 == 0) return load4(from, d0 < r.half ? d0 + r.half : d0 - r.half, d);
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (d0 + e < 2 * r.half) v[e] = from[d0 + e < r.half ? d0 + e + r.half : d0 + e - r.half];
  return v;
}

// What elements d0 .. d0+3 and their partners are multiplied with; a position outside the tables makes the rotated ones NaN.
struct Angles {
  f32x4 c, s;
};
__device__ __forceinline__ Angles angles(const Rotation &r, int position, int d0) {
  Angles a = {{1.f, 1.f, 1.f, 1.f}, {0.f, 0.f, 0.f, 0.f}};
  if (d0 >= 2 * r.half) return a;
  if (position < 0 || position >= r.rows) {
#pragma unroll
    for (int e = 0; e < 4; e++) a.c[e] = a.s[e] = NAN;
    return a;
  }
  const float *cos = r.cos + (long long)position * r.half, *sin = r.sin + (long long)position * r.half;
  if (r.interleaved) {
#pragma unroll
    for (int e = 0; e < 4; e += 2)
      if (d0 + e < 2 * r.half) {
        a.c[e] = a.c[e + 1] = cos[(d0 + e) / 2];
        a.s[e + 1] = sin[(d0 + e) / 2];
        a.s[e] = -a.s[e + 1];
      }
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
  v = dpp_add_d<rowmath::DPP_HALF_MIRROR>(v);
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
// Elements by their head's factor and weights, rounded as wdh_rmsnorm rounds them.
__device__ __forceinline__ f32x4 normed(f32x4 v, rowmath::RowFactor f, f32x4 gamma) {
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = v[e] * f.power * f.t * gamma[e];
  return v;
}

}  // namespace rope
}  // namespace wdh
