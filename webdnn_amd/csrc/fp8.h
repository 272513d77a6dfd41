// The 8-bit type of the serving operators: e4m3 as the OCP 8-bit floating point specification defines it (1 sign, 4 exponent
// and 3 fraction bits, bias 7, largest value 448, steps of 2^-9 below 2^-6, no infinities, NaN = 0x7f or 0xff), and the
// scales that go with it.
#pragma once
#include <hip/hip_runtime.h>
#include <float.h>
#include <math.h>

#include "rowmath.h"

namespace wdh {
namespace fp8 {

constexpr int BLOCK = 128;               // elements along a row that share a scale
constexpr float E4M3_MAX = 448.0f;
constexpr float LEAST_SCALE = 7.8886090522101181e-31f;  // 2^-100: its reciprocal and the elements' quotients are numbers of fp32

// Rows need not start on 16-byte boundaries (odd lengths): global loads and stores of four elements take any address.
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef int i32_any __attribute__((aligned(1)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// A number the compiler knows nothing about: what is computed from it stays where it is used and holds no registers in between.
__device__ __forceinline__ int fresh(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// |x| if x is finite, else 0: a block's scale follows its finite elements.
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= FLT_MAX ? a : 0.0f;
}
// The largest of the 32 lanes of each half wavefront, in all of them.
__device__ __forceinline__ float half_max(float v) {
  using namespace rowmath;
  v = fmaxf(v, dpp_take<DPP_XOR1, 0xf>(0.0f, v));
  v = fmaxf(v, dpp_take<DPP_XOR2, 0xf>(0.0f, v));
  v = fmaxf(v, dpp_take<DPP_HALF_MIRROR, 0xf>(0.0f, v));
  v = fmaxf(v, dpp_take<DPP_MIRROR, 0xf>(0.0f, v));
  return fmaxf(v, __shfl_xor(v, 16, 64));
}
// The scale of a block whose largest finite magnitude is `amax`.
__device__ __forceinline__ float block_scale(float amax) { return fmaxf(amax / E4M3_MAX, LEAST_SCALE); }

// Four elements, two to a conversion, packed in order: rounded to the nearest e4m3 value, ties to even.
__device__ __forceinline__ int convert4(f32x4 v) {
  int q = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], q, true);
}
// Four elements times `inv` to e4m3, for scales that are powers of two: nothing is rounded but the result.  What is not finite becomes NaN.
__device__ __forceinline__ int pack4(f32x4 v, float inv) {
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = fabsf(v[e]) <= FLT_MAX ? v[e] * inv : NAN;
  return convert4(v);
}

// A block's scale as a divisor.  Quotients have to be the fp32 ones: a product with the reciprocal is up to 1.5 steps of fp32 off, and where that
// crosses the middle between two e4m3 values (1 of 10^4 to 10^5 elements) the result is a whole step of e4m3 off.
// Two corrections q <- q + r (v - q c) with the rounded reciprocal r: the first leaves a quotient less than a step off, whose remainder
// is exact, and the second is the quotient rounded to nearest (Markstein's theorem).  Remainders of blocks below 2^-40 could be among the
// subnormal numbers: those are worked on 2^60 times as large.
// Cost (us, so / with the reciprocal alone): quantisation of 5000 rows of 8192 38.4 / 37.9, of 30000 x 1030 in 128 x 128 35.7 / 35.4.
struct Divisor {
  float c, r, up;
};
__device__ __forceinline__ Divisor divisor(float c) {
  Divisor d;
  d.up = c < 0x1p-40f ? 0x1p60f : 1.0f;
  d.c = c * d.up;
  d.r = 1.0f / d.c;
  return d;
}
// Four elements over their block's scale to e4m3.  What is not finite becomes NaN (the remainder of an infinity is none); a quotient beyond 448
// is at most 448 (1 + 2^-22) and rounds to 448.  (Quotients that are subnormal numbers of fp32 may be off: they are 0 as e4m3.)
__device__ __forceinline__ int divide4(f32x4 v, Divisor d) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const float x = v[e] * d.up;
    float q = x * d.r;
    q = __builtin_fmaf(__builtin_fmaf(-q, d.c, x), d.r, q);
    q = __builtin_fmaf(__builtin_fmaf(-q, d.c, x), d.r, q);
    v[e] = copysignf(q, x);  // (the corrections make -0 a 0)
  }
  return convert4(v);
}

// Elements idx .. idx+3 of a row of `len` (0 beyond its end), and back.
__device__ __forceinline__ f32x4 load4(const float *row, long long idx, long long len) {
  if (idx + 4 <= len) return *reinterpret_cast<const f32x4_any *>(row + idx);
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 3; e++)
    if (idx + e < len) v[e] = row[idx + e];
  return v;
}
__device__ __forceinline__ void store4(float *row, long long idx, long long len, f32x4 v) {
  if (idx + 4 <= len) {
    *reinterpret_cast<f32x4_any *>(row + idx) = v;
    return;
  }
#pragma unroll
  for (int e = 0; e < 3; e++)
    if (idx + e < len) row[idx + e] = v[e];
}
__device__ __forceinline__ void store4_bytes(unsigned char *row, long long idx, long long len, int q) {
  if (idx + 4 <= len) {
    *reinterpret_cast<i32_any *>(row + idx) = q;
    return;
  }
#pragma unroll
  for (int e = 0; e < 3; e++)
    if (idx + e < len) row[idx + e] = (unsigned char)(q >> (8 * e));
}

// Products of e4m3 values run on the bfloat16 matrix instructions, at half the rate of the 8-bit ones: those add groups of
// eight products with about 16 bits below the largest (measured: 65536 + 127 * 1 gives 65656, and sums of 128 products of normal
// values are 1.4e-5 off in 2-norm, where these are 1e-8 off).
// Eight e4m3 values as bfloat16 (exact: 4 significant bits of 8).
__device__ __forceinline__ bf16x8 widen(int lo, int hi) {
  union { bf16x2 h[4]; bf16x8 v; } u;
  u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, 1.0f, false);
  u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, 1.0f, true);
  u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, 1.0f, false);
  u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, 1.0f, true);
  return u.v;
}
// ... and as float16 (exact as well: 2^-9 to 448).
__device__ __forceinline__ f16x8 widen_f16(int lo, int hi) {
  union { f16x2 h[4]; f16x8 v; } u;
  u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((unsigned)lo, 1.0f, false);
  u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((unsigned)lo, 1.0f, true);
  u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((unsigned)hi, 1.0f, false);
  u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((unsigned)hi, 1.0f, true);
  return u.v;
}

}  // namespace fp8
}  // namespace wdh
