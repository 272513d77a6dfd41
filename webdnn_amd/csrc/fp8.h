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
constexpr float LEAST_SCALE = 7.8886090522101181e-31f;  // 2^-100: products of two scales and their quotients stay normal numbers

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

// Four elements times `inv` (the reciprocal of their block's scale) to e4m3, rounded to nearest even, packed in order.  What is
// not finite becomes NaN.  A quotient beyond 448 is at most 448 (1 + 2^-22) and rounds to 448.
__device__ __forceinline__ int pack4(f32x4 v, float inv) {
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = fabsf(v[e]) <= FLT_MAX ? v[e] * inv : NAN;
  int q = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], q, true);
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
