// Root-mean-square normalisation of rows (with the residual's addition before it and an 8-bit output behind it) and
// quantisation to e4m3 in blocks.
//
// The reference has no such operators; in its terms the first is the chain Add, Mul, ReduceMean, Add, Sqrt, Div, Mul
// (src/descriptor_runner/operators/cpu/operators/standard/binary7.ts:24-75, reduce.ts:369-405, unary.ts:10-32):
//   s = x + r,  y = (s * t) * g  with  t = 1 / sqrt(mean(s^2) + eps).
// Squares are summed in double (a row of values near 1e20 keeps a finite mean), t is rounded to fp32 once; where it would leave fp32's
// normal numbers (rows of subnormal numbers, or near the largest), a power of two goes into the row's elements first.
// 8 bits: c = max(largest finite |y| of a block / 448, 2^-100), q = e4m3(y / c), the quotient rounded to fp32 first.
//
// Bound: memory.  Every element is read once and written once: a row stays in registers between its sum and its use (8192 rows of 4096
// with residual, sum and 8-bit output: 81.5 us, 5.4 TB/s; quantisation of 5000 rows of 8192: 38.4 us, 5.3 TB/s).
#include "common.h"
#include "fastdiv.h"
#include "fp8.h"

namespace {

using namespace wdh::fp8;

struct NormParams {
  const float *X, *R, *G;
  float *S, *Y;
  unsigned char *Q;
  float *QS;
  long long outer;
  int len, blocks;
  float eps;
};

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// A row's factor as two: t, rounded, and a power of two, 1 for all but extreme rows.
struct RowFactor {
  float power, t;
};
__device__ __forceinline__ RowFactor row_factor(double mean, float eps) {
  const double t = 1.0 / sqrt(mean + (double)eps);
  if (t > 0x1p100) return RowFactor{0x1p60f, (float)(t * 0x1p-60)};
  if (t < 0x1p-100) return RowFactor{0x1p-40f, (float)(t * 0x1p40)};
  return RowFactor{1.0f, (float)t};
}

// One piece (elements idx .. idx+3 of `row`) on its way out; the 32 lanes of a half wavefront hold the 128 elements of a block.
__device__ __forceinline__ void finish_piece(const NormParams &p, long long row, int idx, bool live, RowFactor f, f32x4 v, f32x4 g) {
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = v[e] * f.power * f.t;
  if (p.G)
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = v[e] * g[e];
  if (p.Y && live) store4(p.Y + row * p.len, idx, p.len, v);
  if (!p.Q) return;
  float amax = 0.0f;
#pragma unroll
  for (int e = 0; e < 4; e++) amax = fmaxf(amax, idx + e < p.len ? finite_abs(v[e]) : 0.0f);
  const float c = block_scale(half_max(amax));
  if (!live) return;
  store4_bytes(p.Q + row * p.len, idx, p.len, divide4(v, divisor(c)));
  if ((threadIdx.x & 31) == 0 && idx < p.len) p.QS[row * p.blocks + idx / BLOCK] = c;
}

// WAVES wavefronts to a row, NP pieces of four elements to a lane: a row of up to 256 * WAVES * NP elements in registers.
template <int WAVES, int NP>
__global__ __launch_bounds__(WAVES < 4 ? 256 : 64 * WAVES) void rmsnorm_rows(NormParams p) {
  constexpr int ROWS = WAVES < 4 ? 4 / WAVES : 1;
  __shared__ double part[ROWS * WAVES];
  const int wave = threadIdx.x >> 6, t = threadIdx.x % (64 * WAVES);
  for (long long row0 = (long long)blockIdx.x * ROWS; row0 < p.outer; row0 += (long long)gridDim.x * ROWS) {
    const bool live = row0 + wave / WAVES < p.outer;
    const long long row = live ? row0 + wave / WAVES : p.outer - 1;  // idle wavefronts repeat the last row and store nothing
    const float *x = p.X + row * p.len;
    f32x4 v[NP], g[NP];
#pragma unroll
    for (int i = 0; i < NP; i++) v[i] = load4(x, 4 * (t + 64 * WAVES * i), p.len);
    if (p.R) {
      const float *r = p.R + row * p.len;
      f32x4 w[NP];
#pragma unroll
      for (int i = 0; i < NP; i++) w[i] = load4(r, 4 * (t + 64 * WAVES * i), p.len);
#pragma unroll
      for (int i = 0; i < NP; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) v[i][e] = v[i][e] + w[i][e];
    }
#pragma unroll
    for (int i = 0; i < NP; i++) g[i] = p.G ? load4(p.G, 4 * (t + 64 * WAVES * i), p.len) : f32x4{1.f, 1.f, 1.f, 1.f};
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < NP; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) sum = fma((double)v[i][e], (double)v[i][e], sum);
    sum = wave_sum_d(sum);
    if constexpr (WAVES > 1) {
      if ((threadIdx.x & 63) == 0) part[wave] = sum;
      __syncthreads();
      const double *mine = part + wave / WAVES * WAVES;
      sum = mine[0];
#pragma unroll
      for (int i = 1; i < WAVES; i++) sum += mine[i];
      __syncthreads();  // (the next row's sums go to the same places)
    }
    const RowFactor factor = row_factor(sum / (double)p.len, p.eps);
#pragma unroll
    for (int i = 0; i < NP; i++) {
      const int idx = 4 * (t + 64 * WAVES * i);
      if (p.S && live) store4(p.S + row * p.len, idx, p.len, v[i]);
      finish_piece(p, row, idx, live, factor, v[i], g[i]);
    }
  }
}

// Rows longer than the registers hold: a workgroup goes over its row twice.  (S may be X or R: a lane reads back its own sums.)
__global__ __launch_bounds__(256) void rmsnorm_stream(NormParams p) {
  __shared__ double part[4];
  const int wave = threadIdx.x >> 6, t = threadIdx.x;
  for (long long row = blockIdx.x; row < p.outer; row += gridDim.x) {
    const float *x = p.X + row * p.len, *r = p.R ? p.R + row * p.len : nullptr;
    auto piece = [&](int idx) {
      f32x4 v = load4(x, idx, p.len);
      if (r) {
        const f32x4 w = load4(r, idx, p.len);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = v[e] + w[e];
      }
      return v;
    };
    double sum = 0.0;
    for (long long idx = 4 * t; idx < p.len; idx += 1024) {
      const f32x4 v = piece((int)idx);
#pragma unroll
      for (int e = 0; e < 4; e++) sum = fma((double)v[e], (double)v[e], sum);
      if (p.S) store4(p.S + row * p.len, idx, p.len, v);
    }
    sum = wave_sum_d(sum);
    if ((threadIdx.x & 63) == 0) part[wave] = sum;
    __syncthreads();
    sum = ((part[0] + part[1]) + part[2]) + part[3];
    __syncthreads();
    const RowFactor factor = row_factor(sum / (double)p.len, p.eps);
    for (long long idx0 = 0; idx0 < p.len; idx0 += 1024) {  // (whole wavefronts take part in a block's maximum)
      const int idx = (int)(idx0 + 4 * t < p.len ? idx0 + 4 * t : (long long)p.len);
      f32x4 v = {0.f, 0.f, 0.f, 0.f}, g = {1.f, 1.f, 1.f, 1.f};
      if (idx < p.len) {
        v = p.S ? load4(p.S + row * p.len, idx, p.len) : piece(idx);
        if (p.G) g = load4(p.G, idx, p.len);
      }
      finish_piece(p, row, idx, idx < p.len, factor, v, g);
    }
  }
}

// A scale for each 1 x 128 block: half a wavefront to a block.
constexpr int UNROLL = 4;  // blocks a half wavefront has in flight
__global__ __launch_bounds__(256) void quantize_rows(const float *__restrict__ X, unsigned char *__restrict__ Q, float *__restrict__ QS, int cols,
                                                     wdh::FastDiv blocks, long long units) {
  const int sub = threadIdx.x & 31;
  const long long unit0 = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * UNROLL;
  f32x4 v[UNROLL];
  long long at[UNROLL];
  int idx[UNROLL];
#pragma unroll
  for (int j = 0; j < UNROLL; j++) {
    const int unit = (int)(unit0 + j < units ? unit0 + j : units - 1), row = wdh::fdiv(unit, blocks);
    idx[j] = (unit - row * blocks.d) * BLOCK + 4 * sub;
    at[j] = (long long)row * cols;
    v[j] = idx[j] < cols ? load4(X + at[j], idx[j], cols) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (int j = 0; j < UNROLL; j++) {
    float amax = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; e++) amax = fmaxf(amax, finite_abs(v[j][e]));
    const float c = block_scale(half_max(amax));
    if (unit0 + j >= units) continue;
    store4_bytes(Q + at[j], idx[j], cols, divide4(v[j], divisor(c)));
    if (sub == 0) QS[unit0 + j] = c;
  }
}

// A scale for each 128 x 128 block: a workgroup to a block, which stays in registers.  Workgroups go to the eight XCDs in turn, so each
// XCD is given a run of neighbouring blocks: the lines that two of them share, where rows are no whole lines, meet in one L2 (us, so /
// blocks in turn: 30000 x 1028 24.8 / 32.2, 30000 x 1024 24.6 / 27.4).
__global__ __launch_bounds__(256) void quantize_tiles(const float *__restrict__ X, unsigned char *__restrict__ Q, float *__restrict__ QS, long long rows,
                                                      int cols, int blocks, unsigned units) {
  __shared__ float part[4];
  const unsigned per = gridDim.x / 8, unit = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (unit >= units) return;
  const long long br = unit / blocks;
  const int bc = (int)(unit - br * blocks);
  // 1 << wide lanes to a row: 32, or fewer in a narrow last block, whose rows then take fewer turns (30000 x 1030, whose last block
  // has six columns: 25.4 us, with 32 lanes to every row 28.5)
  const int left = cols - bc * BLOCK, wide = left >= BLOCK / 2 + 1 ? 5 : left > 4 ? 32 - __builtin_clz((left + 3) / 4 - 1) : 0;
  const int turns = wide > 1 ? 1 << (wide - 1) : 1, idx = bc * BLOCK + 4 * (threadIdx.x & ((1 << wide) - 1));
  const long long row0 = br * BLOCK + (threadIdx.x >> wide), end = (br + 1) * BLOCK < rows ? (br + 1) * BLOCK : rows;
  const int step = 256 >> wide;
  f32x4 v[16];
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const long long row = row0 + step * i;
    v[i] = i < turns && row < end && idx < cols ? load4(X + row * cols, idx, cols) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; i++)
#pragma unroll
    for (int e = 0; e < 4; e++) amax = fmaxf(amax, finite_abs(v[i][e]));
  amax = wdh::rowmath::wave_max(amax);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = amax;
  __syncthreads();
  const float c = block_scale(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
  const Divisor by = divisor(c);
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const long long row = row0 + step * i;
    if (i < turns && row < end) store4_bytes(Q + row * cols, idx, cols, divide4(v[i], by));
  }
  if (threadIdx.x == 0) QS[unit] = c;
}

constexpr long long MOST_WGS = 1 << 20;  // (more rows than these hold are taken in turns)
template <int WAVES, int NP>
void launch_rows(const NormParams &p) {
  const long long wgs = WAVES < 4 ? (p.outer + 4 / WAVES - 1) / (4 / WAVES) : p.outer;
  hipLaunchKernelGGL((rmsnorm_rows<WAVES, NP>), dim3((unsigned)(wgs < MOST_WGS ? wgs : MOST_WGS)), dim3(WAVES < 4 ? 256 : 64 * WAVES), 0, wdh::stream(), p);
}

}  // namespace

using wdh::fail;

extern "C" int wdh_rmsnorm(wdh_buf hX, wdh_buf hSkip, wdh_buf hGamma, wdh_buf hSum, wdh_buf hY, wdh_buf hQ, wdh_buf hQScale,
                           int64_t outer, int len, float eps) {
  WDH_REQUIRE_INIT();
  WDH_REQUIRE_COMPUTE_LANE();
  if (outer < 0 || len < 0) return fail(WDH_EINVAL, "wdh_rmsnorm: negative extent");
  if (!hY && !hQ) return fail(WDH_EINVAL, "wdh_rmsnorm: neither Y nor Q given");
  if (!hQ != !hQScale) return fail(WDH_EINVAL, "wdh_rmsnorm: Q and QScale go together");
  if (!(eps >= 0.0f)) return fail(WDH_EINVAL, "wdh_rmsnorm: epsilon %g", (double)eps);
  if (outer == 0 || len == 0) return WDH_OK;
  if (len > (1 << 30) || outer > (1LL << 46) / len) return fail(WDH_EINVAL, "wdh_rmsnorm: too many elements");
  const size_t count = (size_t)outer * len, blocks = ((size_t)len + BLOCK - 1) / BLOCK;
  void *px, *pr = nullptr, *pg = nullptr, *ps = nullptr, *py = nullptr, *pq = nullptr, *pqs = nullptr;
  if (!wdh::operand(hX, count * 4, "wdh_rmsnorm: X", &px)) return WDH_EINVAL;
  if (hSkip && !wdh::operand(hSkip, count * 4, "wdh_rmsnorm: Skip", &pr)) return WDH_EINVAL;
  if (hGamma && !wdh::operand(hGamma, (size_t)len * 4, "wdh_rmsnorm: Gamma", &pg)) return WDH_EINVAL;
  if (hSum && !wdh::operand(hSum, count * 4, "wdh_rmsnorm: Sum", &ps)) return WDH_EINVAL;
  if (hY && !wdh::operand(hY, count * 4, "wdh_rmsnorm: Y", &py)) return WDH_EINVAL;
  if (hQ && !wdh::operand(hQ, count, "wdh_rmsnorm: Q", &pq)) return WDH_EINVAL;
  if (hQScale && !wdh::operand(hQScale, (size_t)outer * blocks * 4, "wdh_rmsnorm: QScale", &pqs)) return WDH_EINVAL;
  const wdh_buf out[4] = {hY, hQ, hQScale, hSum}, in[3] = {hX, hSkip, hGamma};
  for (int i = 0; i < 4; i++) {
    for (int j = 0; j < 3; j++)  // (a row is read whole before it is written, so the sum may take the place of X or Skip)
      if (out[i] && out[i] == in[j] && !(i == 3 && j < 2)) return fail(WDH_EINVAL, "wdh_rmsnorm: a result aliases an input");
    for (int j = 0; j < i; j++)
      if (out[i] && out[i] == out[j]) return fail(WDH_EINVAL, "wdh_rmsnorm: two results share a buffer");
  }
  NormParams p;
  p.X = (const float *)px; p.R = (const float *)pr; p.G = (const float *)pg; p.S = (float *)ps; p.Y = (float *)py;
  p.Q = (unsigned char *)pq; p.QS = (float *)pqs;
  p.outer = outer; p.len = len; p.blocks = (int)blocks; p.eps = eps;
  // As few wavefronts to a row as leave a lane four pieces, and as few pieces as hold it, but for one thing: long rows take more wavefronts,
  // a lane's eight pieces of X and Skip being too many registers.  (us, 100 MB of rows of 782 elements: 1 wavefront of 4 pieces 78.7, 4 of
  // 1 85.6; of 570: 1 of 3 77.5, 4 of 1 107.0; of 6000: 8 of 3 74.7, 4 of 8 94.4; of 8192: 8 of 4 71.2, 4 of 8 79.2.)  Rows beyond 8192
  // elements stay in registers where there are few of them (100 of 12000: 8.2 us, read twice 15.8; 2000: 92.7 and 85.8).
  if (len <= 256) launch_rows<1, 1>(p);
  else if (len <= 512) launch_rows<1, 2>(p);
  else if (len <= 768) launch_rows<1, 3>(p);
  else if (len <= 1024) launch_rows<1, 4>(p);
  else if (len <= 1536) launch_rows<2, 3>(p);
  else if (len <= 2048) launch_rows<4, 2>(p);
  else if (len <= 4096) launch_rows<4, 4>(p);
  else if (len <= 6144) launch_rows<8, 3>(p);
  else if (len <= 8192) launch_rows<8, 4>(p);
  else if (len <= 16384 && outer <= 2 * wdh::compute_units()) launch_rows<16, 4>(p);
  else hipLaunchKernelGGL(rmsnorm_stream, dim3((unsigned)(outer < MOST_WGS ? outer : MOST_WGS)), dim3(256), 0, wdh::stream(), p);
  WDH_LAUNCH_CHECK();
  return WDH_OK;
}

extern "C" int wdh_quantize_fp8(wdh_buf hX, wdh_buf hQ, wdh_buf hQScale, int64_t rows, int cols, int block_rows) {
  WDH_REQUIRE_INIT();
  WDH_REQUIRE_COMPUTE_LANE();
  if (rows < 0 || cols < 0) return fail(WDH_EINVAL, "wdh_quantize_fp8: negative extent");
  if (block_rows != 1 && block_rows != BLOCK)
    return fail(WDH_EINVAL, "wdh_quantize_fp8: blocks of %d rows (1 and %d are built)", block_rows, BLOCK);
  if (rows == 0 || cols == 0) return WDH_OK;
  if (cols > (1 << 30) || rows > (1LL << 46) / cols) return fail(WDH_EINVAL, "wdh_quantize_fp8: too many elements");
  const long long blocks = ((long long)cols + BLOCK - 1) / BLOCK, units = (rows + block_rows - 1) / block_rows * blocks;
  // (a launch has fewer than 2^32 threads: eight to a block of one row, 256 to one of 128)
  if (units > (block_rows == 1 ? 0xffffffLL * 8 * UNROLL : 0xfffff8LL)) return fail(WDH_EINVAL, "wdh_quantize_fp8: too many blocks");
  void *px, *pq, *pqs;
  if (!wdh::operand(hX, (size_t)rows * cols * 4, "wdh_quantize_fp8: X", &px)) return WDH_EINVAL;
  if (!wdh::operand(hQ, (size_t)rows * cols, "wdh_quantize_fp8: Q", &pq)) return WDH_EINVAL;
  if (!wdh::operand(hQScale, (size_t)units * 4, "wdh_quantize_fp8: QScale", &pqs)) return WDH_EINVAL;
  if (hQ == hX || hQScale == hX || hQ == hQScale) return fail(WDH_EINVAL, "wdh_quantize_fp8: operands share a buffer");
  if (block_rows == 1)
    hipLaunchKernelGGL(quantize_rows, dim3((unsigned)((units + 8 * UNROLL - 1) / (8 * UNROLL))), dim3(256), 0, wdh::stream(), (const float *)px,
                       (unsigned char *)pq, (float *)pqs, cols, wdh::make_fastdiv(blocks), units);
  else
    hipLaunchKernelGGL(quantize_tiles, dim3((unsigned)((units + 7) / 8 * 8)), dim3(256), 0, wdh::stream(), (const float *)px, (unsigned char *)pq, (float *)pqs,
                       (long long)rows, cols, (int)blocks, (unsigned)units);
  WDH_LAUNCH_CHECK();
  return WDH_OK;
}
