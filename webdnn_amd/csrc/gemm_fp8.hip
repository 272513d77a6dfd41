// Y = A W^T of e4m3 operands with a scale for each block of 128 along K (and, of W, for 128 rows):
//   Y[i, j] = sum_b SA[i, b] SW[j / 128, b] sum_{x in b} A[i, x] W[j, x]   (+ bias[j]) (+ R[i, j]), then Relu if asked for.
// The inner sums run on the bfloat16 matrix instructions, operands widened from e4m3 in registers (exact products, sums in fp32);
// their results are scaled and added up in fp32.
//
// The product is computed transposed (W is the instruction's first operand): a lane then holds results of one row of A, so that
// the scale of a block is one number to a lane, and four neighbouring results to store.
#include "common.h"
#include "fp8.h"

namespace {

using namespace wdh::fp8;

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct ProductParams {
  const unsigned char *A, *W;
  const float *SA, *SW, *bias, *R;
  float *Y;
  long long m;
  int n, k, blocks, relu;
};

// 32 bytes a lane of each operand: the lanes that share a row hold its 128 elements, in the same order on both sides.
__device__ __forceinline__ f32x4 block_product(i32x8 a, i32x8 b) {
  f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; i++)
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(a[2 * i], a[2 * i + 1]), widen(b[2 * i], b[2 * i + 1]), c, 0, 0, 0);
  return c;
}

// Bytes k .. k+15 of a row of length `len`, 0 beyond its end.
template <bool ALIGNED>
__device__ __forceinline__ i32x4 load16(const unsigned char *row, int k, int len) {
  if (k + 16 <= len)
    return ALIGNED ? *reinterpret_cast<const i32x4 *>(row + k) : (i32x4)*reinterpret_cast<const i32x4_any *>(row + k);
  i32x4 v = {0, 0, 0, 0};
  if (!ALIGNED)  // (rows of whole pieces end where a piece does)
    for (int e = 0; e < 15 && k + e < len; e++) v[e >> 2] |= (int)row[k + e] << (8 * (e & 3));
  return v;
}
template <bool ALIGNED>
__device__ __forceinline__ i32x8 load32(const unsigned char *row, int k, int len) {
  const i32x4 a = load16<ALIGNED>(row, k, len), b = load16<ALIGNED>(row, k + 16, len);
  return i32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// Columns j .. j+3 of row i: bias, residual, Relu, and out.
__device__ __forceinline__ void finish4(const ProductParams &p, long long i, int j, f32x4 v) {
  const int left = p.n - j;
  if (left <= 0) return;
  float *y = p.Y + i * p.n;
  if (p.bias) v = v + load4(p.bias, j, p.n);
  if (p.R) v = v + load4(p.R + i * p.n, j, p.n);
  if (p.relu)
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = !(v[e] > 0.0f) && v[e] == v[e] ? 0.0f : v[e];
  store4(y, j, p.n, v);
}

// Few rows of A: a workgroup has 16 rows of W and 16 MT of A, its wavefronts take K blocks in turn and add up through LDS.
template <int MT, bool ALIGNED>
__global__ __launch_bounds__(256) void product_few(ProductParams p) {
  __shared__ __attribute__((aligned(16))) f32x4 part[4][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const unsigned char *w = p.W + (long long)(n0 + i16 < p.n ? n0 + i16 : p.n - 1) * p.k;
  const float *sw = p.SW + (long long)(n0 / BLOCK) * p.blocks;
  for (long long m0 = (long long)blockIdx.y * (16 * MT); m0 < p.m; m0 += (long long)gridDim.y * (16 * MT)) {
    long long row[MT];
    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) {
      const long long r = m0 + 16 * t + i16;
      row[t] = r < p.m ? r : p.m - 1;
      acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int b = wave; b < p.blocks; b += 4) {
      const i32x8 a = load32<ALIGNED>(w, b * BLOCK + 32 * g, p.k);
      const float s = sw[b];
#pragma unroll
      for (int t = 0; t < MT; t++) {
        const f32x4 x = block_product(a, load32<ALIGNED>(p.A + row[t] * p.k, b * BLOCK + 32 * g, p.k));
        const float c = p.SA[row[t] * p.blocks + b] * s;
#pragma unroll
        for (int e = 0; e < 4; e++) acc[t][e] = __builtin_fmaf(x[e], c, acc[t][e]);
      }
    }
#pragma unroll
    for (int t = 0; t < MT; t++) part[wave][t][lane] = acc[t];
    __syncthreads();
    for (int cell = threadIdx.x; cell < 64 * MT; cell += 256) {
      const int t = cell >> 6, l = cell & 63;
      const f32x4 v = (part[0][t][l] + part[1][t][l]) + (part[2][t][l] + part[3][t][l]);
      const long long i = m0 + 16 * t + (l & 15);
      if (i < p.m) finish4(p, i, n0 + 4 * (l >> 4), v);
    }
    __syncthreads();
  }
}

template <int MT>
void launch_few(const ProductParams &p, bool aligned) {
  const long long rows = (p.m + 16 * MT - 1) / (16 * MT);
  const dim3 grid((unsigned)((p.n + 15) / 16), (unsigned)(rows < 65535 ? rows : 65535));
  if (aligned) hipLaunchKernelGGL((product_few<MT, true>), grid, dim3(256), 0, wdh::stream(), p);
  else hipLaunchKernelGGL((product_few<MT, false>), grid, dim3(256), 0, wdh::stream(), p);
}

// Tiles of NW TN x 32 columns of Y (rows of W) and MW TM x 32 rows: NW x MW wavefronts with TN x TM blocks of 32 x 32 each.
// A slab is a block of K: 128 bytes of every row of the tile, which pass through registers into LDS while the slab before is
// multiplied.  In LDS a row's eight 16-byte pieces are exchanged by its number (piece ^ row % 8), so that the 32 rows that a
// fragment read takes a piece of lie on different banks.  A fragment's 16 bytes serve two instructions (their k are the first and the
// last eight of them, on both sides alike).
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int NW, int MW, int TN, int TM, bool ALIGNED>
__global__ __launch_bounds__(64 * NW * MW, 2) void product_tiles(ProductParams p) {
  constexpr int THREADS = 64 * NW * MW, BN = 32 * NW * TN, BM = 32 * MW * TM, ROWS = BN + BM;
  constexpr int LOADS = ROWS * 8 / THREADS;
  static_assert(ROWS * 8 % THREADS == 0 && BM <= THREADS && BLOCK % (32 * TN) == 0, "tile");
  __shared__ __attribute__((aligned(16))) unsigned char lds[2][ROWS * BLOCK];
  __shared__ float scales[2][BM];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, half = lane >> 5;
  const int wn = wave % NW, wm = wave / NW;
  const int tiles_n = (p.n + BN - 1) / BN;
  const long long m0 = (long long)(blockIdx.x / tiles_n) * BM;
  const int n0 = (int)(blockIdx.x % tiles_n) * BN;

  const unsigned char *row[LOADS];
  int to[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; i++) {
    const int at = tid + THREADS * i, r = at >> 3;
    if (r < BN) row[i] = p.W + (long long)(n0 + r < p.n ? n0 + r : p.n - 1) * p.k;
    else row[i] = p.A + (m0 + r - BN < p.m ? m0 + r - BN : p.m - 1) * p.k;
    to[i] = r * BLOCK + 16 * ((at & 7) ^ (r & 7));
  }
  const int piece = 16 * (tid & 7);
  const float *my_scale = p.SA + (m0 + tid % BM < p.m ? m0 + tid % BM : p.m - 1) * p.blocks;
  const int wide = (n0 + 32 * TN * wn) / BLOCK;  // (columns beyond n: any scale will do)
  const float *sw = p.SW + (long long)(wide * BLOCK < p.n ? wide : 0) * p.blocks;

  i32x4 next[LOADS];
  float next_scale = 0.0f;
  auto fetch = [&](int b) {
#pragma unroll
    for (int i = 0; i < LOADS; i++) next[i] = load16<ALIGNED>(row[i], b * BLOCK + piece, p.k);
    if (tid < BM) next_scale = my_scale[b];
  };
  auto keep = [&](int buf) {
#pragma unroll
    for (int i = 0; i < LOADS; i++) *reinterpret_cast<i32x4 *>(&lds[buf][to[i]]) = next[i];
    if (tid < BM) scales[buf][tid] = next_scale;
  };
  // a 32-row block's fragments: 16 bytes for each quarter of the slab
  auto fragment = [&](int buf, int r0, bf16x8 (&f)[8]) {
    const int r = r0 + li;
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const i32x4 x = *reinterpret_cast<const i32x4 *>(&lds[buf][r * BLOCK + 16 * ((2 * q + half) ^ (r & 7))]);
      f[2 * q] = widen(x[0], x[1]);
      f[2 * q + 1] = widen(x[2], x[3]);
    }
  };

  f32x16 acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; i++)
#pragma unroll
    for (int j = 0; j < TM; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[i][j][e] = 0.0f;
  if (p.blocks > 0) {
    fetch(0);
    keep(0);
  }
  __syncthreads();
  for (int b = 0; b < p.blocks; b++) {
    const int buf = b & 1;
    if (b + 1 < p.blocks) fetch(b + 1);
    const float s = sw[b];
    bf16x8 a[TM][8];
    float c[TM];
#pragma unroll
    for (int j = 0; j < TM; j++) {
      fragment(buf, BN + 32 * (TM * wm + j), a[j]);
      c[j] = scales[buf][32 * (TM * wm + j) + li] * s;
    }
#pragma unroll
    for (int i = 0; i < TN; i++) {
      bf16x8 w[8];
      fragment(buf, 32 * (TN * wn + i), w);
      f32x16 x[TM];
#pragma unroll
      for (int j = 0; j < TM; j++)
#pragma unroll
        for (int e = 0; e < 16; e++) x[j][e] = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; k++)
#pragma unroll
        for (int j = 0; j < TM; j++) x[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[k], a[j][k], x[j], 0, 0, 0);
#pragma unroll
      for (int j = 0; j < TM; j++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[i][j][e] = __builtin_fmaf(x[j][e], c[j], acc[i][j][e]);
    }
    if (b + 1 < p.blocks) keep(buf ^ 1);
    __syncthreads();
  }
  // lane: row li of a block; registers 4 q .. + 3 are columns 8 q + 4 half .. + 3
#pragma unroll
  for (int j = 0; j < TM; j++) {
    const long long i = m0 + 32 * (TM * wm + j) + li;
    if (i >= p.m) continue;
#pragma unroll
    for (int t = 0; t < TN; t++)
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const int col = n0 + 32 * (TN * wn + t) + 8 * q + 4 * half;
        f32x4 v = {acc[t][j][4 * q], acc[t][j][4 * q + 1], acc[t][j][4 * q + 2], acc[t][j][4 * q + 3]};
        finish4(p, i, col, v);
      }
  }
}

template <int NW, int MW, int TN, int TM>
void launch_tiles(const ProductParams &p, bool aligned) {
  constexpr int BN = 32 * NW * TN, BM = 32 * MW * TM;
  const long long tiles = (p.n + BN - 1) / BN * ((p.m + BM - 1) / BM);
  const dim3 grid((unsigned)tiles), wg(64 * NW * MW);
  if (aligned) hipLaunchKernelGGL((product_tiles<NW, MW, TN, TM, true>), grid, wg, 0, wdh::stream(), p);
  else hipLaunchKernelGGL((product_tiles<NW, MW, TN, TM, false>), grid, wg, 0, wdh::stream(), p);
}

}  // namespace

using wdh::fail;

extern "C" int wdh_gemm_fp8(wdh_buf hA, wdh_buf hSA, wdh_buf hW, wdh_buf hSW, wdh_buf hBias, wdh_buf hY, int64_t m, int n, int k, int epilogue,
                            wdh_buf hR) {
  WDH_REQUIRE_INIT();
  WDH_REQUIRE_COMPUTE_LANE();
  if (m < 0 || n < 0 || k < 0) return fail(WDH_EINVAL, "wdh_gemm_fp8: negative extent");
  if (epilogue != WDH_EPI_NONE && epilogue != WDH_EPI_RELU) return fail(WDH_EINVAL, "wdh_gemm_fp8: unknown epilogue %d", epilogue);
  if (m == 0 || n == 0) return WDH_OK;
  if (n > (1 << 30) || k > (1 << 30) || m > (1LL << 46) / n || (k && m > (1LL << 46) / k)) return fail(WDH_EINVAL, "wdh_gemm_fp8: too many elements");
  const size_t blocks = ((size_t)k + BLOCK - 1) / BLOCK, wide = ((size_t)n + BLOCK - 1) / BLOCK, results = (size_t)m * n * 4;
  void *pa, *psa, *pw, *psw, *pb = nullptr, *py, *pr = nullptr;
  if (!wdh::operand(hA, (size_t)m * k, "wdh_gemm_fp8: A", &pa)) return WDH_EINVAL;
  if (!wdh::operand(hSA, (size_t)m * blocks * 4, "wdh_gemm_fp8: AScale", &psa)) return WDH_EINVAL;
  if (!wdh::operand(hW, (size_t)n * k, "wdh_gemm_fp8: W", &pw)) return WDH_EINVAL;
  if (!wdh::operand(hSW, wide * blocks * 4, "wdh_gemm_fp8: WScale", &psw)) return WDH_EINVAL;
  if (hBias && !wdh::operand(hBias, (size_t)n * 4, "wdh_gemm_fp8: Bias", &pb)) return WDH_EINVAL;
  if (!wdh::operand(hY, results, "wdh_gemm_fp8: Y", &py)) return WDH_EINVAL;
  if (hR && !wdh::operand(hR, results, "wdh_gemm_fp8: R", &pr)) return WDH_EINVAL;
  for (wdh_buf h : {hA, hSA, hW, hSW, hBias})  // (R may be Y: an element is read by the lane that stores it)
    if (h == hY) return fail(WDH_EINVAL, "wdh_gemm_fp8: Y aliases an input");
  ProductParams p;
  p.A = (const unsigned char *)pa; p.W = (const unsigned char *)pw;
  p.SA = (const float *)psa; p.SW = (const float *)psw; p.bias = (const float *)pb; p.R = (const float *)pr;
  p.Y = (float *)py;
  p.m = m; p.n = n; p.k = k; p.blocks = (int)blocks; p.relu = epilogue == WDH_EPI_RELU;
  const bool aligned = k % 16 == 0;  // (buffers are)
  if (m <= 16) launch_few<1>(p, aligned);
  else if (m <= 64) launch_few<4>(p, aligned);
  else if ((n + 127) / 128 * ((m + 127) / 128) < 2LL * wdh::compute_units()) launch_tiles<2, 2, 1, 1>(p, aligned);
  else launch_tiles<4, 2, 2, 2>(p, aligned);
  WDH_LAUNCH_CHECK();
  return WDH_OK;
}
