// Y = A W^T of e4m3 operands with a scale for each block of 128 along K (and, of W, for 128 rows):
//   Y[i, j] = sum_b SA[i, b] SW[j / 128, b] sum_{x in b} A[i, x] W[j, x]   (+ bias[j]) (+ R[i, j]), then Relu if asked for.
// The inner sums run on the bfloat16 matrix instructions, operands widened from e4m3 in registers (exact products, sums in fp32);
// their results are scaled and added up in fp32.  The product of a block's two scales is taken first, and is a normal number (or 0) by
// contract: splitting scales into a part whose products are always normal and a power of two that the widening instructions take
// along was built and cost 1 to 8 % (us, so / split: 128 x 8192 x 8192 34.2 / 37.3, 333 x 1000 x 2050 9.8 / 10.2, 64 x 4096 x 4096 8.1 / 8.4).
//
// The product is computed transposed (W is the instruction's first operand): a lane then holds results of one row of A, so that
// the scale of a block is one number to a lane, and four neighbouring results to store.
#include "common.h"
#include "fp8.h"

namespace {

using namespace wdh::fp8;

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct ProductParams {
  const unsigned char *A, *W;
  const float *SA, *SW, *bias, *R;
  float *Y;
  long long m;
  int n, k, blocks, relu;
  long long pitch;  // bytes between rows of A, and of W
  int part;         // blocks of K that a part of the product takes: its results go to Y [part][m][n]
};

// 32 bytes a lane of each operand.
__device__ __forceinline__ f32x4 block_product(i32x8 a, i32x8 b) {
  f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; i++)
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(a[2 * i], a[2 * i + 1]), widen(b[2 * i], b[2 * i + 1]), c, 0, 0, 0);
  return c;
}

// Bytes k .. k+15 of a row of length `len`, 0 beyond its end.  Rows of whole 16-byte pieces are loaded as they lie; others dword by
// dword (the hardware takes loads off dword boundaries, but slowly) and put together where they are used, so that nothing
// waits for them before.  A piece that ends behind the row is cut out of the row's last 16 bytes: every dword read holds a byte of
// the row, and loads are behind no branch that lanes take differently.
template <bool ALIGNED>
struct Piece {
  i32x4 d;
  __device__ __forceinline__ void load(const unsigned char *row, int k, int len) {
    if (k < len) d = *reinterpret_cast<const i32x4 *>(row + k);
    else d = i32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ i32x4 get(const unsigned char *, int, int) const { return d; }
};
template <>
struct Piece<false> {
  i32x4 d;
  int e;
  static __device__ __forceinline__ int begin(int k, int len) { return k + 16 <= len ? k : len > 16 ? len - 16 : 0; }
  __device__ __forceinline__ void load(const unsigned char *row, int k, int len) {
    const int from = begin(k, len);
    const unsigned shift = (unsigned)((uintptr_t)row + from) & 3u;
    const int *base = reinterpret_cast<const int *>(row + from - shift);  // (a number made a pointer again would be loaded from as of any kind)
    if (len >= 16) {
      typedef int i32x4_dwords __attribute__((ext_vector_type(4), aligned(4)));
      d = *reinterpret_cast<const i32x4_dwords *>(base);
      e = base[(shift + 15) >> 2];
    } else {
      const int last = (int)(shift + len - 1) >> 2;
#pragma unroll
      for (int i = 0; i < 4; i++) d[i] = base[i < last ? i : last];
      e = base[last];
    }
  }
  __device__ __forceinline__ i32x4 get(const unsigned char *row, int k, int len) const {
    const int from = begin(k, len);
    const unsigned shift = (unsigned)((uintptr_t)row + from) & 3u;
    i32x4 v;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = (int)__builtin_amdgcn_alignbyte((unsigned)(i < 3 ? d[i + 1] : e), (unsigned)d[i], shift);
    if (k + 16 > len) {
      const int left = len - k, skip = k - from;  // bytes of v that are kept, and those in front of them
      unsigned long long lo = (unsigned)v[0] | (unsigned long long)(unsigned)v[1] << 32, hi = (unsigned)v[2] | (unsigned long long)(unsigned)v[3] << 32;
      const int bits = 8 * (skip & 7);
      if (skip >= 8) lo = hi, hi = 0;
      lo = bits ? lo >> bits | hi << (64 - bits) : lo;
      hi >>= bits;
      lo = left >= 8 ? lo : left > 0 ? lo & ((1ull << (8 * left)) - 1) : 0;
      hi = left >= 16 ? hi : left > 8 ? hi & ((1ull << (8 * (left - 8))) - 1) : 0;
      v = i32x4{(int)lo, (int)(lo >> 32), (int)hi, (int)(hi >> 32)};
    }
    return v;
  }
};
// Columns j .. j+3 of row i: bias, residual, Relu, and out.
__device__ __forceinline__ void finish4(const ProductParams &p, float *Y, long long i, int j, f32x4 v) {
  const int left = p.n - j;
  if (left <= 0) return;
  if (p.bias) v = v + load4(p.bias, j, p.n);
  if (p.R) v = v + load4(p.R + i * p.n, j, p.n);
  if (p.relu)
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = !(v[e] > 0.0f) && v[e] == v[e] ? 0.0f : v[e];
  store4(Y + i * p.n, j, p.n, v);
}

// One or two rows of A: a workgroup has four rows of W, its wavefronts a quarter of K each, a KB of a row at a time; products and sums in
// fp32 on the vector units, which keep up with memory where the matrix ones would work for one row of 16.  Bound: memory (us, so / in
// tiles of 16 rows; one row: 8192 x 8192 13.3 / 16.9, 5.1 TB/s, 4096 columns, K = 14336, 12.3 / 15.9, 14336 columns, K = 4096, 11.9 / 15.0;
// two rows: 14.6 / 17.0, 13.8 / 16.1, 14.0 / 15.0; three would be 17.2 / 17.1, 14.8 / 16.2, 15.8 / 15.0).
template <int M, bool ALIGNED>
__global__ __launch_bounds__(256) void product_rows(ProductParams p) {
  constexpr int R = 4;
  __shared__ float part[4][R * M];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int j0 = blockIdx.x * R; j0 < p.n; j0 += gridDim.x * R) {
    const float *sw = p.SW + (long long)(j0 / BLOCK) * p.blocks;
    auto row = [&](int r) { return p.W + (long long)(j0 + r < p.n ? j0 + r : p.n - 1) * p.pitch; };
    float acc[R][M];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int m = 0; m < M; m++) acc[r][m] = 0.0f;
#pragma unroll(M == 1 ? 2 : 1)
    for (int k = 1024 * wave + 16 * lane; k < p.k; k += 4096) {
      Piece<ALIGNED> a[M], w[R];
      float c[M];
#pragma unroll
      for (int r = 0; r < R; r++) w[r].load(row(r), k, p.k);
#pragma unroll
      for (int m = 0; m < M; m++) a[m].load(p.A + m * p.pitch, k, p.k);
      const float s = sw[k / BLOCK];
#pragma unroll
      for (int m = 0; m < M; m++) c[m] = p.SA[(long long)m * p.blocks + k / BLOCK] * s;
      f32x2 x[M][8];
#pragma unroll
      for (int m = 0; m < M; m++) {
        const i32x4 v = a[m].get(p.A + m * p.pitch, k, p.k);
#pragma unroll
        for (int i = 0; i < 4; i++) x[m][2 * i] = __builtin_amdgcn_cvt_pk_f32_fp8(v[i], false), x[m][2 * i + 1] = __builtin_amdgcn_cvt_pk_f32_fp8(v[i], true);
      }
#pragma unroll
      for (int r = 0; r < R; r++) {
        const i32x4 v = w[r].get(row(r), k, p.k);
        float sum[M];
#pragma unroll
        for (int m = 0; m < M; m++) sum[m] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const f32x2 y = i & 1 ? __builtin_amdgcn_cvt_pk_f32_fp8(v[i / 2], true) : __builtin_amdgcn_cvt_pk_f32_fp8(v[i / 2], false);
#pragma unroll
          for (int m = 0; m < M; m++) sum[m] = __builtin_fmaf(x[m][i][1], y[1], __builtin_fmaf(x[m][i][0], y[0], sum[m]));
        }
#pragma unroll
        for (int m = 0; m < M; m++) acc[r][m] = __builtin_fmaf(sum[m], c[m], acc[r][m]);
      }
    }
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int m = 0; m < M; m++) {
        const float sum = wdh::rowmath::wave_sum(acc[r][m]);
        if (lane == 0) part[wave][m * R + r] = sum;
      }
    __syncthreads();
    const int t = threadIdx.x, j = j0 + t % R, m = t / R;
    if (t < R * M && j < p.n) {
      float v = ((part[0][t] + part[1][t]) + part[2][t]) + part[3][t];
      if (p.bias) v = v + p.bias[j];
      if (p.R) v = v + p.R[(long long)m * p.n + j];
      p.Y[(long long)m * p.n + j] = p.relu && !(v > 0.0f) && v == v ? 0.0f : v;
    }
    __syncthreads();  // (the next rows' sums go to the same places)
  }
}

template <int M>
void launch_rows(const ProductParams &p, bool aligned) {
  const dim3 grid((unsigned)((p.n + 3) / 4 < 1 << 20 ? (p.n + 3) / 4 : 1 << 20));
  if (aligned) hipLaunchKernelGGL((product_rows<M, true>), grid, dim3(256), 0, wdh::stream(), p);
  else hipLaunchKernelGGL((product_rows<M, false>), grid, dim3(256), 0, wdh::stream(), p);
}

// Few rows of A, or few results: a workgroup has 16 NT rows of W and 16 MT of A, its wavefronts take K blocks in turn and add up through
// LDS.  A wavefront brings its blocks itself, eight lanes to a row, the next one while it works on this one, and turns them in a part of LDS
// of its own, where a row's pieces are exchanged by its number (as below), into what the matrix instructions take: a row to each of
// 16 neighbouring lanes, which straight from memory is 16 lines for 16 lanes (us, so / straight from memory: 64 rows, 4096 x 4096, 8.4 /
// 12.9, 333 x 1000 x 2048 7.4 / 9.8, x 2050 10.3 / 12.8).  More than one block on its way is slower
// (64 rows 9.4).  Bound: memory (W is read once for 16 MT rows), or latency.
template <int NT, int MT, int WAVES, bool ALIGNED>
__global__ __launch_bounds__(64 * WAVES) void product_few(ProductParams p) {
  constexpr int ROWS = 16 * (NT + MT), LOADS = ROWS / 8;
  __shared__ __attribute__((aligned(16))) union { unsigned char rows[WAVES][ROWS * BLOCK]; f32x4 part[WAVES][NT * MT][64]; } lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * (16 * NT), begin = blockIdx.z * p.part, end = begin + p.part < p.blocks ? begin + p.part : p.blocks;
  const int piece = 16 * (lane & 7);
  unsigned char *mine = lds.rows[wave];
  const float *sw[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int tile = n0 + 16 * t;
    sw[t] = p.SW + (long long)((tile < p.n ? tile : p.n - 1) / BLOCK) * p.blocks;
  }
  for (long long m0 = (long long)blockIdx.y * (16 * MT); m0 < p.m; m0 += (long long)gridDim.y * (16 * MT)) {
    const unsigned char *w0 = p.W + n0 * p.pitch, *a0 = p.A + m0 * p.pitch;
    const int w_last = p.n - 1 - n0, a_last = p.m - 1 - m0 < 16 * MT ? (int)(p.m - 1 - m0) : 16 * MT;
    auto row = [&](int i) {  // (rows behind the last are the last one again; addresses are worked out where they are used)
      const int r = 8 * i + fresh(lane >> 3) - (8 * i < 16 * NT ? 0 : 16 * NT), last = 8 * i < 16 * NT ? w_last : a_last;
      return (8 * i < 16 * NT ? w0 : a0) + (unsigned long long)(unsigned)(r < last ? r : last) * (unsigned)p.pitch;
    };
    const float *sa[MT];
    f32x4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < MT; t++) {
      sa[t] = p.SA + (m0 + 16 * t + i16 < p.m ? m0 + 16 * t + i16 : p.m - 1) * p.blocks;
#pragma unroll
      for (int q = 0; q < NT; q++) acc[q][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    Piece<ALIGNED> next[LOADS];
    float next_sa[MT], next_sw[NT];
    auto fetch = [&](int b) {
      if (b >= end) return;
      if constexpr (ALIGNED) {
        const int k = b * BLOCK + piece;
        if (k < p.k)
#pragma unroll
          for (int i = 0; i < LOADS; i++) next[i].d = *reinterpret_cast<const i32x4 *>(row(i) + k);
        else
#pragma unroll
          for (int i = 0; i < LOADS; i++) next[i].d = i32x4{0, 0, 0, 0};
      } else {
#pragma unroll
        for (int i = 0; i < LOADS; i++) next[i].load(row(i), b * BLOCK + piece, p.k);
      }
#pragma unroll
      for (int t = 0; t < MT; t++) next_sa[t] = sa[t][b];
#pragma unroll
      for (int q = 0; q < NT; q++) next_sw[q] = sw[q][b];
    };
    // 32 bytes of row r: the lanes that share a row hold its 128 elements, in the same order on both sides
    auto fragment = [&](int r) {
      const i32x4 x = *reinterpret_cast<const i32x4 *>(mine + r * BLOCK + 16 * ((2 * g) ^ (r & 7)));
      const i32x4 y = *reinterpret_cast<const i32x4 *>(mine + r * BLOCK + 16 * ((2 * g + 1) ^ (r & 7)));
      return i32x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    };
    fetch(begin + wave);
    for (int b = begin + wave; b < end; b += WAVES) {
#pragma unroll
      for (int i = 0; i < LOADS; i++) {
        const int r = 8 * i + (lane >> 3);
        *reinterpret_cast<i32x4 *>(mine + r * BLOCK + 16 * ((lane & 7) ^ (r & 7))) = next[i].get(row(i), b * BLOCK + piece, p.k);
      }
      float ca[MT], cw[NT];
#pragma unroll
      for (int t = 0; t < MT; t++) ca[t] = next_sa[t];
#pragma unroll
      for (int q = 0; q < NT; q++) cw[q] = next_sw[q];
      fetch(b + WAVES);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      i32x8 w8[NT];
#pragma unroll
      for (int q = 0; q < NT; q++) w8[q] = fragment(16 * q + i16);
#pragma unroll
      for (int t = 0; t < MT; t++) {
        const i32x8 a8 = fragment(16 * (NT + t) + i16);
#pragma unroll
        for (int q = 0; q < NT; q++) {
          const f32x4 x = block_product(w8[q], a8);
          const float c = ca[t] * cw[q];
#pragma unroll
          for (int e = 0; e < 4; e++) acc[q][t][e] = __builtin_fmaf(x[e], c, acc[q][t][e]);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < NT; q++)
#pragma unroll
      for (int t = 0; t < MT; t++) lds.part[wave][q * MT + t][lane] = acc[q][t];
    __syncthreads();
    for (int cell = threadIdx.x; cell < 64 * NT * MT; cell += 64 * WAVES) {
      const int tile = cell >> 6, l = cell & 63;
      f32x4 v = lds.part[0][tile][l];
#pragma unroll
      for (int i = 1; i < WAVES; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] += lds.part[i][tile][l][e];
      const long long i = m0 + 16 * (tile % MT) + (l & 15);
      if (i < p.m) finish4(p, p.Y + blockIdx.z * p.m * p.n, i, n0 + 16 * (tile / MT) + 4 * (l >> 4), v);
    }
    __syncthreads();
  }
}

unsigned parts_of(const ProductParams &p) { return p.part < p.blocks ? (unsigned)((p.blocks + p.part - 1) / p.part) : 1u; }

template <int NT, int MT, int WAVES>
void launch_few(const ProductParams &p, bool aligned) {
  const long long rows = (p.m + 16 * MT - 1) / (16 * MT);
  const dim3 grid((unsigned)((p.n + 16 * NT - 1) / (16 * NT)), (unsigned)(rows < 65535 ? rows : 65535), parts_of(p)), wg(64 * WAVES);
  if (aligned) hipLaunchKernelGGL((product_few<NT, MT, WAVES, true>), grid, wg, 0, wdh::stream(), p);
  else hipLaunchKernelGGL((product_few<NT, MT, WAVES, false>), grid, wg, 0, wdh::stream(), p);
}

// Tiles of NW TN x 32 columns of Y (rows of W) and MW TM x 32 rows: NW x MW wavefronts with TN x TM blocks of 32 x 32 each.
// A slab is a block of K: 128 bytes of every row of the tile, which pass through registers into LDS while the slab before is
// multiplied.  In LDS a row's eight 16-byte pieces are exchanged by its number (piece ^ row % 8), so that the 32 rows that a
// fragment read takes a piece of lie on different banks.  A fragment's 16 bytes serve two instructions (their k are the first and the
// last eight of them, on both sides alike).  A slab is multiplied by quarters, the next one's fragments on their way from LDS
// meanwhile (8192^3: 1032 to 1080 us from run to run, 1018 to 1065 TFLOP/s; fragments of the whole slab at a time 1146).
// Bound: the matrix cores, the conversions and the way through LDS alternate more than they overlap (without the loads of slabs that
// product takes 890 us, without their way into LDS either 800; library products of bfloat16 operands of that size take 890 in ten calls in a row, 776 in long runs).
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int NW, int MW, int TN, int TM>
__global__ __launch_bounds__(64 * NW * MW, 2) void product_tiles(ProductParams p) {
  constexpr int THREADS = 64 * NW * MW, BN = 32 * NW * TN, BM = 32 * MW * TM, ROWS = BN + BM;
  constexpr int LOADS = ROWS * 8 / THREADS;
  static_assert(ROWS * 8 % THREADS == 0 && BM <= THREADS && BLOCK % (32 * TN) == 0, "tile");
  __shared__ __attribute__((aligned(16))) unsigned char lds[2][ROWS * BLOCK];
  __shared__ float scales[2][BM];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, half = lane >> 5;
  const int wn = wave % NW, wm = wave / NW;
  // (Workgroups go to the eight XCDs in turn: those that run at a time on one of them are a block of several columns by several rows of
  // tiles.  A strip of neighbouring columns for each XCD, which reads W once, is slower: 8192^3, an earlier form of this kernel: 1139 / 1363 us.)
  const int tiles_n = (p.n + BN - 1) / BN;
  const long long m0 = (long long)(blockIdx.x / tiles_n) * BM;
  const int n0 = (int)(blockIdx.x % tiles_n) * BN;
  const unsigned char *row[LOADS];
  int to[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; i++) {
    const int at = tid + THREADS * i, r = at >> 3;
    if (r < BN) row[i] = p.W + (long long)(n0 + r < p.n ? n0 + r : p.n - 1) * p.pitch;
    else row[i] = p.A + (m0 + r - BN < p.m ? m0 + r - BN : p.m - 1) * p.pitch;
    to[i] = r * BLOCK + 16 * ((at & 7) ^ (r & 7));
  }
  const int piece = 16 * (tid & 7);
  const float *my_scale = p.SA + (m0 + tid % BM < p.m ? m0 + tid % BM : p.m - 1) * p.blocks;
  const int wide = (n0 + 32 * TN * wn) / BLOCK;  // (columns beyond n: any scale will do)
  const float *sw = p.SW + (long long)(wide * BLOCK < p.n ? wide : 0) * p.blocks;

  const int begin = blockIdx.y * p.part, end = begin + p.part < p.blocks ? begin + p.part : p.blocks;
  Piece<true> next[LOADS];
  float next_scale;
  auto fetch = [&](int b) {
    if (b >= end) return;
#pragma unroll
    for (int i = 0; i < LOADS; i++) next[i].load(row[i], b * BLOCK + piece, p.k);
    if (tid < BM) next_scale = my_scale[b];
  };
  auto keep = [&](int b) {
    if (b >= end) return;
#pragma unroll
    for (int i = 0; i < LOADS; i++) *reinterpret_cast<i32x4 *>(&lds[b & 1][to[i]]) = next[i].d;
    if (tid < BM) scales[b & 1][tid] = next_scale;
  };
  // 16 bytes of each row of the wavefront's blocks: its share of a quarter of the slab
  i32x4 rw[TN], ra[TM];
  auto quarter = [&](int buf, int q) {
    const int at = 16 * ((2 * q + half) ^ (li & 7));
#pragma unroll
    for (int i = 0; i < TN; i++) rw[i] = *reinterpret_cast<const i32x4 *>(&lds[buf][(32 * (TN * wn + i) + li) * BLOCK + at]);
#pragma unroll
    for (int j = 0; j < TM; j++) ra[j] = *reinterpret_cast<const i32x4 *>(&lds[buf][(BN + 32 * (TM * wm + j) + li) * BLOCK + at]);
  };

  f32x16 acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; i++)
#pragma unroll
    for (int j = 0; j < TM; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[i][j][e] = 0.0f;
  fetch(begin);
  keep(begin);
  fetch(begin + 1);
  __syncthreads();
  quarter(begin & 1, 0);
  for (int b = begin; b < end; b++) {
    const int buf = b & 1;
    const float s = sw[b];
    float c[TM];
#pragma unroll
    for (int j = 0; j < TM; j++) c[j] = scales[buf][32 * (TM * wm + j) + li] * s;
    f32x16 x[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
      for (int j = 0; j < TM; j++)
#pragma unroll
        for (int e = 0; e < 16; e++) x[i][j][e] = 0.0f;
#pragma unroll
    for (int q = 0; q < 4; q++) {
      bf16x8 fw[TN][2], fa[TM][2];
#pragma unroll
      for (int i = 0; i < TN; i++) fw[i][0] = widen(rw[i][0], rw[i][1]), fw[i][1] = widen(rw[i][2], rw[i][3]);
#pragma unroll
      for (int j = 0; j < TM; j++) fa[j][0] = widen(ra[j][0], ra[j][1]), fa[j][1] = widen(ra[j][2], ra[j][3]);
      if (q == 2) {
        keep(b + 1);
        fetch(b + 2);
      }
      if (q < 3) quarter(buf, q + 1);
      else {
        __syncthreads();  // (the slab has been read, the next one is there)
        quarter(buf ^ 1, 0);
      }
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int i = 0; i < TN; i++)
#pragma unroll
          for (int j = 0; j < TM; j++) x[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fw[i][h], fa[j][h], x[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
      for (int j = 0; j < TM; j++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[i][j][e] = __builtin_fmaf(x[i][j][e], c[j], acc[i][j][e]);
  }
  float *Y = p.Y + blockIdx.y * p.m * p.n;
  // Lane: row li of a block; registers 4 q .. + 3 are columns 8 q + 4 half .. + 3.  A wavefront turns 32 rows of them at a time in a part of LDS
  // of its own (nobody reads slabs any more), so that it stores runs of 32 TN columns (8192 x 4096, K = 512: 58 us, straight from the
  // registers 81).
  constexpr int PITCH = 32 * TN + 4, LANES = 8 * TN;
  static_assert(NW * MW * 32 * PITCH * 4 <= (int)sizeof(lds), "room for the results");
  float *turn = reinterpret_cast<float *>(&lds[0][0]) + wave * (32 * PITCH);
#pragma unroll
  for (int j = 0; j < TM; j++) {
#pragma unroll
    for (int t = 0; t < TN; t++)
#pragma unroll
      for (int q = 0; q < 4; q++)
        *reinterpret_cast<f32x4 *>(&turn[li * PITCH + 32 * t + 8 * q + 4 * half]) =
            f32x4{acc[t][j][4 * q], acc[t][j][4 * q + 1], acc[t][j][4 * q + 2], acc[t][j][4 * q + 3]};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int r = 0; r < 32; r += 64 / LANES) {
      const int row = r + lane / LANES, col = 4 * (lane % LANES);
      const long long i = m0 + 32 * (TM * wm + j) + row;
      const f32x4 v = *reinterpret_cast<const f32x4 *>(&turn[row * PITCH + col]);
      if (i < p.m) finish4(p, Y, i, n0 + 32 * TN * wn + col, v);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

template <int NW, int MW, int TN, int TM>
void launch_tiles(const ProductParams &p) {
  constexpr int BN = 32 * NW * TN, BM = 32 * MW * TM;
  const long long tiles = (p.n + BN - 1) / BN * ((p.m + BM - 1) / BM);
  hipLaunchKernelGGL((product_tiles<NW, MW, TN, TM>), dim3((unsigned)tiles, parts_of(p)), dim3(64 * NW * MW), 0, wdh::stream(), p);
}

// The parts of a product together, in order: four results to a lane.
__global__ __launch_bounds__(256) void product_join(ProductParams p, const float *partial, int parts) {
  const int pieces = (p.n + 3) / 4;
  for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < p.m * pieces; at += 256LL * gridDim.x) {
    const long long i = at / pieces;
    const int j = (int)(at - i * pieces) * 4;
    const float *from = partial + i * p.n;
    f32x4 v = load4(from, j, p.n);
#pragma unroll 8
    for (int part = 1; part < parts; part++) v = v + load4(from + part * p.m * p.n, j, p.n);
    finish4(p, p.Y, i, j, v);
  }
}

// Rows of a length that is no multiple of 16, copied to rows that are (zeros behind their end): A's, then W's.
__global__ __launch_bounds__(256) void pack_rows(const unsigned char *A, const unsigned char *W, unsigned char *to, long long m, long long rows, int k,
                                                 long long pitch) {
  for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += 4LL * gridDim.x) {
    const unsigned char *row = r < m ? A + r * k : W + (r - m) * k;
    for (int at = 16 * (threadIdx.x & 63); at < k; at += 4096) {
      Piece<false> x[4];
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (at + 1024 * i < k) x[i].load(row, at + 1024 * i, k);
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (at + 1024 * i < k) *reinterpret_cast<i32x4 *>(to + r * pitch + at + 1024 * i) = x[i].get(row, at + 1024 * i, k);
    }
  }
}

// Which form a product takes, and in how many parts along K.  A workgroup of a form takes `start` + `block` per block of K us (measured
// with every CU busy: K of 2048 to 14336, 1 to 8192 rows).  Wavefronts of the first forms take blocks eight (64 x 64: four) at a time; odd
// rows cost these 1.4 times as much, the others the copy.  Tiles that leave CUs idle are cut along K into as many parts as there are CUs
// for; the parts' join is a launch of 4 us, 0.15 for each part and its bytes.  The cheapest of all wins (us, so / the smallest tile that fits the chip, uncut:
// 4096 columns, K = 14336: 17 rows 16.4 / 19.9, 64 rows 23 / 25, 256 rows 47 / 53; 8192 x 8192: 128 rows 33 / 34, 256 rows 51 / 57, 1024
// rows 139 / 161).
struct Form {
  int cols, rows;
  float start, block;
};
constexpr int FIRST_TILES = 6, FORMS = 9;
constexpr Form forms[FORMS] = {{16, 16, 3.0f, 0.116f}, {32, 16, 1.9f, 0.16f}, {64, 16, 2.2f, 0.21f},   {32, 32, 1.5f, 0.21f},  {64, 32, 2.0f, 0.28f},
                               {64, 64, 5.0f, 0.43f},  {128, 64, 4.0f, 0.85f}, {128, 128, 8.0f, 1.2f}, {256, 128, 9.0f, 2.0f}};
struct Plan {
  int form, parts;
};
Plan cheapest_plan(const ProductParams &p, bool aligned) {
  const long long cus = wdh::compute_units();
  Plan best = {0, 1};
  double least = -1.0;
  for (int f = 0; f < FORMS; f++) {
    const long long tiles = ((p.n + forms[f].cols - 1LL) / forms[f].cols) * ((p.m + forms[f].rows - 1) / forms[f].rows);
    const bool direct = f < FIRST_TILES;
    const double block = forms[f].block * (direct && !aligned ? 1.4 : 1.0);
    const long long turns = f == FIRST_TILES - 1 ? 4 : 8;  // (wavefronts)
    for (int cut = 0; cut < 2; cut++) {
      long long parts = cut ? cus / tiles : 1;
      if (parts > p.blocks) parts = p.blocks;
      if (cut && parts < 2) continue;
      const long long part = parts > 1 ? (p.blocks + parts - 1) / parts : p.blocks;
      if (parts > 1) parts = (p.blocks + part - 1) / part;
      const double rounds = (double)((tiles * parts + cus - 1) / cus);
      double us = rounds * (forms[f].start + block * (double)(direct ? (part + turns - 1) / turns * turns : part));
      if (parts > 1) us += 4.0 + (double)parts * (0.15 + (double)p.m * p.n * 8e-7);
      if (!direct && !aligned) us += 3.0 + (double)(p.m + p.n) * p.k * 4e-7;  // (the copy)
      if (least < 0.0 || us < least) {
        least = us;
        best = Plan{f, (int)parts};
      }
    }
  }
  return best;
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
  if (n > (1 << 28) || k > (1 << 30) || m > (1LL << 46) / n || (k && m > (1LL << 46) / k) || (m + 127) / 128 * (((long long)n + 127) / 128) > 0x7fffff)
    return fail(WDH_EINVAL, "wdh_gemm_fp8: too many elements");
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
  p.pitch = k;
  p.part = p.blocks;
  bool aligned = k % 16 == 0;  // (buffers start on 512-byte boundaries)
  if (m <= 2) {  // (see product_rows)
    if (m == 1) launch_rows<1>(p, aligned);
    else launch_rows<2>(p, aligned);
    WDH_LAUNCH_CHECK();
    return WDH_OK;
  }
  Plan plan = cheapest_plan(p, aligned);
  // Tiles of many rows take rows of whole 16-byte pieces: others are copied first.
  wdh_buf packed = 0;
  if (!aligned && plan.form >= FIRST_TILES) {
    const long long pitch = ((long long)k + 15) / 16 * 16, rows = m + n;
    packed = wdh_alloc((size_t)(rows * pitch));
    size_t have;
    unsigned char *to = packed ? (unsigned char *)wdh::resolve(packed, &have) : nullptr;
    if (to) {
      hipLaunchKernelGGL(pack_rows, dim3((unsigned)(rows < (1 << 18) ? (rows + 3) / 4 : 1 << 16)), dim3(256), 0, wdh::stream(), p.A, p.W, to,
                         (long long)m, rows, k, pitch);
      p.A = to;
      p.W = to + m * pitch;
      p.pitch = pitch;
      aligned = true;
    } else plan = Plan{FIRST_TILES - 1, 1};  // (no room for the copy: the direct form takes any rows)
  }
  // Parts go to a workspace and are joined; without room for it there is one part.
  wdh_buf work = 0;
  ProductParams parts = p;
  float *partial = nullptr;
  if (plan.parts > 1 && (work = wdh_alloc((size_t)plan.parts * results))) {
    size_t have;
    parts.Y = partial = (float *)wdh::resolve(work, &have);
    parts.part = (p.blocks + plan.parts - 1) / plan.parts;
    parts.bias = parts.R = nullptr;
    parts.relu = 0;
  }
  switch (plan.form) {
    case 0: launch_few<1, 1, 8>(parts, aligned); break;
    case 1: launch_few<2, 1, 8>(parts, aligned); break;
    case 2: launch_few<4, 1, 8>(parts, aligned); break;
    case 3: launch_few<2, 2, 8>(parts, aligned); break;
    case 4: launch_few<4, 2, 8>(parts, aligned); break;
    case 5: launch_few<4, 4, 4>(parts, aligned); break;
    case 6: launch_tiles<4, 2, 1, 1>(parts); break;
    case 7: launch_tiles<4, 2, 1, 2>(parts); break;
    default: launch_tiles<4, 2, 2, 2>(parts); break;
  }
  if (work) {
    const long long pieces = m * (((long long)n + 3) / 4);
    hipLaunchKernelGGL(product_join, dim3((unsigned)(pieces < (1LL << 30) ? (pieces + 255) / 256 : 1 << 22)), dim3(256), 0, wdh::stream(), p, partial,
                       plan.parts);
    (void)wdh_free(work);
  }
  if (packed) (void)wdh_free(packed);
  WDH_LAUNCH_CHECK();
  return WDH_OK;
}
