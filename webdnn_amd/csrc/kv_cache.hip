// A cache of keys and values held in e4m3, in pages of 64 tokens, and attention over it.
//
// The reference has neither; its attention is the chain MatMul, Mul, Softmax, MatMul over whole tensors
// (src/descriptor_runner/operators/cpu/operators/standard/matmul.ts:11-111, softmax.ts:34-57).
//
// A page belongs to one sequence and holds, for each of the cache's heads, 64 keys as [token][d] and 64 values as [d][token]
// (what the second product of attention reads along is contiguous), each with one scale: element = e4m3 value * scale.
// Scales are powers of two: when a later token outgrows its page, the earlier ones are scaled down without another rounding
// (but for those that leave the range of normal e4m3 numbers).
#include <stdio.h>

#include "common.h"
#include "fp8.h"

namespace {

using namespace wdh::fp8;

constexpr int PAGE = 64;
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// Which tokens of a call belong to which sequence, and where the sequences lie in the cache.
struct Sequences {
  const int *table;   // [seqs, max_pages]
  const int *lens;    // [seqs], the tokens of the call counted
  const int *starts;  // [seqs + 1]
  int seqs, tokens, max_pages, pages;
};
struct Place {
  int seq, row0, n, len, index;  // rows row0 .. row0+n-1 of the call are the last n of the sequence's len tokens
};

// A sequence's rows; n = 0 for one that has none, or whose numbers do not fit the call or the table.
__device__ __forceinline__ Place sequence(const Sequences &q, int s) {
  Place p;
  p.seq = s;
  p.row0 = q.starts[s];
  p.len = q.lens[s];
  const long long n = (long long)q.starts[s + 1] - p.row0;
  const bool fits = p.row0 >= 0 && n > 0 && p.row0 + n <= q.tokens && n <= p.len && p.len <= (long long)q.max_pages * PAGE;
  p.n = fits ? (int)n : 0;
  p.index = 0;
  return p;
}

// The sequence that holds work item `item` when each has count(place) of them in turn, and which of its items that is; n = 0
// behind the last.  Whole wavefronts call this: 64 sequences are looked at side by side.
template <class Count>
__device__ __forceinline__ Place locate(const Sequences &q, long long item, Count count) {
  const int lane = threadIdx.x & 63;
  for (int s0 = 0; s0 < q.seqs; s0 += 64) {
    Place p = {0, 0, 0, 0, 0};
    if (s0 + lane < q.seqs) p = sequence(q, s0 + lane);
    const int mine = p.n ? count(p) : 0;
    long long upto = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const long long below = __shfl_up(upto, off, 64);
      if (lane >= off) upto += below;
    }
    const unsigned long long has = __ballot(item < upto);
    if (has) {
      const int at = __ffsll(has) - 1;
      const long long before = __shfl(upto - mine, at, 64);
      Place r;
      r.seq = __builtin_amdgcn_readlane(p.seq, at);
      r.row0 = __builtin_amdgcn_readlane(p.row0, at);
      r.n = __builtin_amdgcn_readlane(p.n, at);
      r.len = __builtin_amdgcn_readlane(p.len, at);
      r.index = __builtin_amdgcn_readfirstlane((int)(item - before));
      return r;
    }
    item -= __shfl(upto, 63, 64);
  }
  return Place{0, 0, 0, 0, 0};
}

// ---- append --------------------------------------------------------------------------------
struct AppendParams {
  Sequences q;
  const float *K, *V;
  long long k_stride, v_stride;  // elements between tokens
  unsigned char *KP, *VP;
  float *KS, *VS;
  int heads;
};

// The least power of two c >= 2^-100 with amax <= 448 c (448 = 0.875 * 2^9).
__device__ __forceinline__ float page_scale(float amax) {
  const int bits = __float_as_int(amax);
  int e = (bits >> 23) - 126;
  e = (bits & 0x7fffff) <= 0x600000 ? e - 9 : e - 8;
  return __int_as_float(((e > -100 ? e : -100) + 127) << 23);
}

// Four packed e4m3 values times a factor.
__device__ __forceinline__ int rescale4(int q, float factor) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(q, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(q, true);
  return pack4(f32x4{a[0], a[1], b[0], b[1]}, factor);
}
// Bytes first .. last-1 of four are taken from `fresh`, those below from `old` or, if the page's scale grew, from `old` scaled.
__device__ __forceinline__ int merge4(int old, int fresh, int first, int last, bool grown, float factor) {
  const int again = grown ? rescale4(old, factor) : old;
  unsigned r = 0;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const unsigned from = e < first ? (unsigned)again : e < last ? (unsigned)fresh : (unsigned)old;
    r |= from & (0xffu << (8 * e));
  }
  return (int)r;
}

// A workgroup owns a touched page of one head, keys (blockIdx.z 0) or values: nobody else reads or writes it, and its scale
// needs the largest of the new elements before any of them is stored.  They stay in registers in between.
// Bound: memory for prompts, latency for single tokens.
template <int D>
__global__ __launch_bounds__(256) void cache_append(AppendParams p) {
  constexpr int NP = PAGE * D / 4 / 256;       // pieces of four elements a thread holds
  constexpr int PPT = D / 4;                   // pieces of a token
  __shared__ float part[4];
  __shared__ int turn[PAGE * (D / 4 + 1)];     // values on their way from [token][d] to [d][token], four to a word
  const Place s = locate(p.q, blockIdx.x, [](const Place &s) { return (s.len - 1) / PAGE - (s.len - s.n) / PAGE + 1; });
  if (s.n == 0) return;
  const int before = s.len - s.n, pi = before / PAGE + s.index, id = p.q.table[(long long)s.seq * p.q.max_pages + pi];
  if (id < 0 || id >= p.q.pages) return;
  const bool values = blockIdx.z;
  const int head = blockIdx.y, t = threadIdx.x;
  const int first = before > pi * PAGE ? before - pi * PAGE : 0, last = s.len - pi * PAGE < PAGE ? s.len - pi * PAGE : PAGE;
  const long long stride = values ? p.v_stride : p.k_stride;
  // (token `slot` of the page is row row0 + pi*64 + slot - before of the call)
  const float *x = (values ? p.V : p.K) + head * D;
  const long long row0 = (long long)s.row0 + (long long)pi * PAGE - before;
  const long long at = (long long)id * p.heads + head;
  unsigned char *page = (values ? p.VP : p.KP) + at * (PAGE * D);
  float *scale = (values ? p.VS : p.KS) + at;
  f32x4 v[NP];
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < NP; i++) {
    const int slot = (t + 256 * i) / PPT, d0 = (t + 256 * i) % PPT * 4;
    v[i] = slot >= first && slot < last ? *reinterpret_cast<const f32x4 *>(x + (row0 + slot) * stride + d0) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; e++) amax = fmaxf(amax, finite_abs(v[i][e]));
  }
  const float old = first > 0 ? *scale : 0.0f;
  amax = wdh::rowmath::wave_max(amax);
  if ((t & 63) == 0) part[t >> 6] = amax;
  __syncthreads();
  const float need = page_scale(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
  const float c = first > 0 ? fmaxf(old, need) : need, inv = 1.0f / c, factor = old / c;
  const bool grown = first > 0 && c != old;
  if (!values) {
#pragma unroll
    for (int i = 0; i < NP; i++) {
      const int slot = (t + 256 * i) / PPT;
      int *to = reinterpret_cast<int *>(page) + t + 256 * i;
      if (slot >= first && slot < last) *to = pack4(v[i], inv);
      else if (slot < first && grown) *to = rescale4(*to, factor);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NP; i++) turn[(t + 256 * i) / PPT * (PPT + 1) + (t + 256 * i) % PPT] = pack4(v[i], inv);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NP; i++) {
      const int d = (t + 256 * i) / (PAGE / 4), s0 = (t + 256 * i) % (PAGE / 4) * 4;
      if (s0 >= last || (s0 + 4 <= first && !grown)) continue;
      int fresh = 0;
#pragma unroll
      for (int e = 0; e < 4; e++) fresh |= (int)(((unsigned)turn[(s0 + e) * (PPT + 1) + d / 4] >> (8 * (d & 3))) & 0xffu) << (8 * e);
      int *to = reinterpret_cast<int *>(page) + t + 256 * i;
      *to = s0 >= first && s0 + 4 <= last ? fresh : merge4(*to, fresh, first - s0, last - s0, grown, factor);
    }
  }
  if (t == 0) *scale = c;
}

// ---- attention -------------------------------------------------------------------------------
struct AttendParams {
  Sequences q;
  const float *Q;
  long long q_stride;
  const unsigned char *KP, *VP;
  const float *KS, *VS;
  float *Y;
  int heads, kv_heads, group;
  float scale;       // alpha * log2(e): powers are taken of two
  int splits;
  float *partial;    // splits > 1: [item][kv head][split][16][D + 2]
};

__device__ __forceinline__ float wave_pairs_max(float v) {  // over the four lanes that share lane % 16
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float wave_pairs_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// Eight fp32 values as the sums of three bfloat16 ones each: the upper 8 significant bits, the next 8, the rest.  Exact, so the
// products with e4m3 values (exact in fp32) lose nothing that fp32 operands would keep.
__device__ __forceinline__ void split3(const float (&x)[8], bf16x8 (&part)[3]) {
  union { unsigned u[4]; bf16x8 v; } r[3];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    unsigned a = __float_as_uint(x[2 * i]), b = __float_as_uint(x[2 * i + 1]);
#pragma unroll
    for (int k = 0; k < 3; k++) {
      r[k].u[i] = __builtin_amdgcn_perm(b, a, 0x07060302);  // the upper halves of both
      if (k == 2) break;
      a = __float_as_uint(__uint_as_float(a) - __uint_as_float(a & 0xffff0000u));
      b = __float_as_uint(__uint_as_float(b) - __uint_as_float(b & 0xffff0000u));
    }
  }
#pragma unroll
  for (int k = 0; k < 3; k++) part[k] = r[k].v;
}

// 16 rows (a row is a token and one of the `group` queries that share a head of the cache) against the pages of their sequence;
// the wavefronts of a workgroup, and the workgroups of a split, take pages in turn.  Everything is computed transposed:
//   S^T [key][row] = K Q^T    (v_mfma_f32_16x16x32_bf16, K widened from e4m3, Q in three bfloat16 parts)
//   O^T [d][row]  += V^T P^T  (V^T is how pages hold values, P in three parts)
// so that a lane holds scores of one row, P is an operand of the second product as it stands, and both K and V pass from memory
// into operand registers with 16-byte loads.  That takes an order of keys in which the four that a lane gets from score tile t are
// keys 16 g + 4 t .. + 3 of the page (g = lane / 16), and an order of d in which a lane's 16 bytes serve two products.
template <int D>
__global__ __launch_bounds__(256, 2) void attend_rows(AttendParams p) {
  constexpr int STEPS = D / 32, CH = D >= 64 ? D / 64 : 1, DT = D / 16;
  constexpr int OP = D + 4;
  __shared__ __attribute__((aligned(16))) float outs[4][16 * OP];
  __shared__ float tops[4][16], sums[4][16];
  const int group = p.group;
  const Place s = locate(p.q, blockIdx.x, [group](const Place &s) { return (int)(((long long)s.n * group + 15) / 16); });
  if (s.n == 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i16 = lane & 15, g = lane >> 4;
  const int head = blockIdx.y;
  // this lane's row
  const long long flat = (long long)s.index * 16 + i16;
  const int token = (int)(flat / group), sub = (int)(flat - (long long)token * group);
  const bool live = token < s.n;
  const int limit = live ? s.len - s.n + token : -1;  // its last key
  const float *qrow = p.Q + (long long)(s.row0 + (live ? token : 0)) * p.q_stride + (long long)(head * group + sub) * D;
  bf16x8 q[STEPS][3];
#pragma unroll
  for (int st = 0; st < STEPS; st++) {
    const int d0 = D >= 64 ? 64 * (st / 2) + 16 * g + 8 * (st & 1) : 8 * g;
    const f32x4 a = *reinterpret_cast<const f32x4 *>(qrow + d0), b = *reinterpret_cast<const f32x4 *>(qrow + d0 + 4);
    const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    split3(x, q[st]);
  }
  const int last_token = (int)(((long long)s.index * 16 + 15) / group);
  const int last_key = s.len - s.n + (last_token < s.n ? last_token : s.n - 1);
  const int count = last_key / PAGE + 1, step = 4 * p.splits;
  const int *table = p.q.table + (long long)s.seq * p.q.max_pages;

  f32x4 o[DT];
#pragma unroll
  for (int i = 0; i < DT; i++) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, sum = 0.0f;
  for (int pg = blockIdx.z * 4 + wave; pg < count; pg += step) {
    int id = table[pg];
    const bool known = id >= 0 && id < p.q.pages;  // (a page that is not there makes its rows NaN)
    if (!known) id = 0;
    const long long at = (long long)id * p.kv_heads + head;
    const unsigned char *kp = p.KP + at * (PAGE * D), *vp = p.VP + at * (PAGE * D);
    // (a scale that is no number shows through the scores, which are masked, not through 0 * NaN)
    float ks = p.KS[at], vs = p.VS[at];
    if (!known || !(fabsf(vs) <= FLT_MAX)) ks = NAN, vs = 0.0f;
    i32x4 k[4][CH], v[DT];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const unsigned char *row = kp + (16 * (i16 >> 2) + 4 * t + (i16 & 3)) * D;
      if constexpr (D >= 64) {
#pragma unroll
        for (int c = 0; c < CH; c++) k[t][c] = *reinterpret_cast<const i32x4 *>(row + 64 * c + 16 * g);
      } else {
        const i32x2 h = *reinterpret_cast<const i32x2 *>(row + 8 * g);
        k[t][0] = i32x4{h[0], h[1], 0, 0};
      }
    }
#pragma unroll
    for (int i = 0; i < DT; i++) v[i] = *reinterpret_cast<const i32x4 *>(vp + (16 * i + i16) * PAGE + 16 * g);
    float x[16];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < STEPS; st++) {
        const bf16x8 kw = widen(k[t][st / 2][2 * (st & 1)], k[t][st / 2][2 * (st & 1) + 1]);
#pragma unroll
        for (int part = 2; part >= 0; part--) a = mfma(kw, q[st][part], a);
      }
#pragma unroll
      for (int r = 0; r < 4; r++) x[4 * t + r] = a[r];
    }
    // softmax: keys beyond the row's last, and whatever the page holds behind the sequence, count for nothing
    const float c = p.scale * ks;
    float most = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const bool in = pg * PAGE + 16 * g + e <= limit;
      most = fmaxf(most, in ? x[e] * c : -INFINITY);
    }
    most = wave_pairs_max(fmaxf(most, top));
    const float ref = most == -INFINITY ? 0.0f : most, back = __builtin_amdgcn_exp2f(top - ref);
    top = most;
    sum *= back;
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) o[i][e] *= back;
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const bool in = pg * PAGE + 16 * g + e <= limit;
      x[e] = in ? __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], c, -ref)) : 0.0f;
      sum += x[e];
    }
    bf16x8 pr[2][3];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; e++) y[e] = x[8 * u + e] * vs;
      split3(y, pr[u]);
    }
    // Values of keys that some row of the 16 does not see: those behind the sequence are put to 0 (0 * NaN is NaN), and a NaN among the
    // others is kept from the rows before it by hand.
    const int first_limit = s.len - s.n + (int)((long long)s.index * 16 / group);
    bool poison = false;
    if (pg * PAGE + PAGE - 1 > first_limit) {
      const int behind = s.len - pg * PAGE - 16 * g;  // how many of the lane's 16 keys are the sequence's
      int bad = 0;
#pragma unroll
      for (int i = 0; i < DT; i++)
#pragma unroll
        for (int w = 0; w < 4; w++) {
          const int n = behind - 4 * w;
          unsigned b = (unsigned)v[i][w] & (n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u);
          const unsigned nan = ((b & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
          bad |= (int)nan;
          v[i][w] = (int)(b & ~((nan >> 7) * 0xffu));
        }
      poison = __any(bad != 0);
    }
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const bf16x8 vw = widen(v[i][2 * u], v[i][2 * u + 1]);
#pragma unroll
        for (int part = 2; part >= 0; part--) o[i] = mfma(vw, pr[u][part], o[i]);
      }
    if (poison) {
      for (int j = 0; j < PAGE && pg * PAGE + j <= limit; j++)
#pragma unroll
        for (int i = 0; i < DT; i++)
#pragma unroll
          for (int e = 0; e < 4; e++)
            if ((vp[(16 * i + 4 * g + e) * PAGE + j] & 0x7f) == 0x7f) o[i][e] = NAN;
    }
  }
  sum = wave_pairs_sum(sum);

  // the wavefronts' shares together
#pragma unroll
  for (int i = 0; i < DT; i++) *reinterpret_cast<f32x4 *>(&outs[wave][i16 * OP + 16 * i + 4 * g]) = o[i];
  if (g == 0) {
    tops[wave][i16] = top;
    sums[wave][i16] = sum;
  }
  __syncthreads();
  for (int cell = threadIdx.x; cell < 16 * D; cell += 256) {
    const int row = cell / D, d = cell - row * D;
    float most = fmaxf(fmaxf(tops[0][row], tops[1][row]), fmaxf(tops[2][row], tops[3][row]));
    const float ref = most == -INFINITY ? 0.0f : most;
    float total = 0.0f, y = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float f = __builtin_amdgcn_exp2f(tops[w][row] - ref);
      total += f * sums[w][row];
      y += f * outs[w][row * OP + d];
    }
    const long long flat_row = (long long)s.index * 16 + row;
    const int tk = (int)(flat_row / group);
    if (tk >= s.n) continue;
    if (p.splits == 1) {
      p.Y[((long long)(s.row0 + tk) * p.heads + head * group + (flat_row - (long long)tk * group)) * D + d] = total == 0.0f ? 0.0f : y / total;
    } else {
      float *to = p.partial + ((((long long)blockIdx.x * p.kv_heads + head) * p.splits + blockIdx.z) * 16 + row) * (D + 2);
      to[d] = y;
      if (d == 0) {
        to[D] = most;
        to[D + 1] = total;
      }
    }
  }
}

// The shares of the splits together: a workgroup to the 16 rows of an item.
template <int D>
__global__ __launch_bounds__(256) void attend_join(AttendParams p) {
  const int group = p.group, head = blockIdx.y;
  const Place s = locate(p.q, blockIdx.x, [group](const Place &s) { return (int)(((long long)s.n * group + 15) / 16); });
  if (s.n == 0) return;
  for (int cell = threadIdx.x; cell < 16 * D; cell += 256) {
    const int row = cell / D, d = cell - row * D;
    const long long flat_row = (long long)s.index * 16 + row;
    const int tk = (int)(flat_row / group);
    if (tk >= s.n) continue;
    const float *from = p.partial + ((((long long)blockIdx.x * p.kv_heads + head) * p.splits) * 16 + row) * (D + 2);
    const long long pitch = 16 * (D + 2);
    float most = -INFINITY;
    for (int i = 0; i < p.splits; i++) most = fmaxf(most, from[i * pitch + D]);
    const float ref = most == -INFINITY ? 0.0f : most;
    float total = 0.0f, y = 0.0f;
    for (int i = 0; i < p.splits; i++) {
      const float f = __builtin_amdgcn_exp2f(from[i * pitch + D] - ref);
      total += f * from[i * pitch + D + 1];
      y += f * from[i * pitch + d];
    }
    p.Y[((long long)(s.row0 + tk) * p.heads + head * group + (flat_row - (long long)tk * group)) * D + d] = total == 0.0f ? 0.0f : y / total;
  }
}

template <int D>
int launch_attend(const AttendParams &p, long long items) {
  hipStream_t st = wdh::stream();
  hipLaunchKernelGGL((attend_rows<D>), dim3((unsigned)items, (unsigned)p.kv_heads, (unsigned)p.splits), dim3(256), 0, st, p);
  WDH_LAUNCH_CHECK();
  if (p.splits > 1) {
    hipLaunchKernelGGL((attend_join<D>), dim3((unsigned)items, (unsigned)p.kv_heads), dim3(256), 0, st, p);
    WDH_LAUNCH_CHECK();
  }
  return WDH_OK;
}

using wdh::fail;

// What append and attention ask of their sequences and of the cache.
int check_cache(const char *who, int seqs, int tokens, int kv_heads, int d, int pages, int max_pages) {
  if (seqs < 0 || tokens < 0 || kv_heads < 0 || pages < 0 || max_pages < 0) return fail(WDH_EINVAL, "%s: negative extent", who);
  if (d != 32 && d != 64 && d != 128) return fail(WDH_EINVAL, "%s: head dimension %d (32, 64 and 128 are built)", who, d);
  if (kv_heads == 0 || kv_heads > 65535) return fail(WDH_EINVAL, "%s: %d heads of the cache (1 to 65535)", who, kv_heads);
  if (max_pages > (1 << 24)) return fail(WDH_EINVAL, "%s: tables of %d pages (at most %d)", who, max_pages, 1 << 24);
  if (tokens > (1 << 24) || seqs > (1 << 20)) return fail(WDH_EINVAL, "%s: too many tokens or sequences", who);
  return WDH_OK;
}
int cache_operands(const char *who, wdh_buf hKP, wdh_buf hKS, wdh_buf hVP, wdh_buf hVS, wdh_buf hT, wdh_buf hL, wdh_buf hS, int seqs, int kv_heads,
                   int d, int pages, int max_pages, void **kp, void **ks, void **vp, void **vs, Sequences *q) {
  const size_t cells = (size_t)pages * kv_heads;
  char what[64];
  auto get = [&](wdh_buf h, size_t need, const char *name, void **out) {
    snprintf(what, sizeof(what), "%s: %s", who, name);
    return wdh::operand(h, need, what, out);
  };
  void *t, *l, *s;
  if (!get(hKP, cells * PAGE * d, "KPages", kp) || !get(hKS, cells * 4, "KScales", ks) || !get(hVP, cells * PAGE * d, "VPages", vp) ||
      !get(hVS, cells * 4, "VScales", vs) || !get(hT, (size_t)seqs * max_pages * 4, "Table", &t) || !get(hL, (size_t)seqs * 4, "Lens", &l) ||
      !get(hS, ((size_t)seqs + 1) * 4, "Starts", &s))
    return WDH_EINVAL;
  q->table = (const int *)t;
  q->lens = (const int *)l;
  q->starts = (const int *)s;
  q->seqs = seqs;
  q->max_pages = max_pages;
  q->pages = pages;
  return WDH_OK;
}
// Rows of `width` elements, `stride` apart from element `offset` of the buffer on, that are read 16 bytes at a time.
int check_rows(const char *who, const char *name, int64_t offset, int64_t stride, int64_t width) {
  if (offset < 0 || stride < width || offset > (1LL << 46) || stride > (1LL << 22))
    return fail(WDH_EINVAL, "%s: %s rows of %lld elements from %lld on, %lld apart", who, name, (long long)width, (long long)offset, (long long)stride);
  if (offset % 4 || stride % 4) return fail(WDH_EINVAL, "%s: offset and stride of %s must be multiples of 4 elements", who, name);
  return WDH_OK;
}

}  // namespace

extern "C" int wdh_cache_append(wdh_buf hK, int64_t k_offset, int64_t k_stride, wdh_buf hV, int64_t v_offset, int64_t v_stride, wdh_buf hKP,
                                wdh_buf hKS, wdh_buf hVP, wdh_buf hVS, wdh_buf hTable, wdh_buf hLens, wdh_buf hStarts, int seqs, int tokens,
                                int kv_heads, int d, int pages, int max_pages) {
  WDH_REQUIRE_INIT();
  WDH_REQUIRE_COMPUTE_LANE();
  const char *who = "wdh_cache_append";
  if (int rc = check_cache(who, seqs, tokens, kv_heads, d, pages, max_pages)) return rc;
  const int64_t width = (int64_t)kv_heads * d;
  if (int rc = check_rows(who, "K", k_offset, k_stride, width)) return rc;
  if (int rc = check_rows(who, "V", v_offset, v_stride, width)) return rc;
  if (seqs == 0 || tokens == 0 || pages == 0 || max_pages == 0) return WDH_OK;
  AppendParams p;
  void *pk, *pv, *kp, *ks, *vp, *vs;
  if (!wdh::operand(hK, (size_t)(k_offset + (tokens - 1) * k_stride + width) * 4, "wdh_cache_append: K", &pk)) return WDH_EINVAL;
  if (!wdh::operand(hV, (size_t)(v_offset + (tokens - 1) * v_stride + width) * 4, "wdh_cache_append: V", &pv)) return WDH_EINVAL;
  if (int rc = cache_operands(who, hKP, hKS, hVP, hVS, hTable, hLens, hStarts, seqs, kv_heads, d, pages, max_pages, &kp, &ks, &vp, &vs, &p.q)) return rc;
  const wdh_buf out[4] = {hKP, hKS, hVP, hVS}, in[5] = {hK, hV, hTable, hLens, hStarts};
  for (int i = 0; i < 4; i++) {
    for (wdh_buf h : in)
      if (out[i] == h) return fail(WDH_EINVAL, "%s: a part of the cache aliases an input", who);
    for (int j = 0; j < i; j++)
      if (out[i] == out[j]) return fail(WDH_EINVAL, "%s: two parts of the cache share a buffer", who);
  }
  p.q.tokens = tokens;
  p.K = (const float *)pk + k_offset;
  p.V = (const float *)pv + v_offset;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.KP = (unsigned char *)kp; p.KS = (float *)ks; p.VP = (unsigned char *)vp; p.VS = (float *)vs;
  p.heads = kv_heads;
  // touched pages: each has a new token, and a sequence's are at most n / 64 + 2
  const long long bound = (long long)tokens / PAGE + 2LL * seqs, items = bound < tokens ? bound : tokens;
  const dim3 grid((unsigned)items, (unsigned)kv_heads, 2);
  if (d == 32) hipLaunchKernelGGL((cache_append<32>), grid, dim3(256), 0, wdh::stream(), p);
  else if (d == 64) hipLaunchKernelGGL((cache_append<64>), grid, dim3(256), 0, wdh::stream(), p);
  else hipLaunchKernelGGL((cache_append<128>), grid, dim3(256), 0, wdh::stream(), p);
  WDH_LAUNCH_CHECK();
  return WDH_OK;
}

extern "C" int wdh_cache_attention(wdh_buf hQ, int64_t q_offset, int64_t q_stride, wdh_buf hKP, wdh_buf hKS, wdh_buf hVP, wdh_buf hVS,
                                   wdh_buf hTable, wdh_buf hLens, wdh_buf hStarts, wdh_buf hY, int seqs, int tokens, int heads, int kv_heads,
                                   int d, int pages, int max_pages, float alpha) {
  WDH_REQUIRE_INIT();
  WDH_REQUIRE_COMPUTE_LANE();
  const char *who = "wdh_cache_attention";
  if (int rc = check_cache(who, seqs, tokens, kv_heads, d, pages, max_pages)) return rc;
  if (heads <= 0 || heads % kv_heads || heads > 65536) return fail(WDH_EINVAL, "%s: %d heads on %d of the cache", who, heads, kv_heads);
  const int64_t width = (int64_t)heads * d;
  if (int rc = check_rows(who, "Q", q_offset, q_stride, width)) return rc;
  if (seqs == 0 || tokens == 0 || pages == 0 || max_pages == 0) return WDH_OK;
  AttendParams p;
  void *pq, *py, *kp, *ks, *vp, *vs;
  if (!wdh::operand(hQ, (size_t)(q_offset + (tokens - 1) * q_stride + width) * 4, "wdh_cache_attention: Q", &pq)) return WDH_EINVAL;
  if (!wdh::operand(hY, (size_t)tokens * width * 4, "wdh_cache_attention: Y", &py)) return WDH_EINVAL;
  if (int rc = cache_operands(who, hKP, hKS, hVP, hVS, hTable, hLens, hStarts, seqs, kv_heads, d, pages, max_pages, &kp, &ks, &vp, &vs, &p.q)) return rc;
  for (wdh_buf h : {hQ, hKP, hKS, hVP, hVS, hTable, hLens, hStarts})
    if (h == hY) return fail(WDH_EINVAL, "%s: Y aliases an input", who);
  p.q.tokens = tokens;
  p.Q = (const float *)pq + q_offset;
  p.q_stride = q_stride;
  p.KP = (const unsigned char *)kp; p.KS = (const float *)ks; p.VP = (const unsigned char *)vp; p.VS = (const float *)vs;
  p.Y = (float *)py;
  p.heads = heads; p.kv_heads = kv_heads; p.group = heads / kv_heads;
  p.scale = alpha * 1.44269504088896341f;
  // items of 16 rows: a sequence of n tokens has ceil(n group / 16)
  const long long loose = (long long)tokens * p.group / 16 + seqs, tight = (long long)tokens * ((p.group + 15) / 16);
  const long long items = loose < tight ? loose : tight;
  if (items > 0xffffffffLL / 256) return fail(WDH_EINVAL, "%s: too many rows", who);
  const long long wanted = 2LL * wdh::compute_units(), have = items * kv_heads, most = ((long long)max_pages + 7) / 8;
  long long splits = (wanted + have - 1) / have;
  p.splits = (int)(splits < most ? splits : most);
  p.partial = nullptr;
  wdh_buf work = 0;
  if (p.splits > 1) {
    work = wdh_alloc((size_t)have * p.splits * 16 * (d + 2) * 4);
    if (!work) return WDH_ENOMEM;
    size_t have_bytes;
    p.partial = (float *)wdh::resolve(work, &have_bytes);
  }
  const int rc = d == 32 ? launch_attend<32>(p, items) : d == 64 ? launch_attend<64>(p, items) : launch_attend<128>(p, items);
  if (work) (void)wdh_free(work);
  return rc;
}
