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
#include "fastdiv.h"
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

// A sequence's rows; n = 0 for one that has none, whose numbers do not fit the call or the table, or that is not there.
__device__ __forceinline__ Place sequence(const Sequences &q, int s) {
  Place p = {s, 0, 0, 0, 0};
  if (s >= q.seqs) return p;
  p.row0 = q.starts[s];
  p.len = q.lens[s];
  const long long n = (long long)q.starts[s + 1] - p.row0;
  const bool fits = p.row0 >= 0 && n > 0 && p.row0 + n <= q.tokens && n <= p.len && p.len <= (long long)q.max_pages * PAGE;
  p.n = fits ? (int)n : 0;
  return p;
}

// Sums over the lanes up to and with each: shifts within rows of 16, then the last lanes of rows 0 and 2, and of row 1, into
// those behind them.  They end at the largest int (sequences that contradict each other can claim more rows than the call has).
__device__ __forceinline__ int add_sat(int a, int b) { return __builtin_elementwise_add_sat(a, b); }
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ int dpp_add(int v) {
  return add_sat(v, __builtin_amdgcn_update_dpp(0, v, CTRL, ROW_MASK, 0xf, false));
}
__device__ __forceinline__ int wave_scan(int v) {
  v = dpp_add<0x111, 0xf>(v);
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<wdh::rowmath::DPP_BCAST15, 0xa>(v);
  return dpp_add<wdh::rowmath::DPP_BCAST31, 0xc>(v);
}
// The sequence that holds work item `item` when each has count(place) of them in turn, and which of its items that is; n = 0
// behind the last.  Whole wavefronts call this: they look at 64 sequences side by side.
template <class Count>
__device__ __forceinline__ Place locate(const Sequences &q, int item, Count count) {
  for (int i = 0; i < (q.seqs + 63) / 64; i++) {
    const Place mine = sequence(q, 64 * i + (int)(threadIdx.x & 63));
    const int items = mine.n ? count(mine) : 0, upto = wave_scan(items);
    const unsigned long long has = __ballot(item < upto);
    if (has) {
      const int at = __ffsll(has) - 1;
      return Place{__builtin_amdgcn_readlane(mine.seq, at), __builtin_amdgcn_readlane(mine.row0, at), __builtin_amdgcn_readlane(mine.n, at),
                   __builtin_amdgcn_readlane(mine.len, at), item - __builtin_amdgcn_readlane(upto - items, at)};
    }
    item -= __builtin_amdgcn_readlane(upto, 63);
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
// Bound: memory for prompts (6 of 100 to 2900 tokens, 8 heads of 128: 18.3 us, 5.0 TB/s), latency for single tokens (48: 6.6 us, a
// call's own time 5.3).
template <int D>
__global__ __launch_bounds__(256) void cache_append(AppendParams p) {
  constexpr int NP = PAGE * D / 4 / 256;       // pieces of four elements a thread holds
  constexpr int PPT = D / 4;                   // pieces of a token
  __shared__ float part[4];
  __shared__ int turn[PAGE * (D / 4 + 1)];     // values on their way from [token][d] to [d][token], four to a word
  const Place s = locate(p.q, blockIdx.x, [](const Place &s) { return (s.len - 1) / PAGE - (s.len - s.n) / PAGE + 1; });
  if (s.n == 0) return;
  const int before = s.len - s.n, pi = before / PAGE + s.index, id = p.q.table[(long long)s.seq * p.q.max_pages + pi];
  const bool values = blockIdx.z;
  const int head = blockIdx.y, t = threadIdx.x;
  const int first = before > pi * PAGE ? before - pi * PAGE : 0, last = s.len - pi * PAGE < PAGE ? s.len - pi * PAGE : PAGE;
  const long long stride = values ? p.v_stride : p.k_stride;
  // (token `slot` of the page is row row0 + slot of the call)
  const float *x = (values ? p.V : p.K) + head * D;
  const long long row0 = (long long)s.row0 + (long long)pi * PAGE - before;
  f32x4 v[NP];
#pragma unroll
  for (int i = 0; i < NP; i++) {
    const int slot = (t + 256 * i) / PPT, d0 = (t + 256 * i) % PPT * 4;
    v[i] = slot >= first && slot < last ? *reinterpret_cast<const f32x4 *>(x + (row0 + slot) * stride + d0) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (id < 0 || id >= p.q.pages) return;
  const long long at = (long long)id * p.heads + head;
  unsigned char *page = (values ? p.VP : p.KP) + at * (PAGE * D);
  float *scale = (values ? p.VS : p.KS) + at;
  // values: words of four tokens that the new ones share with others
  int shared[NP];
  if (values)
#pragma unroll
    for (int i = 0; i < NP; i++) {
      const int s0 = (t + 256 * i) % (PAGE / 4) * 4;
      shared[i] = s0 < last && s0 + 4 > first && !(s0 >= first && s0 + 4 <= last) ? reinterpret_cast<const int *>(page)[t + 256 * i] : 0;
    }
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < NP; i++)
#pragma unroll
    for (int e = 0; e < 4; e++) amax = fmaxf(amax, finite_abs(v[i][e]));
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
      if (s0 >= first && s0 + 4 <= last) *to = fresh;
      else *to = merge4(s0 + 4 <= first ? *to : shared[i], fresh, first - s0, last - s0, grown, factor);
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
  int heads, kv_heads;
  wdh::FastDiv group;  // queries that share a head of the cache
  float scale;     // alpha * log2(e): powers are taken of two
  int wgs;         // workgroups for each head of the cache (0: one for each item, which works on the whole of it)
  float *partial;  // results [workgroup][2][kv head][16][D] of items that more than one workgroup works on (null: there are none),
  float *stats;    // and their tops and sums [workgroup][2][kv head][16][2]
};

// Work of attention: items of 16 rows (a row is a token and one of the queries that share a head of the cache), each as many units
// of four pages (one for each wavefront of a workgroup) as its sequence has.  The units of all items stand in a row, and every
// workgroup takes `share` neighbouring ones: all end at the same time, whatever the sequences' lengths.
constexpr int MOST_UNITS = 1 << 30;
constexpr float LARGE_SCORE = 0x1p22f;  // from here on (as powers of two) half a step of fp32 is a quarter of an exponent and more
struct Work {
  Place s;
  int item, unit, units;  // the item, the unit of it that was asked for, and how many it has
  int before;             // units in front of the item
  int share, total;
};
__device__ __forceinline__ int items_of(const Place &s, int group) { return s.n ? (int)(((long long)s.n * group + 15) / 16) : 0; }
__device__ __forceinline__ int units_of(const Place &s) { return (s.len + 4 * PAGE - 1) / (4 * PAGE); }
// 64 sequences side by side, a lane to each; upto: units of these up to and with the lane's.
struct Look {
  Place mine;
  int items, units, upto;
};
__device__ __forceinline__ Look look(const AttendParams &p, int round) {
  Look l;
  l.mine = sequence(p.q, 64 * round + fresh(threadIdx.x & 63));
  l.items = items_of(l.mine, p.group.d);
  l.units = units_of(l.mine);
  l.upto = wave_scan(l.items * l.units);
  return l;
}
__device__ __forceinline__ int total_units(const AttendParams &p, const Look &first) {
  int total = __builtin_amdgcn_readlane(first.upto, 63);
  for (int i = 1; i < (p.q.seqs + 63) / 64; i++) total = add_sat(total, __builtin_amdgcn_readlane(look(p, i).upto, 63));
  return total <= MOST_UNITS ? total : 0;  // (more than the host allows: numbers that contradict each other)
}
// The item that holds unit number `index` of all (or, by_item, item number `index`); s.n = 0 behind the last.
__device__ __forceinline__ Work locate_work(const AttendParams &p, const Look &first, int index, bool by_item) {
  Work w;
  int before = 0, before_items = 0;
  Look l = first;
  for (int i = 0; i < (p.q.seqs + 63) / 64; i++) {
    if (i) l = look(p, i);
    const int upto = add_sat(before, l.upto), upto_items = by_item ? add_sat(before_items, wave_scan(l.items)) : 0;
    const unsigned long long has = __ballot(index < (by_item ? upto_items : upto));
    if (has) {
      const int at = __ffsll(has) - 1;
      w.s.seq = __builtin_amdgcn_readlane(l.mine.seq, at);
      w.s.row0 = __builtin_amdgcn_readlane(l.mine.row0, at);
      w.s.n = __builtin_amdgcn_readlane(l.mine.n, at);
      w.s.len = __builtin_amdgcn_readlane(l.mine.len, at);
      w.units = __builtin_amdgcn_readlane(l.units, at);
      const int begin = __builtin_amdgcn_readlane(upto - l.items * l.units, at);
      w.item = by_item ? index - __builtin_amdgcn_readlane(upto_items - l.items, at) : (index - begin) / w.units;
      w.before = begin + w.item * w.units;
      w.unit = by_item ? 0 : index - w.before;
      return w;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
    before_items = __builtin_amdgcn_readlane(upto_items, 63);
  }
  w.s = Place{0, 0, 0, 0, 0};
  return w;
}

// Element `at`, the same for the whole wavefront, of something no kernel writes meanwhile: through the scalar cache, past the
// queue of vector loads (which come back in order: behind a page's worth of them this one number would wait for all).
template <class T>
__device__ __forceinline__ T scalar(const T *from, long long at) {
  typedef const __attribute__((address_space(4))) T *constant;
  return *(constant)(uintptr_t)(from + at);
}

// A number that all lanes have alike, in a scalar register.
__device__ __forceinline__ float uniform(float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); }

// Over the four lanes that share lane % 16: a swap of a register with itself leaves both halves' values side by side.
template <class Op>
__device__ __forceinline__ float across_groups(float v, Op op) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float wave_pairs_max(float v) {
  return across_groups(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_pairs_sum(float v) {
  return across_groups(v, [](float a, float b) { return a + b; });
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

// The same for values below 2^127, rounded to nearest part by part: two subtractions of a bfloat16 from an fp32 number are one
// instruction each (a dot product with -1 and 0, exact here), 7 instructions a pair where split3 takes 11.
struct Minus { bf16x2 low, high; };
__device__ __forceinline__ Minus minus_one() {
  unsigned l = 0x0000bf80u, h = 0xbf800000u;
  asm volatile("" : "+s"(l), "+s"(h));  // (as literals they would be taken for the inline constants of another type)
  return Minus{__builtin_bit_cast(bf16x2, l), __builtin_bit_cast(bf16x2, h)};
}
__device__ __forceinline__ void split3_nearest(const float (&x)[8], Minus m, bf16x8 (&part)[3]) {
  union { bf16x2 h[4]; bf16x8 v; } r[3];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
    for (int k = 0; k < 3; k++) {
      r[k].h[i] = __builtin_convertvector(f32x2{a, b}, bf16x2);
      if (k == 2) break;
      a = __builtin_amdgcn_fdot2_f32_bf16(r[k].h[i], m.low, a, false);
      b = __builtin_amdgcn_fdot2_f32_bf16(r[k].h[i], m.high, b, false);
    }
  }
#pragma unroll
  for (int k = 0; k < 3; k++) part[k] = r[k].v;
}

// Eight values of at most 2^15 as the sums of two float16 ones: off by at most 2^-23 of each and, where they are below 2^-1, half a
// step of float16's least numbers (2^-25).
__device__ __forceinline__ void split2_f16(const float (&x)[8], f16x8 (&part)[2]) {
  union { f16x2 h[4]; f16x8 v; } r[2];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const f16x2 h = __builtin_convertvector(f32x2{x[2 * i], x[2 * i + 1]}, f16x2);
    r[0].h[i] = h;
    r[1].h[i] = __builtin_convertvector(f32x2{__builtin_fmaf(-1.0f, (float)h[0], x[2 * i]), __builtin_fmaf(-1.0f, (float)h[1], x[2 * i + 1])}, f16x2);
  }
  part[0] = r[0].v;
  part[1] = r[1].v;
}

// Rows of an item against a part of their sequence's pages; the wavefronts of a workgroup take pages in turn.  Everything is
// computed transposed:
//   S^T [key][row] = K Q^T    (v_mfma_f32_16x16x32_bf16, K widened from e4m3, Q in three bfloat16 parts)
//   O^T [d][row]  += V^T P^T  (V^T is how pages hold values, P in three parts)
// so that a lane holds scores of one row, P is an operand of the second product as it stands, and both K and V pass from memory
// into operand registers with 16-byte loads.  That takes an order of keys in which the four that a lane gets from score tile t are
// keys 16 g + 4 t .. + 3 of the page (g = lane / 16), and an order of d in which a lane's 16 bytes serve two products.
// Bound: memory where rows are few (32 tokens behind 500 to 8500, 32 heads of 128 on 8: 56 us, 5.3 TB/s; a copy of this kernel that only
// loads takes 55; pages brought line by line and turned in LDS: 61), so three exact parts cost nothing that two would not; with all rows in use, instructions (1.3 us for a page of each
// wavefront, two workgroups to a CU).
template <int D>
__global__ __launch_bounds__(256, 2) void attend_rows(AttendParams p) {
  constexpr int STEPS = D / 32, CH = D >= 64 ? D / 64 : 1, DT = D / 16;
  constexpr int OP = D + 4;
  // the queries' parts, one fragment to a lane, later the wavefronts' results
  __shared__ __attribute__((aligned(16))) union { bf16x8 q[STEPS][3][64]; float outs[4][16 * OP]; } lds;
  __shared__ float tops[4][16], sums[4][16];
  const int group = p.group.d;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i16 = lane & 15, g = lane >> 4;
  const unsigned k_lane = (16 * (i16 >> 2) + (i16 & 3)) * D + (D >= 64 ? 16 : 8) * g, v_lane = i16 * PAGE + 16 * g;  // (of a page)
  const int head = blockIdx.y;
  const Look first = look(p, 0);
  const Minus minus = minus_one();
  Work w;
  int unit, units_end;
  if (p.wgs) {
    const int total = total_units(p, first), share = (total + p.wgs - 1) / p.wgs;
    unit = blockIdx.x * share;
    units_end = total - unit < share ? total : unit + share;
  } else {
    w = locate_work(p, first, gridDim.x - 1 - blockIdx.x, true);  // (a prompt's last items are its longest)
    unit = w.before;
    units_end = w.s.n ? w.before + w.units : unit;
  }
  for (bool first_segment = true; unit < units_end; first_segment = false) {
  // the item of the last segment has another behind it, or the next sequence's first one follows
  if (!first_segment && (w.item + 1) * 16LL < (long long)w.s.n * group) {
    w.item++;
    w.before = unit;
    w.unit = 0;
  } else if (p.wgs) {
    w = locate_work(p, first_segment ? first : look(p, 0), unit, false);
    if (w.s.n == 0) return;  // (numbers that contradict each other)
  }
  const Place s = w.s;
  // this lane's row
  const int flat = w.item * 16 + fresh(i16), token = wdh::fdiv(flat, p.group), sub = flat - token * group;
  const bool live = token < s.n;
  const int limit = live ? s.len - s.n + token : -1;  // its last key
  const int last_token = wdh::fdiv(w.item * 16 + 15, p.group), first_limit = s.len - s.n + wdh::fdiv(w.item * 16, p.group);
  const int last_key = s.len - s.n + (last_token < s.n ? last_token : s.n - 1);
  const int seg_end = w.units - w.unit < units_end - unit ? w.units : w.unit + (units_end - unit);  // in units of the item
  const int begin = 4 * w.unit, seen = last_key / PAGE + 1, end = seen < 4 * seg_end ? seen : 4 * seg_end;
  const bool alone = w.unit == 0 && seg_end == w.units;  // the whole item is this workgroup's
  const int *table = p.q.table + (long long)s.seq * p.q.max_pages;

  // A page's keys and values are asked for while the page before is worked on: keys once its scores are there, values once its
  // output is.  The number of the page after that comes a turn earlier still.
  struct Page { long long at; float ks, vs; };
  auto find = [&](int pg) {
    const int id = scalar(table, pg < end ? pg : end - 1);
    const bool known = id >= 0 && id < p.q.pages;  // (a page that is not there makes its rows NaN)
    const long long at = (long long)(known ? id : 0) * p.kv_heads + head;
    float ks = scalar(p.KS, at), vs = scalar(p.VS, at);
    // (a scale that is no number shows through the scores, which are masked, not through 0 * NaN)
    if (!known || !(ks > 0.0f && ks <= FLT_MAX) || !(vs > 0.0f && vs <= FLT_MAX)) ks = NAN, vs = 0.0f;
    return Page{at, ks, vs};
  };
  i32x4 k[4][CH], v[DT];
  auto fetch_k = [&](long long at) {
    const unsigned char *kp = p.KP + at * (PAGE * D);
#pragma unroll
    for (int t = 0; t < 4; t++) {
      if constexpr (D >= 64) {
#pragma unroll
        for (int c = 0; c < CH; c++) k[t][c] = *reinterpret_cast<const i32x4 *>(kp + (k_lane + 4 * t * D + 64 * c));
      } else {
        const i32x2 h = *reinterpret_cast<const i32x2 *>(kp + (k_lane + 4 * t * D));
        k[t][0] = i32x4{h[0], h[1], 0, 0};
      }
    }
  };
  auto fetch_v = [&](long long at) {
    const unsigned char *vp = p.VP + at * (PAGE * D);
#pragma unroll
    for (int i = 0; i < DT; i++) v[i] = *reinterpret_cast<const i32x4 *>(vp + (v_lane + 16 * i * PAGE));
  };

  int pg = begin + wave;
  Page now = find(pg), then = find(pg + 4);
  if (pg < end) {
    fetch_k(now.at);
    fetch_v(now.at);
  }
  if (wave < STEPS) {
    const float *qrow = p.Q + (long long)(s.row0 + (live ? token : 0)) * p.q_stride + (long long)(head * group + sub) * D;
    const int d0 = D >= 64 ? 64 * (wave / 2) + 16 * g + 8 * (wave & 1) : 8 * g;
    const f32x4 a = *reinterpret_cast<const f32x4 *>(qrow + d0), b = *reinterpret_cast<const f32x4 *>(qrow + d0 + 4);
    const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    bf16x8 parts[3];
    split3(x, parts);
#pragma unroll
    for (int i = 0; i < 3; i++) lds.q[wave][i][lane] = parts[i];
  }
  __syncthreads();

  f32x4 o[DT];
#pragma unroll
  for (int i = 0; i < DT; i++) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, sum = 0.0f;
  for (; pg < end; pg += 4) {
    const bool more = pg + 4 < end, whole = pg * PAGE + PAGE - 1 <= first_limit;  // whole: every row sees every key
    f32x4 sc[4];
#pragma unroll
    for (int t = 0; t < 4; t++) sc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int st = 0; st < STEPS; st++) {
      bf16x8 q[3];
#pragma unroll
      for (int i = 0; i < 3; i++) q[i] = lds.q[st][i][lane];
#pragma unroll
      for (int t = 0; t < 4; t++) {
        const bf16x8 kw = widen(k[t][st / 2][2 * (st & 1)], k[t][st / 2][2 * (st & 1) + 1]);
#pragma unroll
        for (int i = 2; i >= 0; i--) sc[t] = mfma(kw, q[i], sc[t]);
      }
    }
    if (more) fetch_k(then.at);
    // softmax: keys beyond the row's last, and whatever the page holds behind the sequence, count for nothing
    float c = p.scale * now.ks;
    float x[16], most = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; e++) x[e] = sc[e >> 2][e & 3];
    if (!whole) {
      const int ahead = limit - pg * PAGE - 16 * g;
#pragma unroll
      for (int e = 0; e < 16; e++) most = fmaxf(most, e <= ahead ? x[e] * c : -INFINITY);
    } else {
#pragma unroll
      for (int e = 0; e < 16; e++) most = fmaxf(most, x[e] * c);
    }
    most = wave_pairs_max(fmaxf(most, top));
    const float ref = most == -INFINITY ? 0.0f : most;
    if (__any(most > top)) {  // (false for most pages of a long sequence)
      const float back = __builtin_amdgcn_exp2f(top - ref);
      sum *= back;
#pragma unroll
      for (int i = 0; i < DT; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[i][e] *= back;
    }
    top = most;
    // The largest product was rounded before it became `ref`, these are not: half a step of numbers so large is a power's worth.
    if (__any(fabsf(ref) >= LARGE_SCORE)) {
#pragma unroll
      for (int e = 0; e < 16; e++) x[e] *= c;
      c = 1.0f;
    }
#pragma unroll
    for (int e = 0; e < 16; e++) x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], c, -ref));
    if (!whole) {
      const int ahead = fresh(limit) - pg * PAGE - 16 * g;
#pragma unroll
      for (int e = 0; e < 16; e++) x[e] = e <= ahead ? x[e] : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 16; e++) sum += x[e];
    // Values of keys that some row of the 16 does not see: those behind the sequence are put to 0 (0 * NaN is NaN), and a NaN among the
    // others is kept from the rows before it by hand.
    bool poison = false;
    if (!whole) {
      const int behind = s.len - pg * PAGE - 16 * fresh(g);  // how many of the lane's 16 keys are the sequence's
      int bad = 0;
#pragma unroll
      for (int i = 0; i < DT; i++)
#pragma unroll
        for (int word = 0; word < 4; word++) {
          const int n = behind - 4 * word;
          unsigned b = (unsigned)v[i][word] & (n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u);
          const unsigned nan = ((b & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
          bad |= (int)nan;
          v[i][word] = (int)(b & ~((nan >> 7) * 0xffu));
        }
      poison = __any(bad != 0);
    }
#pragma unroll
    for (int u = 0; u < 2; u++) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; e++) y[e] = x[8 * u + e] * now.vs;
      bf16x8 pr[3];
      split3_nearest(y, minus, pr);
#pragma unroll
      for (int i = 0; i < DT; i++) {
        const bf16x8 vw = widen(v[i][2 * u], v[i][2 * u + 1]);
#pragma unroll
        for (int part = 2; part >= 0; part--) o[i] = mfma(vw, pr[part], o[i]);
      }
    }
    if (poison) {  // (loops kept as loops: registers of this rare path must not weigh on the others)
      const unsigned char *vp = p.VP + now.at * (PAGE * D) + 4 * g * PAGE;
      unsigned nan = 0;
#pragma unroll 1
      for (int i = 0; i < 4 * DT; i++)
#pragma unroll 1
        for (int j = 0; j < PAGE && pg * PAGE + j <= limit; j++)
          if ((vp[(16 * (i >> 2) + (i & 3)) * PAGE + j] & 0x7f) == 0x7f) nan |= 1u << i;
#pragma unroll
      for (int i = 0; i < DT; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[i][e] = (nan >> (4 * i + e)) & 1 ? NAN : o[i][e];
    }
    if (more) fetch_v(then.at);
    now = then;
    then = find(pg + 8);
  }
  sum = wave_pairs_sum(sum);
  __syncthreads();  // the queries' place is free

  // the wavefronts' shares together
#pragma unroll
  for (int i = 0; i < DT; i++) *reinterpret_cast<f32x4 *>(&lds.outs[wave][fresh(i16) * OP + 16 * i + 4 * g]) = o[i];
  if (g == 0) {
    tops[wave][i16] = top;
    sums[wave][i16] = sum;
  }
  __syncthreads();
  for (int cell = fresh(threadIdx.x); cell < 16 * (D / 4); cell += 256) {
    const int row = cell / (D / 4), d = cell % (D / 4) * 4;
    const int flat_row = w.item * 16 + row, tk = wdh::fdiv(flat_row, p.group);
    if (tk >= s.n) continue;
    const float most = fmaxf(fmaxf(tops[0][row], tops[1][row]), fmaxf(tops[2][row], tops[3][row]));
    const float ref = most == -INFINITY ? 0.0f : most;
    float total_p = 0.0f;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float f = __builtin_amdgcn_exp2f(tops[i][row] - ref);
      const f32x4 x = *reinterpret_cast<const f32x4 *>(&lds.outs[i][row * OP + d]);
      total_p = __builtin_fmaf(f, sums[i][row], total_p);
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = __builtin_fmaf(f, x[e], y[e]);
    }
    if (alone) {
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = total_p == 0.0f ? 0.0f : y[e] / total_p;
      *reinterpret_cast<f32x4 *>(p.Y + ((long long)(s.row0 + tk) * p.heads + head * group + (flat_row - tk * group)) * D + d) = y;
    } else if (p.partial) {
      // (an item that more than one workgroup works on is the first or the last of each)
      const long long at = ((2LL * blockIdx.x + (first_segment ? 0 : 1)) * p.kv_heads + head) * 16 + row;
      *reinterpret_cast<f32x4 *>(p.partial + at * D + d) = y;
      if (d == 0) {
        p.stats[2 * at] = most;
        p.stats[2 * at + 1] = total_p;
      }
    }
  }
  unit += seg_end - w.unit;
  __syncthreads();  // the next segment's queries go where the results were
  }
}

// What several workgroups have of an item together: a workgroup to a row (and every gridDim.z-th after it), four elements and
// every (threads / (D/4))th of the shares to a lane.  Bound: latency; so results are asked for together with their tops (100000 tokens,
// 256 shares: 5.9 us, after a pass over the tops 7.2).
template <int D, int THREADS>
__global__ __launch_bounds__(THREADS) void attend_join(AttendParams p) {
  constexpr int LANES = D / 4, SIDE = THREADS / LANES;
  __shared__ __attribute__((aligned(16))) f32x4 results[SIDE][LANES];
  __shared__ float totals[SIDE], tops[SIDE];
  const Look first = look(p, 0);
  const int head = blockIdx.y, total_u = total_units(p, first), share = (total_u + p.wgs - 1) / p.wgs;
  const Work w = locate_work(p, first, blockIdx.x, true);
  if (w.s.n == 0 || share == 0) return;
  const int from_wg = w.before / share, to_wg = (w.before + w.units - 1) / share;
  if (from_wg == to_wg) return;
  const int lane = threadIdx.x % LANES, side = threadIdx.x / LANES;
  for (int row = blockIdx.z; row < 16; row += gridDim.z) {
    const int flat = w.item * 16 + row, token = wdh::fdiv(flat, p.group);
    if (token >= w.s.n) return;
    // the first workgroup has the item at its end, unless its share begins with it; the others begin with it
    auto slot = [&](int wg) {
      return ((2LL * wg + (wg == from_wg && w.before != from_wg * share ? 1 : 0)) * p.kv_heads + head) * 16 + row;
    };
    float top = -INFINITY, total = 0.0f;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = from_wg + side; i <= to_wg; i += SIDE) {
      const long long at = slot(i);
      const float its = p.stats[2 * at], most = fmaxf(top, its), ref = most == -INFINITY ? 0.0f : most;
      const float f = __builtin_amdgcn_exp2f(its - ref), back = __builtin_amdgcn_exp2f(top - ref);
      const f32x4 x = *reinterpret_cast<const f32x4 *>(p.partial + at * D + 4 * lane);
      total = __builtin_fmaf(f, p.stats[2 * at + 1], total * back);
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = __builtin_fmaf(f, x[e], y[e] * back);
      top = most;
    }
    if (lane == 0) tops[side] = top;
    __syncthreads();
    float most = tops[threadIdx.x % (SIDE < 64 ? SIDE : 64)];
    if constexpr (SIDE > 64) most = fmaxf(most, tops[64 + (threadIdx.x & 63)]);
    most = wdh::rowmath::wave_max(most);
    const float back = __builtin_amdgcn_exp2f(top - (most == -INFINITY ? 0.0f : most));
    total *= back;
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] *= back;
    results[side][lane] = y;
    if (lane == 0) totals[side] = total;
    for (int half = SIDE / 2; half; half >>= 1) {
      __syncthreads();
      if (side >= half) continue;
      total += totals[side + half];
      const f32x4 x = results[side + half][lane];
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] += x[e];
      results[side][lane] = y;
      if (lane == 0) totals[side] = total;
    }
    if (side == 0) {
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = total == 0.0f ? 0.0f : y[e] / total;
      *reinterpret_cast<f32x4 *>(p.Y + ((long long)(w.s.row0 + token) * p.heads + head * p.group.d + (flat - token * p.group.d)) * D + 4 * lane) = y;
    }
    __syncthreads();
  }
}

// ---- attention of many rows ------------------------------------------------------------------
// Prompts: items of 128 rows, 32 to a wavefront, that share the pages of their sequence through LDS (v_mfma_f32_32x32x16_f16, the
// same transposed products).  A page's 64 keys are two blocks of 32, in an order that leaves lanes of the lower half of a
// wavefront keys 0..15 and of the upper half keys 16..31 of a block in one run, as the second product wants them.  In LDS, rows
// (128 bytes of a key, 64 of a value's d) have their 16-byte pieces exchanged so that the rows a read takes lie on different banks.
constexpr int MANY = 128;
typedef float f32x16 __attribute__((ext_vector_type(16)));
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ float halves_max(float v) {
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Item number `rank` of `items`, the longest (in pages) first, so that what is left at the end are short ones (three prompts of 1200 to
// 4000 tokens, 976 items for the 512 places of the chip: 257 us, sequence by sequence 279).  Of the items of a sequence, those that see
// at least T pages are the last ones, so their number is one division, the number of all of them one sum over the lanes, and T a search
// over the pages of the longest sequence.  That takes 1 us: items of one sequence need no search, and beyond 64 sequences, which a
// wavefront looks at side by side, they come sequence by sequence.
__device__ __forceinline__ Place many_item(const AttendParams &p, int rank, int items) {
  const int group = p.group.d;
  auto count = [group](const Place &s) { return (int)(((long long)s.n * group + MANY - 1) / MANY); };
  if (p.q.seqs == 1 || p.q.seqs > 64) return locate(p.q, items - 1 - rank, count);
  const Place mine = sequence(p.q, threadIdx.x & 63);
  const int all = mine.n ? count(mine) : 0, past = mine.len - mine.n;
  // the first of the lane's items that sees `pages` pages: its last token is not before 64 (pages - 1), and tokens' rows are `group` each
  auto first = [&](int pages) {
    const long long token = (long long)PAGE * (pages - 1) - past;
    return token <= 0 ? 0 : token >= mine.n ? all : (int)(token * group / MANY);
  };
  auto total = [](int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); };
  if (rank >= total(all)) return Place{0, 0, 0, 0, 0};
  int least = 1, most = __builtin_amdgcn_readfirstlane((int)wdh::rowmath::wave_max(all ? (float)((mine.len - 1) / PAGE + 1) : 0.0f));
  while (least < most) {
    const int middle = (least + most + 1) / 2;
    if (total(all - first(middle)) > rank) least = middle;
    else most = middle - 1;
  }
  const int from = first(least), to = first(least + 1), upto = wave_scan(to - from), left = rank - total(all - to);
  const unsigned long long has = __ballot(left < upto);
  if (!has) return Place{0, 0, 0, 0, 0};  // (numbers that contradict each other)
  const int at = __ffsll(has) - 1;
  return Place{__builtin_amdgcn_readlane(mine.seq, at), __builtin_amdgcn_readlane(mine.row0, at), __builtin_amdgcn_readlane(mine.n, at),
               __builtin_amdgcn_readlane(mine.len, at), __builtin_amdgcn_readlane(from + left - (upto - (to - from)), at)};
}

// Bound: instructions.  A page takes 64 matrix ones of 32 cycles a wavefront and about as long of others (conversions of keys and values,
// powers, splitting weights), which alternate more than they overlap: matrix cores busy 41 % of the time (three prompts of 1200 to 4000
// tokens, 16 heads of 128 on 4: 243 us, 469 TFLOP/s counted once).
template <int D>
__global__ __launch_bounds__(256, 2) void attend_many(AttendParams p) {
  constexpr int QN = D / 32, DT = D / 32;           // runs of 32 elements of d in a key; blocks of 32 rows of O^T
  constexpr int KPIECES = PAGE * D / 16 / 256 > 0 ? PAGE * D / 16 / 256 : 1;  // 16-byte pieces a thread brings of a page's keys, and of its values
  constexpr int KP_ROW = D / 16;                    // pieces of a key
  __shared__ __attribute__((aligned(16))) unsigned char keys[3][PAGE * D], values[3][PAGE * D];
  __shared__ int bad[4];                            // NaN among values that some row does not see
  const int group = p.group.d;
  const int item = blockIdx.x / p.kv_heads, head = blockIdx.x - item * p.kv_heads;
  const Place s = many_item(p, item, gridDim.x / p.kv_heads);
  if (s.n == 0) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, half = lane >> 5;
  const int past = s.len - s.n;
  const int row0 = s.index * MANY, flat = row0 + 32 * wave + li, token = wdh::fdiv(flat, p.group), sub = flat - token * group;
  const bool live = token < s.n;
  const int limit = live ? past + token : -1;
  const int first_limit = past + wdh::fdiv(row0, p.group);  // of the item's first row
  const int last_token = wdh::fdiv(row0 + MANY - 1, p.group), last_key = past + (last_token < s.n ? last_token : s.n - 1);
  const int seen = last_key / PAGE + 1, begin = (int)((long long)seen * blockIdx.y / gridDim.y), end = (int)((long long)seen * (blockIdx.y + 1) / gridDim.y);
  // this wavefront's own pages end earlier
  const int wave_token = wdh::fdiv(row0 + 32 * wave, p.group), wave_last = wdh::fdiv(row0 + 32 * wave + 31, p.group), wave_first = past + wave_token;
  const int wave_end = wave_token < s.n ? (past + (wave_last < s.n ? wave_last : s.n - 1)) / PAGE + 1 : 0;
  const int *table = p.q.table + (long long)s.seq * p.q.max_pages;

  struct Page { long long at; float ks, vs; bool known; };
  auto find = [&](int pg) {
    const int id = scalar(table, pg < seen ? pg : seen - 1);
    bool known = id >= 0 && id < p.q.pages;
    const long long at = (long long)(known ? id : 0) * p.kv_heads + head;
    float ks = scalar(p.KS, at), vs = scalar(p.VS, at);
    // (a page that is not there, or has no scale, makes its rows NaN, at the end of its turn)
    known = known && ks > 0.0f && ks <= FLT_MAX && vs > 0.0f && vs <= FLT_MAX;
    if (!known) ks = FLT_MIN, vs = 0.0f;
    return Page{at, ks, vs, known};
  };
  i32x4 kr[KPIECES], vr[KPIECES];
  const bool brings = PAGE * D / 16 >= 256 || tid < PAGE * D / 16;
  auto fetch = [&](long long at) {
    const unsigned char *kp = p.KP + at * (PAGE * D), *vp = p.VP + at * (PAGE * D);
    if (brings)
#pragma unroll
      for (int i = 0; i < KPIECES; i++) {
        kr[i] = *reinterpret_cast<const i32x4 *>(kp + 16 * (tid + 256 * i));
        vr[i] = *reinterpret_cast<const i32x4 *>(vp + 16 * (tid + 256 * i));
      }
  };
  auto key_place = [](int row, int piece) { return row * D + 16 * (D == 128 ? piece ^ (row & 7) : D == 64 ? piece ^ ((row >> 1) & 3) : piece ^ ((row >> 2) & 1)); };
  auto value_place = [](int row, int piece) { return row * PAGE + 16 * (piece ^ ((row >> 1) & 3)); };
  auto keep = [&](int buf, int pg) {
    if (!brings) return;
#pragma unroll
    for (int i = 0; i < KPIECES; i++) {
      const int at = tid + 256 * i;
      *reinterpret_cast<i32x4 *>(&keys[buf][key_place(at / KP_ROW, at % KP_ROW)]) = kr[i];
      i32x4 v = vr[i];
      if (pg * PAGE + PAGE - 1 > first_limit) {  // some row does not see all of the page: see attend_rows
        const int behind = s.len - pg * PAGE - 16 * (at & 3);
        int nans = 0;
#pragma unroll
        for (int w = 0; w < 4; w++) {
          const int n = behind - 4 * w;
          const unsigned b = (unsigned)v[w] & (n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u);
          const unsigned nan = ((b & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
          nans |= (int)nan;
          v[w] = (int)(b & ~((nan >> 7) * 0xffu));
        }
        if (nans) bad[pg & 3] = 1;
      }
      *reinterpret_cast<i32x4 *>(&values[buf][value_place(at >> 2, at & 3)]) = v;
    }
  };

  // Queries in two float16 parts, 8 elements of the lane's row for each instruction.  A row is brought to [2^14, 2^15) by a power of two:
  // what two parts leave out is at most 2^-23 of an element, or 2^-39 of the row's largest one (half a step of float16's least numbers).
  f16x8 q[2 * QN][2];
  float row_scale;
  {
    const float *qrow = p.Q + (long long)(s.row0 + (live ? token : 0)) * p.q_stride + (long long)(head * group + sub) * D;
    float x[2 * QN][8], most = 0.0f;
#pragma unroll
    for (int i = 0; i < 2 * QN; i++) {
      const int d0 = 32 * (i / 2) + 16 * half + 8 * (i & 1);
      const f32x4 a = *reinterpret_cast<const f32x4 *>(qrow + d0), b = *reinterpret_cast<const f32x4 *>(qrow + d0 + 4);
#pragma unroll
      for (int e = 0; e < 4; e++) x[i][e] = a[e] * p.scale, x[i][4 + e] = b[e] * p.scale;
#pragma unroll
      for (int e = 0; e < 8; e++) most = fmaxf(most, finite_abs(x[i][e]));
    }
    const int exponent = (int)(__float_as_uint(halves_max(most)) >> 23);  // (of zeros and of subnormal rows: 0)
    const int up = 141 - exponent < 126 ? 141 - exponent : 126;           // bias 127: the row times 2^up has exponent 14
    const float to = __uint_as_float((unsigned)(127 + up) << 23);
    row_scale = __uint_as_float((unsigned)(127 - up) << 23);
#pragma unroll
    for (int i = 0; i < 2 * QN; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float y = x[i][e] * to;
        q[i][0][e] = (_Float16)y;
        q[i][1][e] = (_Float16)(y - (float)q[i][0][e]);
      }
  }
  f32x16 o[DT];
#pragma unroll
  for (int i = 0; i < DT; i++)
#pragma unroll
    for (int e = 0; e < 16; e++) o[i][e] = 0.0f;
  float top = -FLT_MAX, sum = 0.0f;
  // Weights go in two float16 parts as well, times their page's scale and in such units that the row's largest product of both so far
  // is in (2^13, 2^15]: what is left out of a key's share is at most 2^-23 of it and 2^-38 of the largest share, whatever the scales of pages
  // that count for less.  `top` is the exponent that weights are relative to, the least whole number no score (as a power of two) is
  // above, and the output is held in units of 2^(top + gap - 15): both change by whole powers of two, which round nothing.
  // Keys of half a page none of whose weights reaches 2^-112 of the row's largest so far count for nothing.
  float gap = -1e30f;

  // Half a page of scores: 32 keys, of which a lane has keys 16 half + r of block t.
  auto scores = [&](int buf, int t) {
    f32x16 sc;
#pragma unroll
    for (int e = 0; e < 16; e++) sc[e] = 0.0f;
    const int row = 32 * t + 16 * ((li >> 2) & 1) + 4 * (li >> 3) + (li & 3);
#pragma unroll
    for (int i = 0; i < QN; i++) {
      const i32x4 x = *reinterpret_cast<const i32x4 *>(&keys[buf][key_place(row, 2 * i + half)]);
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const f16x8 kw = widen_f16(x[2 * j], x[2 * j + 1]);
#pragma unroll
        for (int part = 1; part >= 0; part--) sc = mfma32(kw, q[2 * i + j][part], sc);
      }
    }
    return sc;
  };
  // What a row does not see counts for nothing; the largest of the rest.
  auto mask = [&](f32x16 &sc, int pg, int t) {
    if (pg * PAGE + PAGE - 1 <= wave_first) return;
    const int ahead = limit - pg * PAGE - 32 * t - 16 * half;
#pragma unroll
    for (int r = 0; r < 16; r++) sc[r] = r <= ahead ? sc[r] : -INFINITY;
  };
  auto largest = [&](const f32x16 &sc) {
    float most = sc[0];
#pragma unroll
    for (int r = 1; r < 16; r++) most = fmaxf(most, sc[r]);
    return halves_max(most);
  };

  if (tid < 4) bad[tid] = 0;
  Page now = find(begin), then = find(begin + 1), after = find(begin + 2), later = after;
  __syncthreads();
  if (begin < end) {
    fetch(now.at);
    keep(0, begin);
    if (begin + 1 < end) fetch(then.at);
  }
  __syncthreads();
  // The scores of the next half page are multiplied while the present one's weights are worked out, in one stretch of
  // instructions without branches: a wavefront then keeps the matrix cores busy by itself.  So keys have to be in LDS half a
  // page early, and a page's place is free again a page and a half later: three places, one barrier a page.
  f32x16 sc = scores(0, 0);
  mask(sc, begin, 0);
  float most = largest(sc);
  int buf = 0;
  for (int pg = begin; pg < end; pg++) {
    const int next_buf = buf == 2 ? 0 : buf + 1;
    const bool active = pg < wave_end;
    const float vs_exponent = uniform((float)__builtin_amdgcn_frexp_expf(now.vs)), vs_mantissa = uniform(__builtin_amdgcn_frexp_mantf(now.vs));  // (0 of 0)
#pragma unroll
    for (int t = 0; t < 2; t++) {
      if (active) {
        float c = fmaxf(now.ks * row_scale, FLT_MIN);  // (never 0: -inf * 0 is NaN; scores that need less are all 0 to the softmax)
        const float mine = ceilf(most * c), up = fmaxf(mine, top), below = mine - up;  // (none seen: mine = -inf)
        const bool counts = below >= -112.0f;
        const float had = gap + (top - up), has = counts ? fmaxf(had, below + vs_exponent) : had;
        if (__any(has > had || up > top)) {  // (false for most pages of a long sequence)
          sum *= __builtin_amdgcn_exp2f(top - up);
          const float back = __builtin_amdgcn_exp2f(had - has);
#pragma unroll
          for (int i = 0; i < DT; i++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[i][e] *= back;
        }
        top = up;
        gap = has;
        if (__any(fabsf(up) >= LARGE_SCORE && up != -FLT_MAX)) {  // (see attend_rows)
#pragma unroll
          for (int r = 0; r < 16; r++) sc[r] *= c;
          c = 1.0f;
        }
        const float weight = counts ? vs_mantissa * __builtin_amdgcn_exp2f(vs_exponent - has + 15.0f) : 0.0f;
        const f32x16 next = scores(t == 0 ? buf : next_buf, 1 - t);
#pragma unroll
        for (int r = 0; r < 16; r++) sc[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], c, -up));
#pragma unroll
        for (int r = 0; r < 16; r++) sum += sc[r];
#pragma unroll
        for (int u = 0; u < 2; u++) {
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; e++) y[e] = sc[8 * u + e] * weight;
          f16x8 pr[2];
          split2_f16(y, pr);
#pragma unroll
          for (int i = 0; i < DT; i++) {
            const i32x2 v = *reinterpret_cast<const i32x2 *>(&values[buf][value_place(32 * i + li, 2 * t + half) + 8 * u]);
            const f16x8 vw = widen_f16(v[0], v[1]);
#pragma unroll
            for (int part = 1; part >= 0; part--) o[i] = mfma32(vw, pr[part], o[i]);
          }
        }
        sc = next;
      }
      if (t == 0) {
        if (pg + 1 < end) keep(next_buf, pg + 1);
        __syncthreads();
        if (tid == 0) bad[(pg + 3) & 3] = 0;  // (of the page before, which nobody reads any more; written again three pages on)
        if (pg + 2 < end) fetch(after.at);
        later = find(pg + 3);
        mask(sc, pg, 1);
      } else {
        mask(sc, pg + 1, 0);
      }
      if (active) most = largest(sc);
    }
    if (active && bad[pg & 3]) {
      const unsigned char *vp = p.VP + now.at * (PAGE * D);
#pragma unroll
      for (int i = 0; i < DT; i++) {
        unsigned nan = 0;
#pragma unroll 1
        for (int e = 0; e < 16; e++)
#pragma unroll 1
          for (int j = 0; j < PAGE && pg * PAGE + j <= limit; j++)
            if ((vp[(32 * i + 8 * (e >> 2) + 4 * half + (e & 3)) * PAGE + j] & 0x7f) == 0x7f) nan |= 1u << e;
#pragma unroll
        for (int e = 0; e < 16; e++) o[i][e] = (nan >> e) & 1 ? NAN : o[i][e];
      }
    }
    if (active && !now.known && limit >= pg * PAGE) sum = NAN;
    now = then;
    then = after;
    after = later;
    buf = next_buf;
  }
  {
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
    sum = __uint_as_float(b[0]) + __uint_as_float(b[1]);
  }
  const int exponent = (int)fmaxf(gap - 15.0f, -1000.0f);  // (a row that has seen nothing: 0 times whatever)
  if (!live) return;
  // lane: row li of the wavefront's 32; registers 4 a .. + 3 of block i are elements 32 i + 8 a + 4 half .. + 3
  if (gridDim.y == 1) {
    float *y = p.Y + ((long long)(s.row0 + token) * p.heads + head * group + sub) * D;
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
      for (int a = 0; a < 4; a++) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = sum == 0.0f ? 0.0f : __builtin_amdgcn_ldexpf(o[i][4 * a + e] / sum, exponent);
        *reinterpret_cast<f32x4 *>(y + 32 * i + 8 * a + 4 * half) = v;
      }
  } else {
    const long long at = (((long long)item * p.kv_heads + head) * gridDim.y + blockIdx.y) * MANY + 32 * wave + li;
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
      for (int a = 0; a < 4; a++) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = __builtin_amdgcn_ldexpf(o[i][4 * a + e], exponent);
        *reinterpret_cast<f32x4 *>(p.partial + at * D + 32 * i + 8 * a + 4 * half) = v;
      }
    if (half == 0) {
      p.stats[2 * at] = top;
      p.stats[2 * at + 1] = sum;
    }
  }
}

// The parts of an item's pages together: a lane to four elements of a row, few parts.  Bound: memory.
template <int D>
__global__ __launch_bounds__(256) void attend_many_join(AttendParams p, int parts) {
  constexpr int LANES = D / 4, ROWS = 256 / LANES;
  const int group = p.group.d, head = blockIdx.y;
  const Place s = many_item(p, blockIdx.x, gridDim.x);
  const int row = blockIdx.z * ROWS + threadIdx.x / LANES, lane = threadIdx.x % LANES;
  const int flat = s.index * MANY + row, token = wdh::fdiv(flat, p.group);
  if (token >= s.n) return;
  const long long at = ((long long)blockIdx.x * p.kv_heads + head) * parts * MANY + row;
  float top = -INFINITY;
  for (int i = 0; i < parts; i++) top = fmaxf(top, p.stats[2 * (at + (long long)i * MANY)]);
  const float ref = top == -INFINITY ? 0.0f : top;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  float total = 0.0f;
  for (int i = 0; i < parts; i++) {
    const long long one = at + (long long)i * MANY;
    const float f = __builtin_amdgcn_exp2f(p.stats[2 * one] - ref);
    const f32x4 x = *reinterpret_cast<const f32x4 *>(p.partial + one * D + 4 * lane);
    total = __builtin_fmaf(f, p.stats[2 * one + 1], total);
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = __builtin_fmaf(f, x[e], y[e]);
  }
#pragma unroll
  for (int e = 0; e < 4; e++) y[e] = total == 0.0f ? 0.0f : y[e] / total;
  *reinterpret_cast<f32x4 *>(p.Y + ((long long)(s.row0 + token) * p.heads + head * group + (flat - token * group)) * D + 4 * lane) = y;
}

template <int D>
int launch_many(const AttendParams &p, long long items, int parts) {
  hipStream_t st = wdh::stream();
  hipLaunchKernelGGL((attend_many<D>), dim3((unsigned)(items * p.kv_heads), (unsigned)parts), dim3(256), 0, st, p);
  WDH_LAUNCH_CHECK();
  if (parts > 1) {
    hipLaunchKernelGGL((attend_many_join<D>), dim3((unsigned)items, (unsigned)p.kv_heads, MANY * D / 1024), dim3(256), 0, st, p, parts);
    WDH_LAUNCH_CHECK();
  }
  return WDH_OK;
}

template <int D>
int launch_attend(const AttendParams &p, long long items) {
  hipStream_t st = wdh::stream();
  hipLaunchKernelGGL((attend_rows<D>), dim3((unsigned)(p.wgs ? p.wgs : items), (unsigned)p.kv_heads), dim3(256), 0, st, p);
  WDH_LAUNCH_CHECK();
  if (p.partial) {
    // (an item of hundreds of shares is a wide workgroup's work, one of a few shares a small one's)
    const long long rows = ((long long)p.q.tokens * p.group.d + p.q.seqs - 1) / p.q.seqs;  // (of a sequence, on average)
    const dim3 grid((unsigned)items, (unsigned)p.kv_heads, (unsigned)(rows < 16 ? rows : 16));
    if (p.wgs >= 32 * items) hipLaunchKernelGGL((attend_join<D, 1024>), grid, dim3(1024), 0, st, p);
    else hipLaunchKernelGGL((attend_join<D, 256>), grid, dim3(256), 0, st, p);
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
  if (seqs == 0 || tokens == 0 || max_pages == 0) return WDH_OK;
  if (pages == 0) return fail(WDH_EINVAL, "%s: a cache without pages", who);
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
  p.heads = heads; p.kv_heads = kv_heads; p.group = wdh::make_fastdiv(heads / kv_heads);
  p.scale = alpha * 1.44269504088896341f;
  // items of 16 or 128 rows: a sequence of n tokens has ceil(n group / rows); whichever bound of their number is lower
  auto items_of_rows = [&](int rows) {
    const long long loose = (long long)tokens * p.group.d / rows + seqs, tight = (long long)tokens * ((p.group.d + rows - 1) / rows);
    return loose < tight ? loose : tight;
  };
  // Items of 128 rows read a page once for eight times the rows, but need more of them to fill the chip: they are taken where sequences
  // fill half an item on average, and the call has 80 rows of 128 elements for each CU (us, 16 / 128 rows an item; 32 heads of 128 on 8,
  // behind nothing: 3 x 256 tokens 29 / 22, 1 x 2000 140 / 94, 1 x 512 26 / 31; 16 heads of 64 on 4: 3 x 1000 42 / 38, 1 x 2000 42 / 59).
  const long long rows = (long long)tokens * p.group.d;
  const bool many = rows >= 64LL * seqs && (long long)tokens * width >= 80LL * 128 * wdh::compute_units();
  const long long items = items_of_rows(many ? MANY : 16);
  if (items > 0xffffffLL / 2) return fail(WDH_EINVAL, "%s: too many rows", who);
  p.partial = p.stats = nullptr;
  wdh_buf work = 0;
  auto workspace = [&](size_t rows) {
    work = wdh_alloc(rows * (d + 2) * 4);
    if (!work) return false;
    size_t have_bytes;
    p.partial = (float *)wdh::resolve(work, &have_bytes);
    p.stats = p.partial + rows * d;
    return true;
  };
  int rc;
  if (many) {
    // Pages are cut into parts where there are fewer items than the chip holds at a time: into as many as make one and a half times its
    // places, items being of different lengths (us, so / for its places: 8 heads on 2, prompts of 624, 1247 and 1870 tokens 69 / 80, 700 tokens
    // behind 8000, 32 on 8, 232 / 254; 848 on average, 8 on 1, 68 / 64).
    if (items * kv_heads > 0xffffffLL / 2) return fail(WDH_EINVAL, "%s: too many rows", who);
    const long long have = items * kv_heads, wanted = 2LL * wdh::compute_units();
    long long parts = have >= wanted ? 1 : 3 * wanted / (2 * have);
    if (parts > (max_pages + 3) / 4) parts = (max_pages + 3) / 4;
    if (parts > 1 && !workspace((size_t)have * parts * MANY)) return WDH_ENOMEM;
    rc = d == 32 ? launch_many<32>(p, items, (int)parts) : d == 64 ? launch_many<64>(p, items, (int)parts) : launch_many<128>(p, items, (int)parts);
  } else {
    // as many workgroups as the chip holds at a time, or as there can be units
    const long long units = items * ((max_pages + 3) / 4), resident = 2LL * wdh::compute_units() / kv_heads;
    if (units > MOST_UNITS) return fail(WDH_EINVAL, "%s: too many rows of tables so wide", who);
    p.wgs = (int)(units < resident ? units : resident > 0 ? resident : 1);
    // Shares end together whatever the sequences' lengths, but cost their join, and the first rows of a prompt, which see few pages, leave theirs
    // half empty.  A workgroup to an item, the last ones first, is faster where there are many items for the pages that one can have: for
    // prompts 14 to a unit, for single tokens, whose lengths nothing is known about, 64 (us, shared / so: one prompt of 1024, 32 heads
    // of 128 on 8, behind nothing 97 / 57, 256 behind 2000 47 / 38, 128 behind 8000 71 / 99; single tokens of 128 sequences of 100 to 4000 137
    // / 117, of 64 of which one has 8000 and the others 500 31 / 92).
    const long long most_units = (max_pages + 3) / 4;
    if (most_units <= 2 || most_units * (rows >= 16LL * seqs ? 14 : 64) <= items * kv_heads) p.wgs = 0;
    if (p.wgs > 1 && !workspace((size_t)p.wgs * 2 * kv_heads * 16)) return WDH_ENOMEM;  // (items of one unit are never cut)
    rc = d == 32 ? launch_attend<32>(p, items) : d == 64 ? launch_attend<64>(p, items) : launch_attend<128>(p, items);
  }
  if (work) (void)wdh_free(work);
  return rc;
}
