// What the cache's operators share: which tokens of a call belong to which sequence, the 8-bit forms of pages, and what the
// entry points ask of their arguments.  Layouts are told in kv_cache.hip.
#pragma once
#include <stdio.h>

#include "common.h"
#include "fastdiv.h"
#include "fp8.h"

namespace wdh {
namespace kv {

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
  v = dpp_add<rowmath::DPP_BCAST15, 0xa>(v);
  return dpp_add<rowmath::DPP_BCAST31, 0xc>(v);
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

// ---- attention -------------------------------------------------------------------------------
struct AttendParams {
  Sequences q;
  const float *Q;
  long long q_stride;
  const unsigned char *KP, *VP;
  const float *KS, *VS;
  float *Y;
  int heads, kv_heads;
  FastDiv group;  // queries that share a head of the cache
  float scale;     // alpha * log2(e): powers are taken of two
  int wgs;         // workgroups for each head of the cache (0: one for each item, which works on the whole of it)
  float *partial;  // results [workgroup][2][kv head][ROWS][D] of items that more than one workgroup works on (null: there are none),
  float *stats;    // and their tops and sums [workgroup][2][kv head][ROWS][2]
  const int *mask; // trees: [tokens][words], bit j: the row sees row j of its sequence
  int words;
};

// Work of attention: items of ROWS rows (a row is a token and one of the queries that share a head of the cache), each as many units
// of UNIT pages (one for each wavefront of a workgroup, or for some that share it) as its sequence has.  The units of all items stand in a row, and every
// workgroup takes `share` neighbouring ones: all end at the same time, whatever the sequences' lengths.
constexpr int MOST_UNITS = 1 << 30;
struct Work {
  Place s;
  int item, unit, units;  // the item, the unit of it that was asked for, and how many it has
  int before;             // units in front of the item
  int ordinal;            // items in front of it (where that is asked for)
  int share, total;
};
template <int ROWS>
__device__ __forceinline__ int items_of(const Place &s, int group) { return s.n ? (int)(((long long)s.n * group + ROWS - 1) / ROWS) : 0; }
template <int UNIT>
__device__ __forceinline__ int units_of(const Place &s) { return (s.len + UNIT * PAGE - 1) / (UNIT * PAGE); }
// 64 sequences side by side, a lane to each; upto: units of these up to and with the lane's.
struct Look {
  Place mine;
  int items, units, upto;
};
template <int ROWS, int UNIT>
__device__ __forceinline__ Look look(const AttendParams &p, int round) {
  Look l;
  l.mine = sequence(p.q, 64 * round + fresh(threadIdx.x & 63));
  l.items = items_of<ROWS>(l.mine, p.group.d);
  l.units = units_of<UNIT>(l.mine);
  l.upto = wave_scan(l.items * l.units);
  return l;
}
template <int ROWS, int UNIT>
__device__ __forceinline__ int total_units(const AttendParams &p, const Look &first) {
  int total = __builtin_amdgcn_readlane(first.upto, 63);
  for (int i = 1; i < (p.q.seqs + 63) / 64; i++) total = add_sat(total, __builtin_amdgcn_readlane(look<ROWS, UNIT>(p, i).upto, 63));
  return total <= MOST_UNITS ? total : 0;  // (more than the host allows: numbers that contradict each other)
}
// The item that holds unit number `index` of all (or, by_item, item number `index`); s.n = 0 behind the last.
template <int ROWS, int UNIT, bool ORDINAL = false>
__device__ __forceinline__ Work locate_work(const AttendParams &p, const Look &first, int index, bool by_item) {
  Work w;
  int before = 0, before_items = 0;
  Look l = first;
  for (int i = 0; i < (p.q.seqs + 63) / 64; i++) {
    if (i) l = look<ROWS, UNIT>(p, i);
    const int upto = add_sat(before, l.upto), upto_items = by_item || ORDINAL ? add_sat(before_items, wave_scan(l.items)) : 0;
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
      if constexpr (ORDINAL) w.ordinal = __builtin_amdgcn_readlane(upto_items - l.items, at) + w.item;
      return w;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
    before_items = __builtin_amdgcn_readlane(upto_items, 63);
  }
  w.s = Place{0, 0, 0, 0, 0};
  return w;
}

// All items of a call (where there are units at all).
template <int ROWS, int UNIT>
__device__ __forceinline__ int total_items(const AttendParams &p, const Look &first) {
  int total = __builtin_amdgcn_readlane(wave_scan(first.items), 63);
  for (int i = 1; i < (p.q.seqs + 63) / 64; i++) total = add_sat(total, __builtin_amdgcn_readlane(wave_scan(look<ROWS, UNIT>(p, i).items), 63));
  return total;
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

// Trees: which of 32 tokens from `at` on (counted from the sequence's first row; those before it are seen by all) a row sees, as bits.
__device__ __forceinline__ unsigned tree_bits(const int *row, int words, int at) {
  const int w = at >> 5;
  auto word = [&](int i) { return i < 0 ? ~0u : i < words ? (unsigned)row[i] : 0u; };
  return __builtin_amdgcn_alignbit(word(w + 1), word(w), at & 31);
}

// ---- bytes of pages ----------------------------------------------------------------------------
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

// What append and attention ask of their sequences and of the cache.
inline int check_cache(const char *who, int seqs, int tokens, int kv_heads, int d, int pages, int max_pages) {
  if (seqs < 0 || tokens < 0 || kv_heads < 0 || pages < 0 || max_pages < 0) return fail(WDH_EINVAL, "%s: negative extent", who);
  if (d != 32 && d != 64 && d != 128) return fail(WDH_EINVAL, "%s: head dimension %d (32, 64 and 128 are built)", who, d);
  if (kv_heads == 0 || kv_heads > 65535) return fail(WDH_EINVAL, "%s: %d heads of the cache (1 to 65535)", who, kv_heads);
  if (max_pages > (1 << 24)) return fail(WDH_EINVAL, "%s: tables of %d pages (at most %d)", who, max_pages, 1 << 24);
  if (tokens > (1 << 24) || seqs > (1 << 20)) return fail(WDH_EINVAL, "%s: too many tokens or sequences", who);
  return WDH_OK;
}
inline int cache_operands(const char *who, wdh_buf hKP, wdh_buf hKS, wdh_buf hVP, wdh_buf hVS, wdh_buf hT, wdh_buf hL, wdh_buf hS, int seqs, int kv_heads,
                   int d, int pages, int max_pages, void **kp, void **ks, void **vp, void **vs, Sequences *q) {
  const size_t cells = (size_t)pages * kv_heads;
  char what[64];
  auto get = [&](wdh_buf h, size_t need, const char *name, void **out) {
    snprintf(what, sizeof(what), "%s: %s", who, name);
    return operand(h, need, what, out);
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
inline int check_rows(const char *who, const char *name, int64_t offset, int64_t stride, int64_t width) {
  if (offset < 0 || stride < width || offset > (1LL << 46) || stride > (1LL << 22))
    return fail(WDH_EINVAL, "%s: %s rows of %lld elements from %lld on, %lld apart", who, name, (long long)width, (long long)offset, (long long)stride);
  if (offset % 4 || stride % 4) return fail(WDH_EINVAL, "%s: offset and stride of %s must be multiples of 4 elements", who, name);
  return WDH_OK;
}

// Attention of trees (kv_tree.hip): rows of p.mask.
int attend_trees(const char *who, AttendParams &p, int d);

}  // namespace kv
}  // namespace wdh
