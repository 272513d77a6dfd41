// What the cache's operators share: which tokens of a call belong to which sequence, the 8-bit forms of pages, and what the
// entry points ask of their arguments.  Layouts are told in kv_cache.hip.
#pragma once
#include <stdio.h>

#include "common.h"
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

}  // namespace kv
}  // namespace wdh
