// What comes after a forward pass over drafted tokens: which of them the target's probabilities accept, and keeping those in the cache.
//
// The reference has no such operators.
//
// Verification.  A sequence's rows are a tree, parents first; p_c is the target's distribution behind row c, and its children's tokens were
// drawn one by one and independently from q_c.  At node c the first child is accepted with probability min(1, p/q) of its token, and
// after each rejection p gives way to its normed part above q.  Since max(max(a, 0) - b, 0) = max(a - b, 0) for b >= 0, what is left of p after k
// rejections is
//   r_k(x) = max(p(x) - t_k q(x), 0),  s_k = sum_x r_k(x),  t_0 = 0, s_0 = 1, t_{k+1} = t_k + s_k:
// one number for all of a row's history, so that a test needs two elements (u s_k q(x) < r_k(x)), and a rejection one pass over two rows.
// Drafts that were chosen, not drawn (no q), are accepted with their share of what is left, u s < p(x); a rejected one is taken out: s -= p(x).
// Where no child is accepted a token is drawn from what is left, by its cumulative sum.  A token so found has the target's distribution.
// All of it in 64 bits, sums in a fixed order: the token drawn goes by where a sum passes a number.
#include "common.h"
#include "fp8.h"
#include "kv_cache.h"

namespace {

using namespace wdh::fp8;
using namespace wdh::kv;
using wdh::fail;

constexpr int MOST_ROWS = WDH_DRAFT_ROWS;

struct VerifyParams {
  const float *P, *Q, *U;
  const int *tokens, *parents, *starts;
  int *next, *count, *path;
  int seqs, rows, vocab;
};

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
// Sums over the lanes up to and with each.
__device__ __forceinline__ double wave_scan_d(double v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double below = __shfl_up(v, off, 64);
    if (lane >= off) v += below;
  }
  return v;
}

// What is left of an element.  Negative probabilities and NaN count as 0.
__device__ __forceinline__ double left_of(float p, float q, double t) { return fmax(__builtin_fma(-t, (double)fmaxf(q, 0.0f), (double)fmaxf(p, 0.0f)), 0.0); }
// What is left of a row: of elements idx .. idx+3, 0 behind `end`.
struct Rest {
  const float *p, *q;      // (q null: nothing but the taken-out tokens is missing)
  double t;
  const int *out;          // tokens that are taken out
  int outs, vocab;
};
__device__ __forceinline__ void rest4(const Rest &r, int idx, int end, double (&v)[4]) {
  const f32x4 p = load4(r.p, idx, end);
  const f32x4 q = r.q ? load4(r.q, idx, end) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = left_of(p[e], q[e], r.t);
  for (int i = 0; i < r.outs; i++) {
    const int at = r.out[i] - idx;
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (at == e) v[e] = 0.0;
  }
}
// Sum of elements lo .. hi-1, by a wavefront: AT_ONCE turns of it are on their way together.  Behind the row's end its last four elements are loaded once more;
// what is not counted is put to 0 before it becomes a number of 64 bits, whose instructions are what bounds this on one compute unit.
constexpr int AT_ONCE = 4;
template <bool DRAFT>
__device__ __forceinline__ double wave_rest(const Rest &r, int lo, int hi) {
  const int lane = threadIdx.x & 63;
  double sum = 0.0;
  for (int turn = lo; turn < hi; turn += 256 * AT_ONCE) {
    f32x4 p[AT_ONCE], q[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; i++) {
      const int idx = turn + 256 * i + 4 * lane, at = idx < r.vocab - 4 ? idx : r.vocab - 4;
      p[i] = *reinterpret_cast<const f32x4_any *>(r.p + at);
      if constexpr (DRAFT) q[i] = *reinterpret_cast<const f32x4_any *>(r.q + at);
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; i++) {
      const int from = turn + 256 * i, idx = from + 4 * lane, at = idx < r.vocab - 4 ? idx : r.vocab - 4;
      if (from >= hi) break;
      if (from + 256 > hi)
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (at + e < idx || at + e >= hi) {
            p[i][e] = 0.0f;
            if constexpr (DRAFT) q[i][e] = 0.0f;
          }
      if constexpr (!DRAFT)
        for (int j = 0; j < r.outs; j++) {
          const int gone = r.out[j];
          if (gone >= from && gone < from + 256)
#pragma unroll
            for (int e = 0; e < 4; e++) p[i][e] = at + e == gone ? 0.0f : p[i][e];
        }
#pragma unroll
      for (int e = 0; e < 4; e++) sum += DRAFT ? left_of(p[i][e], q[i][e], r.t) : (double)fmaxf(p[i][e], 0.0f);
    }
  }
  return wave_sum_d(sum);
}
__device__ __forceinline__ double wave_rest(const Rest &r, int lo, int hi) {
  if (r.vocab >= 4) return r.q ? wave_rest<true>(r, lo, hi) : wave_rest<false>(r, lo, hi);
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  if (lo == 0 && hi > 0 && (threadIdx.x & 63) == 0) rest4(r, 0, hi, v);
  return wave_sum_d((v[0] + v[1]) + (v[2] + v[3]));
}

constexpr int WAVES = 16;
__device__ __forceinline__ int wave_of() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
// The sixteenth of lo .. hi-1 that is `i`'s, in whole turns of a wavefront.
__device__ __forceinline__ int part_begin(int lo, int hi, int i) {
  const int each = ((hi - lo + WAVES - 1) / WAVES + 255) / 256 * 256;
  const long long at = lo + (long long)each * i;
  return at < hi ? (int)at : hi;
}
// The sums of all sixteen; their sum in order.
__device__ __forceinline__ double parts_of(const Rest &r, int lo, int hi, double *sums) {
  const int wave = wave_of();
  const double mine = wave_rest(r, part_begin(lo, hi, wave), part_begin(lo, hi, wave + 1));
  __syncthreads();  // (who still reads the sums before)
  if ((threadIdx.x & 63) == 0) sums[wave] = mine;
  __syncthreads();
  double total = 0.0;
#pragma unroll
  for (int i = 0; i < WAVES; i++) total += sums[i];
  return total;
}
// The part in which the running sum, `base` before the first, passes `target`, else the last that is not empty; base moves on.
__device__ __forceinline__ int part_of(const double *sums, double target, double &base) {
  int last = 0;
  double before = base, last_before = base;
  for (int i = 0; i < WAVES; i++) {
    if (sums[i] > 0.0) last = i, last_before = before;
    if (before + sums[i] > target) break;
    before += sums[i];
  }
  base = last_before;
  return last;
}

// Long rows are summed by sixteen workgroups, in a launch of its own, which more sequences take longer to be through with.  One launch / two (us): a tree of
// 33 chosen drafts over 16000 tokens 9.6 / 10.0, over 32000 11.3 / 10.1, over 50001 13.5 / 10.5, over 128000 22 / 11.5; 32 sequences of 5 drawn in a row over 32000
// 10.1 / 12.2, over 50001 13.6 / 12.9, over 128000 20 / 14.4; 64 sequences of 8 drawn over 50001 20 / 26; trees of 33 drawn, 8 of them, over 50001 23 / 24
// (later sums of a tree are one workgroup's either way).
bool in_two(int seqs, int vocab) { return vocab >= 32768 + 512LL * seqs; }

// Where a walk has come to: the node, how many drafts were accepted, the last child that was rejected (-1: none), and t.
struct Walk {
  int node, taken, tried;
  double t;
};
// What the first of two launches leaves for the second, for each sequence.
struct Halfway {
  Walk walk;
  double sums[WAVES][WAVES];  // of the parts' parts
};

// ALL: a workgroup to a sequence.  FIRST and SECOND: sixteen, which all take the walk to the first sum that it needs (or to its end) and have a part
// of that sum each, and one that goes on from there.  Bound: latency (of a row that one workgroup reads, its rate).
enum Stage { ALL, FIRST, SECOND };
template <int STAGE>
__global__ __launch_bounds__(64 * WAVES, STAGE == FIRST ? 8 : 4) void verify_drafts(VerifyParams a, Halfway *halfway) {
  __shared__ int parent[MOST_ROWS], token[MOST_ROWS], path[MOST_ROWS], out[MOST_ROWS];
  __shared__ float px[MOST_ROWS], qx[MOST_ROWS], us[MOST_ROWS];
  __shared__ double sums[WAVES], sums_of[WAVES][WAVES];
  __shared__ int found, outs_found;
  const int seq = blockIdx.x, row0 = a.starts[seq], tid = threadIdx.x, lane = tid & 63;
  const long long rows = (long long)a.starts[seq + 1] - row0;
  if (row0 < 0 || rows <= 0 || rows > MOST_ROWS || row0 + rows > a.rows) return;
  const int n = (int)rows;
  for (int i = tid; i < MOST_ROWS; i += 64 * WAVES) {
    const int up = i < n ? a.parents[row0 + i] : -1;
    parent[i] = i > 0 && up >= 0 && up < i ? up : -1;
    token[i] = i < n ? a.tokens[row0 + i] : 0;
    us[i] = i < n ? a.U[row0 + i] : 0.0f;
  }
  auto fetch = [&]() {  // the elements that tests need
    for (int i = tid; i < n; i += 64 * WAVES) {
      const int up = parent[i], x = token[i];
      const bool real = up >= 0 && x >= 0 && x < a.vocab;
      const long long at = ((long long)row0 + (real ? up : 0)) * a.vocab + (real ? x : 0);
      px[i] = real ? a.P[at] : 0.0f;
      qx[i] = real && a.Q ? a.Q[at] : 0.0f;
    }
    __syncthreads();
  };
  Walk walk = {0, 0, -1, 0.0};
  double mass = 1.0;
  int outs = 0;
  bool summed = false, fine = false;  // mass is the sum of `sums`; and those are sums of `sums_of`
  if constexpr (STAGE == SECOND) {
    const Halfway &from = halfway[seq];
    walk = from.walk;
    if (tid < WAVES * WAVES) sums_of[tid / WAVES][tid % WAVES] = from.sums[tid / WAVES][tid % WAVES];
    if (tid == 0) outs_found = 0;
    __syncthreads();
    if (tid < WAVES) {
      double sum = 0.0;
#pragma unroll
      for (int i = 0; i < WAVES; i++) sum += sums_of[tid][i];
      sums[tid] = sum;
    }
    if (!a.Q && walk.tried >= 0)  // chosen drafts: the walk is at its end, the node's children have all been taken out
      for (int i = tid; i < n; i += 64 * WAVES)
        if (parent[i] == walk.node) out[atomicAdd(&outs_found, 1)] = token[i];
    __syncthreads();
    outs = outs_found;
    mass = 0.0;
#pragma unroll
    for (int i = 0; i < WAVES; i++) mass += sums[i];
    summed = fine = true;
  } else {
    if (tid == 0) path[0] = 0;
    fetch();
  }
  const int known = walk.taken;
  auto rest_of = [&]() {
    const long long row = ((long long)row0 + walk.node) * a.vocab;
    return Rest{a.P + row, a.Q && walk.tried >= 0 ? a.Q + row : nullptr, walk.t, out, outs, a.vocab};
  };
  // All wavefronts take the same walk.
  bool fetched = STAGE != SECOND;
  for (;;) {
    int child = -1;
    if (STAGE != SECOND || a.Q)
      for (int base = (walk.tried < 0 ? walk.node : walk.tried) / 64 * 64; base < n && child < 0; base += 64) {
        const unsigned long long children = __ballot(parent[base + lane] == walk.node && base + lane > walk.tried);
        if (children) child = base + __ffsll(children) - 1;
      }
    if (child < 0) break;
    if (!fetched) {
      fetch();
      fetched = true;
    }
    const double u = us[child], likely = a.Q ? (double)fmaxf(qx[child], 0.0f) : 1.0;
    double left = left_of(px[child], qx[child], walk.t);  // (t is 0 where drafts were chosen)
    if (!a.Q) {
      for (int i = 0; i < outs; i++)
        if (out[i] == token[child]) left = 0.0;
    }
    if (u * mass * likely < left) {
      walk = Walk{child, walk.taken + 1, -1, 0.0};
      if (tid == 0) path[walk.taken] = child;
      mass = 1.0;
      outs = 0;
      summed = fine = false;
      continue;
    }
    walk.tried = child;
    if (a.Q) {
      walk.t += mass;
      if constexpr (STAGE == FIRST) break;
      mass = parts_of(rest_of(), 0, a.vocab, sums);
      summed = true;
      fine = false;
    } else {
      mass -= left;
      __syncthreads();  // (who still reads the list)
      if (tid == 0) out[outs] = token[child];
      outs++;
      __syncthreads();
    }
  }
  Rest rest = rest_of();
  if constexpr (STAGE == FIRST) {
    const int lo = part_begin(0, a.vocab, blockIdx.y), hi = part_begin(0, a.vocab, blockIdx.y + 1);
    const double mine = wave_rest(rest, part_begin(lo, hi, wave_of()), part_begin(lo, hi, wave_of() + 1));
    if (lane == 0) halfway[seq].sums[blockIdx.y][wave_of()] = mine;
    if (blockIdx.y) return;
    if (tid == 0) halfway[seq].walk = walk;
  } else {
    // a token from what is left of the last row, or, if that is nothing, from the row
    double total = summed ? mass : parts_of(rest, 0, a.vocab, sums);
    if (!(total > 0.0) && (rest.outs || rest.q)) {
      rest.outs = 0;
      rest.q = nullptr;
      rest.t = 0.0;
      total = parts_of(rest, 0, a.vocab, sums);
      fine = false;
    }
    if (tid == 0) found = -1;
    __syncthreads();
    if (total > 0.0 && total <= DBL_MAX) {
      const double target = (double)us[0] * total;
      double base = 0.0;
      int part = part_of(sums, target, base);
      const int lo = part_begin(0, a.vocab, part), hi = part_begin(0, a.vocab, part + 1);
      if (!fine) parts_of(rest, lo, hi, sums);
      part = part_of(fine ? sums_of[part] : sums, target, base);
      const int begin = part_begin(lo, hi, part), end = part_begin(lo, hi, part + 1);
      if (tid < 64) {
        int at = -1;
        bool done = false;
        for (int turn = begin; turn < end && !done; turn += 256) {
          const int idx = turn + 4 * lane;
          double v[4] = {0.0, 0.0, 0.0, 0.0};
          if (idx < end) rest4(rest, idx, end, v);
          const double mine = (v[0] + v[1]) + (v[2] + v[3]), upto = wave_scan_d(mine);
          double before = base + (upto - mine);
          int first = -1, last = -1;
#pragma unroll
          for (int e = 0; e < 4; e++) {
            before += v[e];
            if (v[e] > 0.0) {
              last = idx + e;
              if (first < 0 && before > target) first = idx + e;
            }
          }
          const unsigned long long passed = __ballot(first >= 0), some = __ballot(last >= 0);
          if (passed) {
            at = __shfl(first, __ffsll(passed) - 1, 64);
            done = true;
          } else if (some) {
            at = __shfl(last, 63 - __clzll(some), 64);  // (the last so far: what is found if rounding leaves the sum short)
          }
          base += __shfl(upto, 63, 64);
        }
        if (lane == 0) found = at;
      }
    }
  }
  __syncthreads();
  for (int i = tid + (STAGE == SECOND ? known + 1 : 0); i < (STAGE == SECOND ? walk.taken + 1 : n); i += 64 * WAVES) a.path[row0 + i] = i <= walk.taken ? path[i] : -1;
  if (STAGE != FIRST && tid == 0) {
    a.next[seq] = found;
    a.count[seq] = walk.taken;
  }
}

// ---- keeping accepted tokens -------------------------------------------------------------------
struct KeepParams {
  Sequences q;
  const int *path, *count;
  unsigned char *KP, *VP;
  float *KS, *VS;
  int heads;
};

// What takes elements of a page of scale `scale` to one of scale 1 / inv.  The new scale holds 1/448 of each element, the least of which is 2^-9: more than 2^18 is
// for zeros alone, which an infinite ratio (scales of 2^28 and 2^-100) would make NaN.  A scale that is no number leaves none.
__device__ __forceinline__ float to_scale(float scale, float inv) {
  const float ratio = scale * inv;
  return ratio > 0x1p18f && scale <= FLT_MAX ? 0x1p18f : ratio;
}

// Tokens of a path go behind each other: slot past + i takes what slot past + path[i] holds, which is never before it.  So a workgroup has a
// sequence's pages of one head, keys (blockIdx.z 0) or values, and goes over them in order; what a page takes is in registers before any of
// it is written, and what later pages take lies behind.  Bound: latency, of five rounds of loads after each other (numbers of rows; path; tables; scales and
// elements; and words to be kept).  The ways to two pages are found at a time, and threads go to the words that are written: with a way and all words for each page
// 16 sequences of 32 rows took 10.8 us, 200 of 9 rows 14.2; so 5.6 and 7.1.
template <int D>
__global__ __launch_bounds__(256) void cache_keep(KeepParams p) {
  constexpr int NP = PAGE * D / 4 / 256, PPT = D / 4;
  __shared__ float part[2][4], scales_of[2][PAGE], had_of[2];
  __shared__ long long froms[2][PAGE], at_of[2];   // where a slot's token comes from, and the page's own cell
  __shared__ int moves_of[2];
  const int given = p.count[blockIdx.x];
  const Place s = sequence(p.q, blockIdx.x);
  if (s.n == 0) return;
  const int kept = given < 0 ? 0 : given < s.n - 1 ? given + 1 : s.n, past = s.len - s.n;
  if (kept == 0) return;
  const bool values = blockIdx.z;
  const int head = blockIdx.y, t = threadIdx.x;
  unsigned char *pages = values ? p.VP : p.KP;
  float *scales = values ? p.VS : p.KS;
  const int *table = p.q.table + (long long)s.seq * p.q.max_pages;
  const int end = (past + kept - 1) / PAGE + 1;
  for (int two = past / PAGE; two < end; two += 2) {
    __syncthreads();  // (the pages before are done with the lists)
    float scale = 0.0f;
    if (t < 2 * PAGE) {
      const int page = two + t / PAGE, i = page * PAGE + t % PAGE - past, id = page < end ? table[page] : -1;
      const int j = page < end && i >= 0 && i < kept ? p.path[s.row0 + i] : -1;
      const bool known = id >= 0 && id < p.q.pages;
      const long long at = known ? (long long)id * p.heads + head : 0;
      long long cell = at;
      int slot = t % PAGE;
      bool moves = false;
      if (known && j > i && j < s.n) {
        const int there = table[(past + j) / PAGE];
        if (there >= 0 && there < p.q.pages) {
          cell = (long long)there * p.heads + head;
          slot = (past + j) % PAGE;
          moves = true;
        }
      }
      scale = scales[cell];
      froms[t / PAGE][t % PAGE] = cell * (PAGE * D) + (values ? slot : slot * D);
      const unsigned long long any = __ballot(moves);
      if (t % PAGE == 0) {
        moves_of[t / PAGE] = any != 0;
        at_of[t / PAGE] = at;
        had_of[t / PAGE] = scales[at];
      }
      scales_of[t / PAGE][t % PAGE] = scale;
    }
    __syncthreads();
#pragma unroll 1
    for (int which = 0; which < 2; which++) {
      if (!moves_of[which]) continue;
      const int page0 = (two + which) * PAGE, first = past > page0 ? past - page0 : 0, last = past + kept - page0 < PAGE ? past + kept - page0 : PAGE;
      const long long *from = froms[which];
      const float *scale_of = scales_of[which];
      unsigned char *page = pages + at_of[which] * (PAGE * D);
      // the words that are written: keys: all of the new tokens'; values: those of each element that a new token is in
      const int word0 = first / 4, each = (last + 3) / 4 - word0, words = values ? D * each : (last - first) * PPT;
      const int inverse = (65536 + each - 1) / each;  // (exact for numbers up to 2048)
      auto word_of = [&](int k) { return values ? (k * inverse >> 16) * (PAGE / 4) + word0 + k - (k * inverse >> 16) * each : first * PPT + k; };
      f32x4 v[NP];
      int old[NP];
      float amax = 0.0f;
#pragma unroll
      for (int i = 0; i < NP; i++) {
        if (256 * i >= words) break;
        const int k = t + 256 * i, w = word_of(k), s0 = values ? w % (PAGE / 4) * 4 : w / PPT;
        v[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        old[i] = 0;
        if (k >= words) continue;
        int q = 0;
        if (!values) {
          q = *reinterpret_cast<const int *>(pages + from[s0] + w % PPT * 4);
        } else {
          old[i] = reinterpret_cast<const int *>(page)[w];
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (s0 + e >= first && s0 + e < last) q |= (int)pages[from[s0 + e] + w / (PAGE / 4) * PAGE] << (8 * e);
        }
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(q, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(q, true);
        v[i] = f32x4{a[0], a[1], b[0], b[1]};
#pragma unroll
        for (int e = 0; e < 4; e++) {  // (a value that was rounded up may stand for more than fp32 holds; fmaxf passes NaN by)
          const float x = fabsf(v[i][e] * scale_of[values ? s0 + e : s0]);
          amax = fmaxf(amax, x > FLT_MAX ? FLT_MAX : x);
        }
      }
      const float had = had_of[which];
      amax = wdh::rowmath::wave_max(amax);
      if ((t & 63) == 0) part[which][t >> 6] = amax;
      __syncthreads();
      const float *pt = part[which], c = fmaxf(had, page_scale(fmaxf(fmaxf(pt[0], pt[1]), fmaxf(pt[2], pt[3])))), inv = 1.0f / c, factor = had / c;
      const bool grown = c != had;
#pragma unroll
      for (int i = 0; i < NP; i++) {
        if (256 * i >= words) break;
        const int k = t + 256 * i, w = word_of(k), s0 = values ? w % (PAGE / 4) * 4 : w / PPT;
        if (k >= words) continue;
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = v[i][e] * to_scale(scale_of[values ? s0 + e : s0], inv);
        reinterpret_cast<int *>(page)[w] = values ? merge4(old[i], pack4(y, 1.0f), first - s0, last - s0, grown, factor) : pack4(y, 1.0f);
      }
      if (grown) {  // the tokens before
        for (int w = t; w < PAGE * D / 4; w += 256) {
          if (values ? w % (PAGE / 4) >= word0 : w >= first * PPT) continue;
          int *to = reinterpret_cast<int *>(page) + w;
          *to = rescale4(*to, factor);
        }
        if (t == 0) scales[at_of[which]] = c;
      }
    }
  }
}

}  // namespace

extern "C" int wdh_verify_drafts(wdh_buf hP, wdh_buf hDraft, wdh_buf hTokens, wdh_buf hParents, wdh_buf hUniform, wdh_buf hStarts, wdh_buf hNext,
                                 wdh_buf hCount, wdh_buf hPath, int seqs, int tokens, int vocab) {
  WDH_REQUIRE_INIT();
  WDH_REQUIRE_COMPUTE_LANE();
  if (seqs < 0 || tokens < 0 || vocab < 0) return fail(WDH_EINVAL, "wdh_verify_drafts: negative extent");
  if (tokens > (1 << 24) || seqs > (1 << 20)) return fail(WDH_EINVAL, "wdh_verify_drafts: too many tokens or sequences");
  if (vocab > (1 << 30)) return fail(WDH_EINVAL, "wdh_verify_drafts: a vocabulary of %d tokens (at most %d)", vocab, 1 << 30);
  if (seqs == 0 || tokens == 0) return WDH_OK;
  if (vocab == 0) return fail(WDH_EINVAL, "wdh_verify_drafts: an empty vocabulary");
  void *pp, *pd = nullptr, *pt, *pa, *pu, *ps, *pn, *pc, *ph;
  const size_t rows = (size_t)tokens * 4;
  if (!wdh::operand(hP, rows * vocab, "wdh_verify_drafts: P", &pp)) return WDH_EINVAL;
  if (hDraft && !wdh::operand(hDraft, rows * vocab, "wdh_verify_drafts: Draft", &pd)) return WDH_EINVAL;
  if (!wdh::operand(hTokens, rows, "wdh_verify_drafts: Tokens", &pt) || !wdh::operand(hParents, rows, "wdh_verify_drafts: Parents", &pa) ||
      !wdh::operand(hUniform, rows, "wdh_verify_drafts: Uniform", &pu) ||
      !wdh::operand(hStarts, ((size_t)seqs + 1) * 4, "wdh_verify_drafts: Starts", &ps) ||
      !wdh::operand(hNext, (size_t)seqs * 4, "wdh_verify_drafts: Next", &pn) ||
      !wdh::operand(hCount, (size_t)seqs * 4, "wdh_verify_drafts: Count", &pc) || !wdh::operand(hPath, rows, "wdh_verify_drafts: Path", &ph))
    return WDH_EINVAL;
  const wdh_buf out[3] = {hNext, hCount, hPath}, in[6] = {hP, hDraft, hTokens, hParents, hUniform, hStarts};
  for (int i = 0; i < 3; i++) {
    for (wdh_buf h : in)
      if (out[i] == h) return fail(WDH_EINVAL, "wdh_verify_drafts: a result aliases an input");
    for (int j = 0; j < i; j++)
      if (out[i] == out[j]) return fail(WDH_EINVAL, "wdh_verify_drafts: two results share a buffer");
  }
  const VerifyParams p = {(const float *)pp, (const float *)pd, (const float *)pu, (const int *)pt, (const int *)pa, (const int *)ps,
                          (int *)pn, (int *)pc, (int *)ph, seqs, tokens, vocab};
  hipStream_t st = wdh::stream();
  if (!in_two(seqs, vocab)) {
    hipLaunchKernelGGL(verify_drafts<ALL>, dim3((unsigned)seqs), dim3(64 * WAVES), 0, st, p, nullptr);
  } else {
    const wdh_buf work = wdh_alloc((size_t)seqs * sizeof(Halfway));
    if (!work) return WDH_ENOMEM;
    size_t have;
    Halfway *halfway = (Halfway *)wdh::resolve(work, &have);
    hipLaunchKernelGGL(verify_drafts<FIRST>, dim3((unsigned)seqs, WAVES), dim3(64 * WAVES), 0, st, p, halfway);
    hipLaunchKernelGGL(verify_drafts<SECOND>, dim3((unsigned)seqs), dim3(64 * WAVES), 0, st, p, halfway);
    (void)wdh_free(work);
  }
  WDH_LAUNCH_CHECK();
  return WDH_OK;
}

extern "C" int wdh_cache_keep(wdh_buf hKP, wdh_buf hKS, wdh_buf hVP, wdh_buf hVS, wdh_buf hTable, wdh_buf hLens, wdh_buf hStarts, wdh_buf hPath,
                              wdh_buf hCount, int seqs, int tokens, int kv_heads, int d, int pages, int max_pages) {
  WDH_REQUIRE_INIT();
  WDH_REQUIRE_COMPUTE_LANE();
  const char *who = "wdh_cache_keep";
  if (int rc = check_cache(who, seqs, tokens, kv_heads, d, pages, max_pages)) return rc;
  if (seqs == 0 || tokens == 0 || pages == 0 || max_pages == 0) return WDH_OK;
  KeepParams p;
  void *kp, *ks, *vp, *vs, *path, *count;
  if (int rc = cache_operands(who, hKP, hKS, hVP, hVS, hTable, hLens, hStarts, seqs, kv_heads, d, pages, max_pages, &kp, &ks, &vp, &vs, &p.q)) return rc;
  if (!wdh::operand(hPath, (size_t)tokens * 4, "wdh_cache_keep: Path", &path) || !wdh::operand(hCount, (size_t)seqs * 4, "wdh_cache_keep: Count", &count))
    return WDH_EINVAL;
  const wdh_buf out[4] = {hKP, hKS, hVP, hVS}, in[5] = {hTable, hLens, hStarts, hPath, hCount};
  for (int i = 0; i < 4; i++) {
    for (wdh_buf h : in)
      if (out[i] == h) return fail(WDH_EINVAL, "%s: a part of the cache aliases an input", who);
    for (int j = 0; j < i; j++)
      if (out[i] == out[j]) return fail(WDH_EINVAL, "%s: two parts of the cache share a buffer", who);
  }
  p.q.tokens = tokens;
  p.path = (const int *)path;
  p.count = (const int *)count;
  p.KP = (unsigned char *)kp; p.KS = (float *)ks; p.VP = (unsigned char *)vp; p.VS = (float *)vs;
  p.heads = kv_heads;
  const dim3 grid((unsigned)seqs, (unsigned)kv_heads, 2);
  if (d == 32) hipLaunchKernelGGL((cache_keep<32>), grid, dim3(256), 0, wdh::stream(), p);
  else if (d == 64) hipLaunchKernelGGL((cache_keep<64>), grid, dim3(256), 0, wdh::stream(), p);
  else hipLaunchKernelGGL((cache_keep<128>), grid, dim3(256), 0, wdh::stream(), p);
  WDH_LAUNCH_CHECK();
  return WDH_OK;
}
