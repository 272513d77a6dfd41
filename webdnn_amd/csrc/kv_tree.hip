// Attention over the cache for rows that see all of their sequence's earlier tokens and, of its newest ones, those that their masks name: trees of
// drafted tokens.  Nothing but the last pages of a sequence needs a mask, and all rows of a sequence read all of its pages.
//
// The reference has no such operator (its attention: see kv_cache.hip).
//
// As in kv_cache.hip everything is computed transposed, 32 rows to a wavefront:
//   S^T [key][row] = K Q^T,  O^T [d][row] += V^T P^T   (v_mfma_f32_32x32x16_f16)
// keys and values widened from e4m3, queries and weights in two float16 parts.
#include "common.h"
#include "fastdiv.h"
#include "kv_cache.h"

#include <type_traits>

namespace {

using namespace wdh::fp8;
using namespace wdh::kv;
using wdh::fail;

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(127 + e) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ int exponent_of(float x) { return (int)((__float_as_uint(x) >> 23) & 0xff) - 127; }  // (of 0 and subnormal numbers: -127)

// x less a float16 number, one half of a pair: one instruction, where conversion and subtraction are two (and a dot product with -1 would take
// the matrix cores' place).
__device__ __forceinline__ float less_low(float x, f16x2 h) {
  float r;
  asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
  return r;
}
__device__ __forceinline__ float less_high(float x, f16x2 h) {
  float r;
  asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
  return r;
}
// Eight values of at most 2^15 as the sums of two float16 ones.
__device__ __forceinline__ void split2(const float *x, f16x8 (&part)[2]) {
  union { f16x2 h[4]; f16x8 v; } r[2];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const f16x2 h = __builtin_convertvector(f32x2{x[2 * i], x[2 * i + 1]}, f16x2);
    r[0].h[i] = h;
    r[1].h[i] = __builtin_convertvector(f32x2{less_low(x[2 * i], h), less_high(x[2 * i + 1], h)}, f16x2);
  }
  part[0] = r[0].v;
  part[1] = r[1].v;
}
// A number that is new in a branch: what is computed from it is computed there, and not before the branch in case it is taken.
__device__ __forceinline__ float rarely(float v) {
  asm volatile("" : "+v"(v));
  return v;
}
// Waits until no more than N of the wavefront's loads are on their way (those into LDS are not waited for otherwise).
template <int N>
__device__ __forceinline__ void loads_left() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
__device__ __forceinline__ float both_halves(float v, float (*op)(float, float)) {
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// The largest of the LANES neighbouring lanes that share a row, in all of them.
template <int CTRL>
__device__ __forceinline__ unsigned max_with(unsigned v) {
  const unsigned other = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
  return v > other ? v : other;
}
template <int LANES>
__device__ __forceinline__ unsigned lanes_max(unsigned v) {
  using namespace wdh::rowmath;
  v = max_with<DPP_HALF_MIRROR>(max_with<DPP_XOR2>(max_with<DPP_XOR1>(v)));
  if constexpr (LANES > 8) v = max_with<DPP_MIRROR>(v);
  if constexpr (LANES > 16) {
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = b[0] > b[1] ? b[0] : b[1];
  }
  return v;
}
__device__ __forceinline__ float max2(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float add2(float a, float b) { return a + b; }

// Sixteen values of a row of which the first `behind` are the sequence's: the others are put to 0 (0 * NaN is NaN), and so is a NaN among them, which is
// kept from the rows that do not see it by hand.
__device__ __forceinline__ i32x4 seen_values(i32x4 v, int behind, bool &bad) {
#pragma unroll
  for (int word = 0; word < 4; word++) {
    const int n = behind - 4 * word;
    const unsigned b = (unsigned)v[word] & (n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u);
    const unsigned nan = ((b & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    bad = bad || nan;
    v[word] = (int)(b & ~((nan >> 7) * 0xffu));
  }
  return v;
}

// A row's weights go into the second product times their pages' scales (a power of two and a rest between 1/2 and 1), as 2^(score + ref + shift) rest with
// shift = lift + the power's exponent.  lift brings the largest share so far to 2^7 .. 2^9 when the row first sees something, and again only when a larger one might
// pass 2^15, beyond which float16 parts end.  What two parts leave out of a share is at most 2^-23 of it or 2^-25, 2^-32 of the row's largest, whatever the scales of
// pages that count for less.  The sum of weights is in units of 2^-ref, in which the first page's largest weight is 1/2 to 1, and none passes 2^MOST_WEIGHT: shares and
// weights may be far apart (values of 2^110 behind weights of 2^-200, beside values of 2^-100).  Where a page's shares are so far below others' that its weights
// would leave fp32 on the way to their sum, LEAST_SHIFT keeps them from that, with which they are still nothing to float16.
constexpr float AIM = 9.0f, MOST = 15.0f, MOST_WEIGHT = 50.0f, LEAST_SHIFT = -80.0f;
static_assert(MOST_WEIGHT + LEAST_SHIFT < -25.0f, "half of float16's least number");
constexpr float LARGE_SCORE = 0x1p20f;  // from here on fp32 numbers are too far apart for ref and shift to be added first

// What the join has to know of an item.
struct Joint {
  int row0, n, item;         // the sequence's rows, and which of its items
  int from, count, first;    // workgroups that have a part of it (1: it is done); which of the first one's two places holds its part
};

// RB blocks of 32 rows to an item, WAVES / RB wavefronts to a block, which take the item's pages in turn.
// Bound: matrix instructions, which take 50 % of the time, and what they leave half of theirs to, conversions and the softmax: 64 rows of 16 heads on 2
// of 128 take 89 us for each 102400 tokens behind them, 1210 TFLOP/s with the second parts (a large library product has 1240 in ten calls in a row, 1417 in
// long runs).  Pages' scales in the weights' exponents take as long as they did in the widening of values.  Beside its pages an item
// costs a workgroup 13 us, 3.5 of them a page's instructions on their first way into the cache.  The pages' order in a workgroup is fixed, no sum
// depends on another workgroup's time.
template <int D, int RB, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 8 / WAVES) void attend_tree(AttendParams p, Joint *joints, int most_joints) {
  constexpr int STEPS = D / 16, VT = D / 32, S = WAVES / RB, ROWS = 32 * RB, OP = D + 4;
  // Pages pass through LDS, from where all blocks of rows read them: in operand order a page's rows are 16-byte pieces of 32 lines to a load, and where every
  // wavefront asked for them itself the L1 cache looked up lines 85 % of the time.  (That took as long, but left no registers to load ahead.)
  // Four blocks have two places for a page, and a barrier a page; two have one place, and two barriers; a block's own wavefront needs none.
  constexpr int BUFS = RB == 4 ? 2 : 1;
  constexpr int CHUNKS = PAGE * D / 1024;          // what a wavefront brings of a page at a time
  struct Input { f16x8 q[RB][STEPS][2][64]; unsigned char keys[S][BUFS][PAGE * D], values[S][BUFS][PAGE * D]; };
  __shared__ __attribute__((aligned(16))) union { Input in; float outs[WAVES][32 * OP]; } lds;
  __shared__ float tops[WAVES][32], sums[WAVES][32];
  __shared__ int bad_values[S][2];                 // the stream's page holds NaN that some row does not see; of this turn and the next
  const int group = p.group.d;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, half = lane >> 5;
  const int rb = wave % RB, stream = wave / RB;
  const int head = blockIdx.y;
  // Rows of a key tile are tokens in an order that leaves lanes of the lower half of a wavefront scores of tokens 0 .. 15 of a half page, and of the upper
  // half 16 .. 31: eight neighbours for each instruction of the second product.
  const int key_row = 16 * ((li >> 2) & 1) + 4 * (li >> 3) + (li & 3);
  const Look first = look<ROWS, S>(p, 0);
  Work w;
  int unit, units_end, share = 1;
  if (p.wgs) {
    const int total = total_units<ROWS, S>(p, first);
    share = (total + p.wgs - 1) / p.wgs;
    unit = blockIdx.x * share;
    units_end = total - unit < share ? total : unit + share;
    if (joints && blockIdx.x == 0)  // places that no item has
      for (int i = (total ? total_items<ROWS, S>(p, first) : 0) + threadIdx.x; i < most_joints; i += 64 * WAVES) joints[i * p.kv_heads + head].count = 1;
  } else {
    w = locate_work<ROWS, S>(p, first, blockIdx.x, true);
    unit = w.before;
    units_end = w.s.n ? w.before + w.units : unit;
  }
  for (bool first_segment = true; unit < units_end; first_segment = false) {
  // the item of the last segment has another behind it, or the next sequence's first one follows
  if (!first_segment && (w.item + 1) * (long long)ROWS < (long long)w.s.n * group) {
    w.item++;
    w.ordinal++;
    w.before = unit;
    w.unit = 0;
  } else if (p.wgs) {
    w = locate_work<ROWS, S, true>(p, first_segment ? first : look<ROWS, S>(p, 0), unit, false);
    if (w.s.n == 0) return;  // (numbers that contradict each other)
  }
  const Place s = w.s;
  const int past = s.len - s.n, row0 = w.item * ROWS + 32 * rb, flat = row0 + li, token = wdh::fdiv(flat, p.group), sub = flat - token * group;
  const bool live = token < s.n;
  const int seg_end = w.units - w.unit < units_end - unit ? w.units : w.unit + (units_end - unit);  // in units of the item
  const int seen = (s.len - 1) / PAGE + 1, begin = S * w.unit, end = seen < S * seg_end ? seen : S * seg_end;
  const bool alone = w.unit == 0 && seg_end == w.units;  // the whole item is this workgroup's
  const int *table = p.q.table + (long long)s.seq * p.q.max_pages;
  // which of the 16 keys from `key` on the lane's row sees
  auto sees = [&](int key) {
    const int behind = s.len - key;
    const unsigned bits = tree_bits(p.mask + (long long)(s.row0 + (live ? token : 0)) * p.words, p.words, key - past);
    return live ? bits & (behind >= 16 ? 0xffffu : behind > 0 ? (1u << behind) - 1u : 0u) : 0u;
  };

  // The wavefront's pages, 64 at a time, a lane to each: numbers and scales come in two rounds of loads, and none is waited for in between (scalar loads
  // would be, with every read of LDS: both are counted alike, and scalar ones return in any order).
  int held_id = 0, taken = 0;
  float held_ks = 0.0f, held_vs = 0.0f;
  struct Page { long long at; float ks, vs; };
  auto number_of = [&](int i) {  // (behind the last: the last once more, which is loaded and not used: no branch about registers)
    const int at = begin + stream + S * i;
    return table[at < end ? at : end - 1];
  };
  auto cell_of = [&](int i) { return (long long)__builtin_amdgcn_readlane(held_id, i) * p.kv_heads + head; };
  auto hold = [&](int id) {
    const bool known = id >= 0 && id < p.q.pages;
    held_id = known ? id : 0;
    held_ks = p.KS[(long long)held_id * p.kv_heads + head];
    held_vs = p.VS[(long long)held_id * p.kv_heads + head];
    if (!known) held_vs = 0.0f;
  };
  // (a page that is not there, or has no scale, makes its rows NaN, at the end of its turn)
  auto check_held = [&]() {
    if (!(held_ks > 0.0f && held_ks <= FLT_MAX) || !(held_vs > 0.0f && held_vs <= FLT_MAX)) held_ks = FLT_MIN, held_vs = 0.0f;
  };
  auto next_page = [&]() {
    const int which = taken++ & 63;
    if (which == 0 && taken > 1) {
      hold(number_of(taken - 1 + lane));
      check_held();
    }
    return Page{cell_of(which), __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(held_ks), which)),
              __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(held_vs), which))};
  };
  // The way to the first page: its number, and the queries at the same time, a row to D / 4 lanes.
  const int at_lane = fresh(lane), first_id = number_of(at_lane);
  constexpr int LANES = D / 4, Q_ROWS = 64 / LANES, Q_LOADS = 32 / S / Q_ROWS;
  f32x4 x[Q_LOADS];
#pragma unroll
  for (int i = 0; i < Q_LOADS; i++) {
    const int flat_q = row0 + stream * (32 / S) + Q_ROWS * i + at_lane / LANES, t = wdh::fdiv(flat_q, p.group), tk = t < s.n ? t : 0;
    x[i] = *reinterpret_cast<const f32x4 *>(p.Q + (long long)(s.row0 + tk) * p.q_stride + (long long)(head * group + flat_q - t * group) * D + 4 * (at_lane % LANES));
  }
  hold(first_id);
  // (lanes that write a row's elements would meet in one bank, 16 at a time: they write them two at a time; 16 sequences of 32 nodes 109 -> 106 us)
  auto query_place = [](int block, int half, int row) { return 32 * half + (row ^ (2 * block + half)); };
  // A row's 16-byte pieces change places in LDS, so that rows of a tile lie on different banks.  Loads go there directly, a lane's 16 bytes behind the
  // lane's before it: so it is the pieces' addresses in memory that change.
  auto key_piece = [](int row, int piece) { return D == 128 ? piece ^ (row & 7) : D == 64 ? piece ^ ((row >> 1) & 3) : piece ^ ((row >> 2) & 1); };
  auto value_piece = [](int row, int piece) { return piece ^ ((row >> 1) & 3); };
  const int k_from = lane / (D / 16) * D + 16 * key_piece(lane / (D / 16), lane % (D / 16)), v_from = lane / 4 * PAGE + 16 * value_piece(lane / 4, lane % 4);
  auto bring = [&](const unsigned char *from, unsigned char *to) {
#pragma unroll
    for (int i = 0; i < (CHUNKS + RB - 1) / RB; i++)
      if (CHUNKS >= RB || rb < CHUNKS)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(from + 1024 * (rb + RB * i)),
                                         (__attribute__((address_space(3))) void *)(to + 1024 * (rb + RB * i)), 16, 0, 0);
  };
  auto bring_keys = [&](long long at, int buf) { bring(p.KP + at * (PAGE * D) + k_from, lds.in.keys[stream][buf]); };
  auto bring_values = [&](long long at, int buf) { bring(p.VP + at * (PAGE * D) + v_from, lds.in.values[stream][buf]); };
  int pg = begin + stream;
  bring_keys(cell_of(0), 0);
  bring_values(cell_of(0), 0);
  if (lane < 2) bad_values[stream][lane] = 0;

  // Queries times alpha log2(e) in two float16 parts, a row brought to [2^14, 2^15) by a power of two: what two parts leave out is at most 2^-23 of an
  // element, or 2^-39 of the row's largest one.
#pragma unroll
  for (int i = 0; i < Q_LOADS; i++) {
    unsigned most = 0;  // (numbers without their signs, as integers)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      x[i][e] *= p.scale;
      most = max(most, __float_as_uint(fabsf(x[i][e])));
    }
    const int exponent = exponent_of(__uint_as_float(lanes_max<LANES>(most)));  // (of zeros and of subnormal rows: -127)
    const int up = 14 - exponent < 126 ? 14 - exponent : 126;
    const float times = exponent < 128 ? power_of_two(up) : NAN;  // (a row that is not finite has no scores that are)
    const int r = stream * (32 / S) + Q_ROWS * i + at_lane / LANES, d = 4 * (at_lane % LANES);
    union { f16x2 h[2]; f16x4 v; } parts[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const f32x2 y = {x[i][2 * e] * times, x[i][2 * e + 1] * times};
      parts[0].h[e] = __builtin_convertvector(y, f16x2);
      parts[1].h[e] = __builtin_convertvector(f32x2{less_low(y[0], parts[0].h[e]), less_high(y[1], parts[0].h[e])}, f16x2);
    }
#pragma unroll
    for (int part = 0; part < 2; part++)
      reinterpret_cast<f16x4 *>(&lds.in.q[rb][2 * (d / 32) + (d >> 3 & 1)][part][query_place(d / 32, d >> 4 & 1, r)])[d >> 2 & 1] = parts[part].v;
    if (d == 0) tops[rb][r] = power_of_two(-up);
  }
  check_held();
  Page now = next_page(), then = next_page();
  loads_left<0>();
  __syncthreads();
  const float row_scale = tops[rb][li];

  f32x16 o[VT];
#pragma unroll
  for (int i = 0; i < VT; i++)
#pragma unroll
    for (int e = 0; e < 16; e++) o[i][e] = 0.0f;
  float sum = 0.0f, ref = 0.0f, lift = 0.0f;  // o is in units of 2^-(ref + lift), the sum of 2^-ref
  bool has_seen = false, far = false;                  // far: some row's ref is a LARGE_SCORE
  // Between wavefronts that share pages; a block's own wavefront has to wait for its own reads of LDS alone.
  auto sync = [] {
    if constexpr (RB > 1) __syncthreads();
    else asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
  };
  const bool has_rows = wdh::fdiv(row0, p.group) < s.n;
  const int whole_end = past / PAGE < end ? past / PAGE : end;  // pages before this one hold no token of the tree
  const int turns = (end - begin + S - 1) / S, whole = whole_end > begin ? (whole_end - begin) / S : 0;
  auto sees_in = [&](int page, int at) { return page < end ? sees(page * PAGE + at) : 0u; };
  unsigned bits_of[2] = {0u, 0u};
  if (whole < turns)
#pragma unroll
    for (int t = 0; t < 2; t++) bits_of[t] = sees_in(pg + S * whole, 32 * t + 16 * half);
  // A page of all wavefronts; `tail`: it may hold tokens which not every row sees; `rows`: the block has rows (one without takes part in loads and barriers).
  int n = 0;
  auto turn = [&](auto tail, auto rows) {
    constexpr bool TAIL = decltype(tail)::value, HAS_ROWS = decltype(rows)::value;
    const int buf = BUFS == 2 ? n & 1 : 0;
    unsigned char *keys = lds.in.keys[stream][buf], *values = lds.in.values[stream][buf];
    // (the next page's bits are asked for a turn ahead)
    const unsigned bits_now[2] = {bits_of[0], bits_of[1]};
    if constexpr (TAIL)
#pragma unroll
      for (int t = 0; t < 2; t++) bits_of[t] = sees_in(pg + S, 32 * t + 16 * half);
    // The values' scale: a power of two and what is left, between 1/2 and 1; both go into the weights' exponents, and out of their sum.
    const bool known = now.vs > 0.0f, even = (__float_as_uint(now.ks) & 0x7fffffu) == 0;
    const float ve = known ? (float)__builtin_amdgcn_frexp_expf(now.vs) : 0.0f, rest = known ? __builtin_amdgcn_frexp_mantf(now.vs) : 0.5f;
    auto key_at = [&](int t, int j) {
      const int row = 32 * t + key_row;
      return *reinterpret_cast<const i32x4 *>(keys + row * D + 16 * key_piece(row, 2 * j + half));
    };
    if constexpr (BUFS == 2) {
      bring_keys(then.at, buf ^ 1);
      bring_values(then.at, buf ^ 1);
    }
    f32x16 sc[2];
    float c, shift;
    // (Where what is there has to be brought to other units, rarely, the page is begun again, so that the accumulators change in its products, in one
    // place beside them, and not in a branch on the way; once, after which its own shares and weights are in range.)
    bool again = false;
    for (; HAS_ROWS;) {
      // (the queries' place hidden from the compiler, which would hold them all in registers that the loop has better use for)
      const int hidden = fresh(lane), hidden_row = hidden & 31;
      auto query = [&](int i, int part) { return lds.in.q[rb][i][part][query_place(i / 2, hidden >> 5, hidden_row)]; };
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) sc[t][e] = 0.0f;
      // A step's products with the next step's queries on their way and its keys being widened in between.
      i32x4 piece[2];
#pragma unroll
      for (int t = 0; t < 2; t++) piece[t] = key_at(t, 0);
      f16x8 q_low = query(0, 1), q_high = query(0, 0), kw[2];
#pragma unroll
      for (int t = 0; t < 2; t++) kw[t] = widen_f16(piece[t][0], piece[t][1]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < STEPS; i++) {
        f16x8 next_low, next_high, next_kw[2];
        i32x4 next_piece[2];
        if (i + 1 < STEPS) {
          next_low = query(i + 1, 1), next_high = query(i + 1, 0);
#pragma unroll
          for (int t = 0; t < 2; t++) {
            if (i % 2 == 0 && i + 2 < STEPS) next_piece[t] = key_at(t, i / 2 + 1);
            next_kw[t] = widen_f16(piece[t][2 * ((i + 1) & 1)], piece[t][2 * ((i + 1) & 1) + 1]);
            if (i % 2 == 0 && i + 2 < STEPS) piece[t] = next_piece[t];
          }
        }
#pragma unroll
        for (int t = 0; t < 2; t++) sc[t] = mfma32(kw[t], q_low, sc[t]);
#pragma unroll
        for (int t = 0; t < 2; t++) sc[t] = mfma32(kw[t], q_high, sc[t]);
        if (i + 1 < STEPS) {
          q_low = next_low, q_high = next_high;
#pragma unroll
          for (int t = 0; t < 2; t++) kw[t] = next_kw[t];
          if (i % 2 == 0 && i + 2 < STEPS) __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
          else __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
          for (int j = 0; j < 4; j++) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (TAIL)
#pragma unroll
        for (int t = 0; t < 2; t++) {
          const unsigned bits = fresh(bits_now[t]);  // (not tested before the loop, into more scalar registers than there are)
#pragma unroll
          for (int e = 0; e < 16; e++) sc[t][e] = (bits >> e) & 1 ? sc[t][e] : -INFINITY;
        }
      float most = sc[0][0];
      c = fmaxf(now.ks * row_scale, FLT_MIN);  // (never 0: -inf * 0 is NaN; scores that need less are all 0 to the softmax)
#pragma unroll
      for (int e = 1; e < 32; e++) most = fmaxf(most, sc[e / 16][e % 16]);
      most = both_halves(most, max2) * c;
      if (__any(!has_seen && most > -INFINITY)) {
        if (!has_seen && most > -INFINITY) {
          ref = -ceilf(most);
          lift = AIM - ve;
          has_seen = true;
        }
        far = __any(fabsf(ref) >= LARGE_SCORE);
      }
      float above = most + ref;
      shift = fmaxf(ve + lift, LEAST_SHIFT);
      if (again || !__any(above > MOST_WEIGHT || above + shift > MOST)) break;
      again = true;
      float to = ref, by = lift;
      if (above > MOST_WEIGHT) {  // (o's units stay)
        to = -ceilf(most);
        by += ref - to;
        above = most + to;
      }
      if (above + fmaxf(ve + by, LEAST_SHIFT) > MOST) by = AIM - ceilf(above) - ve;
      const float scaled = __builtin_amdgcn_exp2f((to - ref) + (by - lift));
      sum *= __builtin_amdgcn_exp2f(to - ref);
      ref = to;
      lift = by;
      far = __any(fabsf(ref) >= LARGE_SCORE);
#pragma unroll
      for (int i = 0; i < VT; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[i][e] *= scaled;
    }
    if constexpr (BUFS == 1) {
      // the keys' place is free, and the values have come
      if constexpr (RB > 1) loads_left<0>();
      sync();
      bring_keys(then.at, 0);
      if constexpr (RB == 1) loads_left<CHUNKS>();
    }
    if constexpr (TAIL) {
      bool bad = false;
#pragma unroll 1
      for (int at = 64 * rb + lane; at < PAGE * D / 16; at += 64 * RB) {
        i32x4 *here = reinterpret_cast<i32x4 *>(values) + at;
        *here = seen_values(*here, s.len - pg * PAGE - 16 * value_piece(at >> 2, at & 3), bad);
      }
      if (bad) bad_values[stream][n & 1] = 1;
      sync();
      bad_values[stream][~n & 1] = 0;  // (read a turn ago, written in the next: there is a barrier on both sides)
    }
    if constexpr (HAS_ROWS) {
      // A scale that is no power of two rounds products with it: the largest was rounded before ref was taken from it, so are the others.
      float from = ref;
      if (!even || far) {
        const float factor = rarely(c);
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int e = 0; e < 16; e++) sc[t][e] *= factor;
        c = 1.0f;
        if (far) {
          const float less = rarely(ref);
#pragma unroll
          for (int t = 0; t < 2; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) sc[t][e] += less;
          from = 0.0f;
        }
      }
      const float scale = shift + __builtin_amdgcn_logf(rest), of_sum = __builtin_amdgcn_exp2f(-scale);
      from += scale;
#pragma unroll
      for (int t = 0; t < 2; t++) {
        i32x4 vp[VT];
#pragma unroll
        for (int i = 0; i < VT; i++) vp[i] = *reinterpret_cast<const i32x4 *>(values + (32 * i + li) * PAGE + 16 * value_piece(li, 2 * t + half));
#pragma unroll
        for (int e = 0; e < 16; e++) sc[t][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][e], c, from));
        float added = sc[t][0];
#pragma unroll
        for (int e = 1; e < 16; e++) added += sc[t][e];
        sum = __builtin_fmaf(added, of_sum, sum);
#pragma unroll
        for (int u = 0; u < 2; u++) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; e++) x[e] = sc[t][8 * u + e];
          f16x8 pr[2];
          split2(x, pr);
#pragma unroll
          for (int i = 0; i < VT; i++) {
            const f16x8 vw = widen_f16(vp[i][2 * u], vp[i][2 * u + 1]);
#pragma unroll
            for (int part = 1; part >= 0; part--) o[i] = mfma32(vw, pr[part], o[i]);
          }
        }
      }
      if constexpr (TAIL)
        if (bad_values[stream][n & 1]) {  // (loops kept as loops: registers of this rare path must not weigh on the others)
          const unsigned char *vp = p.VP + now.at * (PAGE * D);
#pragma unroll
          for (int i = 0; i < VT; i++) {
            unsigned nan = 0;
#pragma unroll 1
            for (int j = 0; j < PAGE && pg * PAGE + j < s.len; j++) {
              if (!(sees_in(pg, j) & 1)) continue;
#pragma unroll 1
              for (int e = 0; e < 16; e++)
                if ((vp[(32 * i + 8 * (e >> 2) + 4 * half + (e & 3)) * PAGE + j] & 0x7f) == 0x7f) nan |= 1u << e;
            }
#pragma unroll
            for (int e = 0; e < 16; e++) o[i][e] = (nan >> e) & 1 ? NAN : o[i][e];
          }
        }
      if (!known) {
        bool any = true;
        if constexpr (TAIL) any = (sees_in(pg, 0) | sees_in(pg, 16) | sees_in(pg, 32) | sees_in(pg, 48)) != 0;
        if (any) sum = NAN;
      }
    }
    if constexpr (BUFS == 2 || RB > 1) loads_left<0>();
    sync();  // the values' place is free, and the next page's keys (of two places: both) have come
    if constexpr (BUFS == 1) {
      bring_values(then.at, 0);
      if constexpr (RB == 1) loads_left<CHUNKS>();
    }
    now = then;
    then = next_page();
    pg += S;
    n++;
  };
  auto all = [&](auto rows) {
    while (n < whole) turn(std::false_type(), rows);
    while (n < turns) turn(std::true_type(), rows);
  };
  if (has_rows) all(std::true_type());
  else all(std::false_type());
  loads_left<0>();
  sum = both_halves(sum, add2);

  // The wavefronts' shares of a block together: each as an average of values, which is in no danger of leaving fp32, with its weight.
  // lane: row li; registers 4 a .. + 3 of block i are elements 32 i + 8 a + 4 half .. + 3
  const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
  __syncthreads();  // the queries' place is free
#pragma unroll
  for (int i = 0; i < VT; i++)
#pragma unroll
    for (int a = 0; a < 4; a++) {
      f32x4 y;
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = __builtin_amdgcn_ldexpf(o[i][4 * a + e] * inverse, -(int)lift);
      *reinterpret_cast<f32x4 *>(&lds.outs[wave][li * OP + 32 * i + 8 * a + 4 * half]) = y;
    }
  if (half == 0) {
    tops[wave][li] = sum == 0.0f ? -INFINITY : -ref;
    sums[wave][li] = sum;
  }
  __syncthreads();
  const int thread = fresh(threadIdx.x);  // (what is computed of it is computed here, and holds no registers before)
  const long long place = ((2LL * blockIdx.x + (first_segment ? 0 : 1)) * p.kv_heads + head) * ROWS;  // (an item of several workgroups is the first or the last of each)
  if (thread < ROWS) {
    const int block = thread / 32, r = thread % 32;
    float most = -INFINITY, total = 0.0f;
#pragma unroll
    for (int i = 0; i < S; i++) most = fmaxf(most, tops[block + RB * i][r]);
    const float ref = most == -INFINITY ? 0.0f : most;
#pragma unroll
    for (int i = 0; i < S; i++) total += sums[block + RB * i][r] *= __builtin_amdgcn_exp2f(tops[block + RB * i][r] - ref);
    tops[block][r] = total == 0.0f ? 0.0f : 1.0f / total;
    if (!alone && p.partial) *reinterpret_cast<f32x2 *>(p.stats + 2 * (place + thread)) = f32x2{most, total};
  }
  __syncthreads();
#pragma unroll 4
  for (int cell = thread; cell < ROWS * LANES; cell += 64 * WAVES) {
    const int row = cell / LANES, d = 4 * (cell % LANES), block = row / 32, r = row % 32;
    const int flat_row = w.item * ROWS + row, tk = wdh::fdiv(flat_row, p.group);
    const float part = tops[block][r];
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < S; i++) {
      const f32x4 x = *reinterpret_cast<const f32x4 *>(&lds.outs[block + RB * i][r * OP + d]);
      const float f = sums[block + RB * i][r] * part;
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = __builtin_fmaf(f, x[e], y[e]);
    }
    if (tk >= s.n) continue;
    if (alone) *reinterpret_cast<f32x4 *>(p.Y + ((long long)(s.row0 + tk) * p.heads + head * group + (flat_row - tk * group)) * D + d) = y;
    else if (p.partial) *reinterpret_cast<f32x4 *>(p.partial + (place + row) * D + d) = y;
  }
  if (joints && threadIdx.x == 0 && w.unit == 0 && w.ordinal < most_joints)
    joints[w.ordinal * p.kv_heads + head] =
        Joint{s.row0, s.n, w.item, (int)blockIdx.x, (w.before + w.units - 1) / share - (int)blockIdx.x + 1, first_segment ? 0 : 1};
  unit += seg_end - w.unit;
  __syncthreads();  // the next segment's queries go where the results were
  }
}

// What several workgroups have of item blockIdx.x together: D / 4 lanes to a row, SIDES groups of lanes that take
// the parts in turn.  Bound: latency: a joint, then its parts' tops and sums side by side, then the parts.
template <int D, int ROWS, int SIDES>
__global__ __launch_bounds__(256) void tree_join(AttendParams p, const Joint *joints) {
  constexpr int LANES = D / 4, AT_ONCE = 256 / (LANES * SIDES);
  __shared__ __attribute__((aligned(16))) f32x4 results[SIDES > 1 ? 256 : 1];
  const int head = blockIdx.y;
  const Joint joint = joints[blockIdx.x * p.kv_heads + head];
  const int lane = threadIdx.x % LANES, side = threadIdx.x / LANES % SIDES, row = blockIdx.z * AT_ONCE + threadIdx.x / (LANES * SIDES);
  const int flat = joint.item * ROWS + row, token = wdh::fdiv(flat, p.group);
  if (joint.count <= 1) return;
  const bool live = token < joint.n;
  auto slot = [&](int i) { return ((2LL * (joint.from + i) + (i == 0 ? joint.first : 0)) * p.kv_heads + head) * ROWS + row; };
  const f32x2 *stats = reinterpret_cast<const f32x2 *>(p.stats);
  float most = -INFINITY;
  for (int i = lane; i < joint.count; i += LANES) most = fmaxf(most, stats[slot(i)][0]);
#pragma unroll
  for (int off = LANES / 2; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor(most, off, 64));
  const float ref = most == -INFINITY ? 0.0f : most;
  float total = 0.0f;
  for (int i = lane; i < joint.count; i += LANES) total += stats[slot(i)][1] * __builtin_amdgcn_exp2f(stats[slot(i)][0] - ref);
#pragma unroll
  for (int off = LANES / 2; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
  const float part = total == 0.0f ? 0.0f : 1.0f / total;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = side; i < joint.count; i += SIDES) {
    const f32x2 one = stats[slot(i)];
    const f32x4 x = *reinterpret_cast<const f32x4 *>(p.partial + slot(i) * D + 4 * lane);
    const float f = one[1] * __builtin_amdgcn_exp2f(one[0] - ref) * part;
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = __builtin_fmaf(f, x[e], y[e]);
  }
  if constexpr (SIDES > 1) {
    results[threadIdx.x] = y;
    __syncthreads();
    if (side) return;
#pragma unroll
    for (int i = 1; i < SIDES; i++) {
      const f32x4 x = results[threadIdx.x + i * LANES];
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] += x[e];
    }
  }
  if (live) *reinterpret_cast<f32x4 *>(p.Y + ((long long)(joint.row0 + token) * p.heads + head * p.group.d + (flat - token * p.group.d)) * D + 4 * lane) = y;
}

template <int D, int RB, int WAVES>
int launch(const char *who, AttendParams &p, long long rows) {
  constexpr int ROWS = 32 * RB, UNIT = WAVES / RB;
  const long long tokens = p.q.tokens, loose = tokens * p.group.d / ROWS + p.q.seqs, tight = tokens * ((p.group.d + ROWS - 1) / ROWS);
  const long long items = loose < tight ? loose : tight, most_units = (p.q.max_pages + UNIT - 1) / UNIT, units = items * most_units;
  if (items * p.kv_heads > 0xffffffLL / 2 || units > MOST_UNITS) return fail(WDH_EINVAL, "%s: too many rows of tables so wide", who);
  // As many workgroups as the chip holds at a time, or as there can be units.  Or one to each item, where the chip is full of them: the longest item's turns,
  // less those that a share of all would be, have to be worth the join and the second item that a share has parts of (four turns or so).  Heads of 64 with
  // 8 nodes and 500 to 1500 tokens each, shares / items: 64 sequences 25.2 / 21.6 us, with three times as many tokens 36.3 / 44.4, then 128 sequences 67 / 54.
  const long long chip = 8LL / WAVES * wdh::compute_units(), resident = chip / p.kv_heads;
  const long long likely = p.q.seqs * ((rows + ROWS - 1) / ROWS) * p.kv_heads, idle = (likely + chip - 1) / chip * chip - likely;
  p.wgs = (int)(units < resident ? units : resident > 0 ? resident : 1);
  if (most_units == 1 || most_units * idle <= 4 * chip) p.wgs = 0;
  wdh_buf work = 0;
  Joint *joints = nullptr;
  if (p.wgs > 1) {  // (items of one unit are never cut)
    const size_t rows = (size_t)p.wgs * 2 * p.kv_heads * ROWS;
    work = wdh_alloc(rows * (D + 2) * 4 + (size_t)items * p.kv_heads * sizeof(Joint));
    if (!work) return WDH_ENOMEM;
    size_t have;
    p.partial = (float *)wdh::resolve(work, &have);
    p.stats = p.partial + rows * D;
    joints = (Joint *)(p.stats + rows * 2);
  }
  hipStream_t st = wdh::stream();
  hipLaunchKernelGGL((attend_tree<D, RB, WAVES>), dim3((unsigned)(p.wgs ? p.wgs : items), (unsigned)p.kv_heads), dim3(64 * WAVES), 0, st, p, joints, (int)items);
  if (joints) {
    const unsigned wgs = (unsigned)items, heads = (unsigned)p.kv_heads;
    if (p.wgs >= 8 * items) hipLaunchKernelGGL((tree_join<D, ROWS, 8>), dim3(wgs, heads, ROWS * D / 4 * 8 / 256), dim3(256), 0, st, p, joints);
    else hipLaunchKernelGGL((tree_join<D, ROWS, 1>), dim3(wgs, heads, ROWS * D / 4 / 256), dim3(256), 0, st, p, joints);
  }
  if (work) (void)wdh_free(work);
  WDH_LAUNCH_CHECK();
  return WDH_OK;
}
template <int D>
int launch_rows(const char *who, AttendParams &p) {
  const long long rows = ((long long)p.q.tokens * p.group.d + p.q.seqs - 1) / p.q.seqs;  // (of a sequence, on average)
  // More rows to an item read the cache fewer times, and are fewer and longer items.  32, 64 and 128 rows to an item (us), heads of 128, 4 of them in the cache:
  //   32 sequences behind 1500 tokens: of 32 rows 22 / 28 / 34, of 64 rows 28 / 30 / 46, of 128 rows 52 / 36 / 50, of 192 rows 93 / 73 / 60
  //   and one sequence of 512 rows, 2 heads: behind 6400 30 / 24 / 30, behind 25600 49 / 47 / 49, behind 102400 135 / 120 / 118
  // For 33 to 64 rows, 4 heads of 128, items of 64 are the faster ones in 42 of 48 kinds of calls measured (32 / 64 rows to an item: 32 sequences behind 500 25.1 / 22.7, 64 behind
  // 1500 57 / 43, 128 behind 700 90 / 54, one behind 25600 28 / 23); not for 32 sequences behind 1500 (27.6 / 30.6) or one of heads of 64 behind 1500 (12.9 / 14.0).
  if (rows <= 32) return launch<D, 1, D == 128 ? 8 : 4>(who, p, rows);
  const long long pages = p.q.seqs * ((rows + 127) / 128) * p.kv_heads * p.q.max_pages;  // for items of 128 rows, at most
  if (rows <= 64 || pages < 20LL * wdh::compute_units()) return launch<D, 2, 8>(who, p, rows);
  return launch<D, 4, 8>(who, p, rows);
}

}  // namespace

int wdh::kv::attend_trees(const char *who, AttendParams &p, int d) {
  p.partial = p.stats = nullptr;
  return d == 32 ? launch_rows<32>(who, p) : d == 64 ? launch_rows<64>(who, p) : launch_rows<128>(who, p);
}
