// Positions of queries and keys: each head normed (or not) and rotated by the angles of its token's position, in one pass.
//
// The reference has no such operators; in its terms they are the chain of a norm (see norm_fp8.hip), Split, Neg, Concat, Mul, Add
// (src/descriptor_runner/operators/cpu/operators/standard/binary7.ts:24-75, split.ts:12-87, concat.ts:21-84).
//
// A head stays in the registers of 8 to 64 lanes between its sum of squares and its use.  Bound: memory, then instructions.
#include "common.h"
#include "fastdiv.h"
#include "rope.h"

namespace {

using namespace wdh::rope;
using wdh::fail;
using wdh::rowmath::RowFactor;

struct RopeParams {
  const float *X;
  float *Y;
  long long x_stride, x_head, y_stride, y_head;  // elements between tokens, and between a token's heads
  const float *q_gamma, *k_gamma;
  const int *positions;
  Rotation r;
  long long units;      // tokens * heads
  wdh::FastDiv heads;   // q_heads of one kind, then those of the other
  int q_heads, d;
  double of_d;          // 1 / d
  float eps;
};

// LANES lanes to a head, NP pieces of four elements to a lane.  FACING: a head of 8 LANES elements is rotated whole, by halves, so that a lane's two pieces
// are each other's partners.  A lane has two pieces wherever there are as many, for it is instructions that bound this: 8192 tokens of 40 heads of 128 take
// 86 us with one piece to a lane, 62 so.  EXCHANGED: halves of a part of the head; 64 of 128 elements 73 us with partners loaded again, 65 so.  (More heads to a lane take longer: 2 95 us, 4 121.)
template <int LANES, int NP, int PAIRS>
__global__ __launch_bounds__(256) void head_rope(RopeParams p) {
  const int lane = threadIdx.x % LANES;
  const long long at = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int unit = (int)(at < p.units ? at : p.units - 1);  // (behind the last: the last once more, not stored)
  const int token = wdh::fdiv(unit, p.heads), head = unit - token * p.heads.d, d = PAIRS == FACING ? 8 * LANES : p.d;
  const float *x = p.X + token * p.x_stride + head * p.x_head, *g = head < p.q_heads ? p.q_gamma : p.k_gamma;
  const int position = p.positions ? p.positions[token] : token;
  f32x4 v[NP], o[NP], gamma[NP], other_gamma[NP];
  Angles a[NP];
#pragma unroll
  for (int i = 0; i < NP; i++) {
    const int d0 = 4 * (lane + LANES * i);
    v[i] = load4(x, d0, d);
    if (g) gamma[i] = load4(g, d0, d);
    if constexpr (PAIRS == ANYWHERE) {
      o[i] = partners(p.r, x, d0, d);
      if (g) other_gamma[i] = partners(p.r, g, d0, d);
    }
    if ((PAIRS != FACING && PAIRS != EXCHANGED) || i == 0) a[i] = angles<PAIRS>(p.r, position, d0);
  }
  if (g) {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < NP; i++) sum += squares(v[i]);
    const RowFactor f = head_factor(group_sum<LANES>(sum) * p.of_d, p.eps);
#pragma unroll
    for (int i = 0; i < NP; i++) {
      v[i] = normed(v[i], f, gamma[i]);
      if constexpr (PAIRS == ANYWHERE) o[i] = normed(o[i], f, other_gamma[i]);
    }
  }
  if constexpr (PAIRS == EXCHANGED) {
#pragma unroll
    for (int e = 0; e < 4; e++) o[0][e] = __shfl_xor(v[0][e], p.r.half / 4, LANES);
    v[0] = turn(p.r, 4 * lane, v[0], o[0], a[0]);
  }
  if (at >= p.units) return;
  if constexpr (PAIRS == FACING) turn_facing(v[0], v[1], a[0]);
  float *y = p.Y + token * p.y_stride + head * p.y_head;
#pragma unroll
  for (int i = 0; i < NP; i++) {
    const int d0 = 4 * (lane + LANES * i);
    if constexpr (PAIRS == ANYWHERE) v[i] = turn(p.r, d0, v[i], o[i], a[i]);
    if constexpr (PAIRS == NEIGHBOURS) v[i] = turn_neighbours(p.r, d0, v[i], a[i]);
    store4(y, d0, d, v[i]);
  }
}

template <int LANES, int NP, int PAIRS>
int launch(const RopeParams &p) {
  constexpr int PER = 256 / LANES;
  const long long wgs = (p.units + PER - 1) / PER;
  if (wgs > 0xffffff) return fail(WDH_EINVAL, "wdh_rope: too many heads");  // (a launch has fewer than 2^32 threads)
  hipLaunchKernelGGL((head_rope<LANES, NP, PAIRS>), dim3((unsigned)wgs), dim3(256), 0, wdh::stream(), p);
  WDH_LAUNCH_CHECK();
  return WDH_OK;
}
template <int LANES, int NP>
int launch_pairs(const RopeParams &p, bool neighbours) {
  if (neighbours) return launch<LANES, NP, NEIGHBOURS>(p);
  if constexpr (NP == 2)
    if (p.r.half == 4 * LANES) return launch<LANES, 2, FACING>(p);
  // (a power of two of four elements, within the lanes' first pieces)
  if (p.r.half >= 4 && (p.r.half & (p.r.half - 1)) == 0 && p.r.half <= 2 * LANES) return launch<LANES, NP, EXCHANGED>(p);
  return launch<LANES, NP, ANYWHERE>(p);
}

}  // namespace

extern "C" int wdh_rope(wdh_buf hX, int64_t x_offset, int64_t x_stride, int64_t x_head, wdh_buf hY, int64_t y_offset, int64_t y_stride,
                        int64_t y_head, wdh_buf hQGamma, wdh_buf hKGamma, wdh_buf hCos, wdh_buf hSin, wdh_buf hPositions, int64_t tokens,
                        int heads, int k_heads, int d, int rotary, int rows, int interleaved, float eps) {
  WDH_REQUIRE_INIT();
  WDH_REQUIRE_COMPUTE_LANE();
  if (tokens < 0 || heads < 0 || k_heads < 0 || rows < 0) return fail(WDH_EINVAL, "wdh_rope: negative extent");
  if (d < 1 || d > 1024) return fail(WDH_EINVAL, "wdh_rope: heads of %d elements (1 to 1024)", d);
  if (rotary < 0 || rotary > d || rotary % 2) return fail(WDH_EINVAL, "wdh_rope: %d rotated elements of %d (an even number)", rotary, d);
  if ((rotary > 0) != (hCos != 0) || (rotary > 0) != (hSin != 0)) return fail(WDH_EINVAL, "wdh_rope: Cos and Sin go with rotated elements");
  if (!(eps >= 0.0f)) return fail(WDH_EINVAL, "wdh_rope: epsilon %g", (double)eps);
  if (heads > 65536 || k_heads > 65536) return fail(WDH_EINVAL, "wdh_rope: too many heads");
  const int64_t all = (int64_t)heads + k_heads;
  if (tokens == 0 || all == 0) return WDH_OK;
  if (tokens > 0x7fffffffLL / all) return fail(WDH_EINVAL, "wdh_rope: too many heads");
  const int64_t most = 1LL << 40;
  for (int64_t v : {x_offset, x_stride, x_head, y_offset, y_stride, y_head})
    if (v < 0 || v > most) return fail(WDH_EINVAL, "wdh_rope: an offset or a stride of %lld elements", (long long)v);
  const int64_t x_last = (tokens - 1) * x_stride + (all - 1) * x_head, y_last = (tokens - 1) * y_stride + (all - 1) * y_head;
  if (x_last > most || y_last > most) return fail(WDH_EINVAL, "wdh_rope: rows span too much");
  const bool rows_of_heads = (all == 1 || y_head >= d) && (tokens == 1 || y_stride >= (all - 1) * y_head + d);
  const bool heads_of_rows = (tokens == 1 || y_stride >= d) && (all == 1 || y_head >= (tokens - 1) * y_stride + d);
  if (!rows_of_heads && !heads_of_rows) return fail(WDH_EINVAL, "wdh_rope: heads of Y overlap");
  if (hX == hY && (x_offset != y_offset || x_stride != y_stride || x_head != y_head))
    return fail(WDH_EINVAL, "wdh_rope: Y is X in another layout");
  for (wdh_buf h : {hQGamma, hKGamma, hCos, hSin, hPositions})
    if (h && h == hY) return fail(WDH_EINVAL, "wdh_rope: Y aliases an input");
  void *px, *py, *qg = nullptr, *kg = nullptr, *pc = nullptr, *ps = nullptr, *pp = nullptr;
  if (!wdh::operand(hX, (size_t)(x_offset + x_last + d) * 4, "wdh_rope: X", &px)) return WDH_EINVAL;
  if (!wdh::operand(hY, (size_t)(y_offset + y_last + d) * 4, "wdh_rope: Y", &py)) return WDH_EINVAL;
  if (hQGamma && !wdh::operand(hQGamma, (size_t)d * 4, "wdh_rope: QGamma", &qg)) return WDH_EINVAL;
  if (hKGamma && !wdh::operand(hKGamma, (size_t)d * 4, "wdh_rope: KGamma", &kg)) return WDH_EINVAL;
  const size_t table = (size_t)rows * (rotary / 2) * 4;
  if (hCos && !wdh::operand(hCos, table, "wdh_rope: Cos", &pc)) return WDH_EINVAL;
  if (hSin && !wdh::operand(hSin, table, "wdh_rope: Sin", &ps)) return WDH_EINVAL;
  if (hPositions && !wdh::operand(hPositions, (size_t)tokens * 4, "wdh_rope: Positions", &pp)) return WDH_EINVAL;
  RopeParams p;
  p.X = (const float *)px + x_offset;
  p.Y = (float *)py + y_offset;
  p.x_stride = x_stride; p.x_head = x_head; p.y_stride = y_stride; p.y_head = y_head;
  p.q_gamma = (const float *)qg; p.k_gamma = (const float *)kg;
  p.positions = (const int *)pp;
  p.r = Rotation{(const float *)pc, (const float *)ps, rotary / 2, rows};
  p.units = tokens * all;
  p.heads = wdh::make_fastdiv(all);
  p.q_heads = heads; p.d = d; p.of_d = 1.0 / d; p.eps = eps;
  const bool neighbours = interleaved || rotary == 0;  // (no pairs: none that need others)
  if (d <= 32) return launch_pairs<8, 1>(p, neighbours);
  if (d <= 64) return launch_pairs<8, 2>(p, neighbours);
  if (d <= 128) return launch_pairs<16, 2>(p, neighbours);
  if (d <= 256) return launch_pairs<32, 2>(p, neighbours);
  return d <= 512 ? launch_pairs<64, 2>(p, neighbours) : launch_pairs<64, 4>(p, neighbours);
}
