// rope.h -- rotary positions: the table of cosines and sines, and its application to query and key heads.
//
//   table[s][j] = m (cos, sin)(p[s][axis(j)] f_j)       pairs j in axis order; f_j, m from the host (op_rope_table lists the scalings)
//   (x_a, x_b) <- (x_a c - x_b s, x_a s + x_b c)         pair j = elements (2j, 2j + 1) (interleaved) or (j, j + rot / 2) (half); elements from `rot` on stay
#pragma once
#include "operators.h"
#include "row_ops.h"

namespace ecad {

constexpr int ROPE_MAX_PAIRS = 256, ROPE_MAX_AXES = 8;

struct RopeTableArgs {
  const void* positions;
  float* table;
  int positions_float, axes, S, pairs;
  int rows_per_block;                 // rows that a workgroup works on at a time
  float size;
  double quarters[ROPE_MAX_PAIRS];    // 2 f_j / pi: quarter turns per unit of position
  unsigned char axis[ROPE_MAX_PAIRS];
};

// The angle is counted in quarter turns and reduced in 64 bits: the remainder of p (2 f / pi) from the nearest whole one, |r| <= 1/2, is one fma; only r pi / 2 becomes
// fp32, so a position of 10^7 is as exact as position 1.  (The frequency itself has 53 bits: the angle
// is off by 2^-53 of it, which is all of a turn from 2^53 turns on.  Positions beyond come out on the circle, somewhere.)  On |a| <= pi / 4 the Taylor sums below end 2e-9 (sine, a^9) and 2e-10 (cosine, a^10) from the function;
// their fp32 arithmetic, with the rounding of a, stays within 4.5 2^-24 (1.3 2^-24 at the worst of 6.4 million pairs, 1.7 with YaRN's factor; rounded once: 0.5).  That is
// a choice: what the roundings lose, carried along in the small terms, gave 0.71 2^-24 and took 131072 x 64 pairs from 15.4 to 16.9 us, for rows that turn 16-bit heads.
// A thread keeps its pair (frequency and axis are read once) and steps through rows; half a dozen 64-bit operations per pair keep the kernel near its stores (8
// bytes per pair): 131072 x 64 pairs in 15.5 us (4.4 TB/s; with a division per pair to find the row 22.9), 16384 x 64 in 5.3.
__global__ __launch_bounds__(1024) void rope_table_kernel(const RopeTableArgs p) {
  const int r0 = threadIdx.x / (unsigned)p.pairs, j = threadIdx.x - r0 * p.pairs;
  if (r0 >= p.rows_per_block) return;
  const double quarters = p.quarters[j];
  const int axis = p.axis[j];
  const int64_t step = (int64_t)gridDim.x * p.rows_per_block;
  for (int64_t row = (int64_t)blockIdx.x * p.rows_per_block + r0; row < p.S; row += step) {
    const int64_t at = row * p.axes + axis;
    const double pos = p.positions_float ? (double)reinterpret_cast<const float*>(p.positions)[at] : (double)reinterpret_cast<const int32_t*>(p.positions)[at];
    double whole = rint(pos * quarters), rest = __builtin_fma(pos, quarters, -whole);
    if (fabs(whole) >= 0x1p50) {  // the product's own rounding is no longer small: whole quarters are left in the rest
      const double more = rint(rest);
      rest -= more;
      whole = 4.0 * (0.25 * whole - floor(0.25 * whole)) + 4.0 * (0.25 * more - floor(0.25 * more));
    }
    const float a = (float)(rest * 1.5707963267948966);
    const float a2 = a * a;
    const float sn = a * (1.f + a2 * (-1.f / 6 + a2 * (1.f / 120 + a2 * (-1.f / 5040 + a2 * (1.f / 362880)))));
    const float cs = 1.f + a2 * (-0.5f + a2 * (1.f / 24 + a2 * (-1.f / 720 + a2 * (1.f / 40320 + a2 * (-1.f / 3628800)))));
    const double turn = 0.25 * whole;
    const int quadrant = (int)(4.0 * (turn - floor(turn)));  // exact; not-a-number goes to 0 and stays in a
    const float c = quadrant & 1 ? sn : cs, s = quadrant & 1 ? cs : sn;
    const f32x2 o = {p.size * (quadrant == 1 || quadrant == 2 ? -c : c), p.size * (quadrant >= 2 ? -s : s)};
    *reinterpret_cast<f32x2*>(p.table + 2 * (row * p.pairs + j)) = o;
  }
}

struct RopeArgs {
  EcadRopeHeads q, k;
  const float* table;
  const int32_t* index;
  int64_t index_stride;
  int S, D, rot, table_rows, copy;  // copy: out is not x, elements that do not turn are copied
  int units, turning, groups;       // pieces of a head, those of them that turn, head groups of a token
  int tokens_per_block;
  int64_t tokens;
  float sign;                       // -1: turn back
};

constexpr int ROPE_HEADS = 4;  // heads a thread turns with the cosines it has read: four loads in flight, a quarter of the table traffic

// A thread owns one piece of ROPE_HEADS heads of a token: HALF: eight pairs (two pieces half a rotation apart); else four pairs side by side.  Pieces behind the
// rotation are copied.  Rows of the table are picked per token; an index outside the table leaves its token as it is.
// Bound by memory, 4 bytes per value and the table once: 2 x 4608 x (16 + 16) x 128 in 25.5 us side by side and 25.0 in halves (5.9, 6.0 TB/s: part of it from the last-level
// cache), (32 + 8) heads in 35.1 and 30.3 (5.4, 6.2); 8 tokens of 40 heads x 72 in 4.7 us (launch, index, table row and head one after the other).
template <typename T, bool HALF>
__global__ __launch_bounds__(256) void rope_kernel(const RopeArgs p) {
  const int64_t token0 = (int64_t)blockIdx.x * p.tokens_per_block;
  const int per_token = p.units * p.groups;
  const int here = (int)(p.tokens - token0 < p.tokens_per_block ? p.tokens - token0 : p.tokens_per_block);
  const int half = p.rot >> 1;
  for (unsigned it = threadIdx.x; it < (unsigned)(here * per_token); it += 256) {
    const unsigned tk = it / (unsigned)per_token, in = it - tk * per_token;
    const unsigned grp = in / (unsigned)p.units, unit = in - grp * p.units;
    const int64_t token = token0 + tk;
    const int64_t b = token / p.S, s = token - b * p.S;
    const int64_t row = p.index ? p.index[b * p.index_stride + s] : s;
    const bool known = row >= 0 && row < p.table_rows;
    const bool turns = (int)unit < p.turning;
    // first element of the piece (HALF: of its lower part) and how many of the eight belong to it
    const int at = HALF ? (turns ? (int)unit * 8 : p.rot + ((int)unit - p.turning) * 8) : (int)unit * 8;
    const int n = HALF && turns ? half - at : p.D - at;
    if (!(turns && known) && !p.copy) continue;
    float c[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = 1.f, sn[e] = 0.f;
    if (turns && known) {
      const float* t = p.table + row * (int64_t)p.rot + (HALF ? 2 * at : at);
      const int left = HALF ? half - at : (p.rot - at) >> 1;  // pairs of this piece
      float f[16];
      load_floats(t, 2 * left, *reinterpret_cast<float(*)[8]>(f));
      if constexpr (HALF) load_floats(t + 8, 2 * left - 8, *reinterpret_cast<float(*)[8]>(f + 8));
#pragma unroll
      for (int e = 0; e < (HALF ? 8 : 4); ++e)
        if (e < left) c[e] = f[2 * e], sn[e] = p.sign * f[2 * e + 1];
    }
    const int heads = (int)(p.q.H + p.k.H), head0 = (int)grp * ROPE_HEADS;
    Pack8 lo[ROPE_HEADS], hi[ROPE_HEADS];
    T* dst[ROPE_HEADS];
#pragma unroll
    for (int i = 0; i < ROPE_HEADS; ++i) {
      const int h = head0 + i < heads ? head0 + i : heads - 1;
      const bool key = h >= p.q.H;
      const EcadRopeHeads& x = key ? p.k : p.q;
      const int hh = key ? h - (int)p.q.H : h;
      const T* src = reinterpret_cast<const T*>(x.x) + b * x.sample + s * x.token + hh * x.head + at;
      dst[i] = reinterpret_cast<T*>(x.out) + b * x.out_sample + s * x.out_token + hh * x.out_head + at;
      lo[i] = load_piece<T>(src, n);
      if constexpr (HALF)
        if (turns) hi[i] = load_piece<T>(src + half, n);
    }
#pragma unroll
    for (int i = 0; i < ROPE_HEADS; ++i) {
      if (head0 + i >= heads) break;
      if (turns && known) {
        float x[8];
        unpack8<T>(lo[i], x);
        if constexpr (HALF) {
          float y[8], u[8], v[8];
          unpack8<T>(hi[i], y);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            u[e] = x[e] * c[e] - y[e] * sn[e];
            v[e] = x[e] * sn[e] + y[e] * c[e];
          }
          lo[i] = pack8<T>(u);
          hi[i] = pack8<T>(v);
        } else {
          float u[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            u[2 * e] = x[2 * e] * c[e] - x[2 * e + 1] * sn[e];
            u[2 * e + 1] = x[2 * e] * sn[e] + x[2 * e + 1] * c[e];
          }
          // pairs behind the rotation in its last piece: as they are, bit for bit
          const int turned = p.rot - at;
          Pack8 w = pack8<T>(u);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (2 * e < turned) lo[i].u[e] = w.u[e];
        }
      }
      store_piece<T>(dst[i], lo[i], n);
      if constexpr (HALF)
        if (turns) store_piece<T>(dst[i] + half, hi[i], n);
    }
  }
}

}  // namespace ecad
