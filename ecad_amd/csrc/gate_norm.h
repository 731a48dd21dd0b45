// gate_norm.h -- what stands between two sub-layers of a transformer block, in one pass over the hidden rows, and the 8-bit rows that a quantised Linear takes.
//
//   u  = post(y)                       post, pre: none, RMS x / sqrt(mean(x^2) + eps), or layer (x - mean) / sqrt(var + eps), times a weight per channel if given
//   h' = a h + g u                     g = gate_table[d] + gate_mod[sample][d] (1 where neither is given), a = residual scale
//   n  = pre(h') (1 + s) + t           s, t = tables + modulations in the same way (0 where neither is given)
//
// h' goes out rounded once; n is taken from the 32-bit h' before that rounding and rounded once (T, and from there to 8 bits where asked: exactly what
// quantize_rows_kernel makes of the rounded rows, so the fused and the separate path agree bit for bit).  Statistics are two passes over the 32-bit values in
// registers: a one-pass variance of rows with a large mean would cancel.
#pragma once
#include "row_ops.h"

namespace ecad {

enum NormKind { NORM_NONE = 0, NORM_RMS = 1, NORM_LAYER = 2 };

struct GateNormArgs {
  const void* h;
  const void* y;
  void* h_out;
  void* n_out;
  int8_t* q;
  float* q_scale;
  const float *post_weight, *pre_weight, *gate_table, *table_shift, *table_scale;
  const void *gate_mod, *mod_shift, *mod_scale;
  int64_t ldh, ldy, ldho, ldn, ldq, gate_stride, mod_stride;
  int M, D, rows_per_batch, rows_per_group;
  int post, pre;
  float resid_scale, eps;
};

// mean (layer) and 1 / sqrt(. + eps) of the values of a row that is spread over WAVES waves, CH pieces per lane; lanes and pieces beyond the row hold zeros
template <int WAVES, int CH>
ECAD_DEV void row_statistics(const float (&x)[CH][8], int kind, int first, int D, float eps, unsigned (*scratch)[WAVES], int& turn, float& mean, float& rstd) {
  const float inv_d = 1.0f / (float)D;
  mean = 0.f;
  if (kind == NORM_LAYER) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += x[i][e];
    mean = row_all<WAVES>(sum, AddOp{}, scratch, turn) * inv_d;
  }
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int left = D - (first + i * WAVES * 512);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = e < left ? x[i][e] - mean : 0.f;
      sq += d * d;
    }
  }
  rstd = 1.0f / sqrtf(row_all<WAVES>(sq, AddOp{}, scratch, turn) * inv_d + eps);
}

// A row on WAVES waves, CH pieces of eight elements per lane; a workgroup of 256 threads (or WAVES waves) takes rows_per_group consecutive rows.  The channel
// vectors g, 1 + s, t of a sample stay in registers from row to row: read anew for every row they are up to 26 bytes per element out of L2 against the 8 that
// the rows themselves move.
template <typename T, int WAVES, int CH>
__global__ __launch_bounds__(WAVES > 4 ? WAVES * 64 : 256) void gate_norm_kernel(const GateNormArgs p) {
  constexpr int SLOTS = WAVES >= 4 ? 1 : 4 / WAVES;  // rows a workgroup works on at a time
  __shared__ unsigned scratch_all[SLOTS][2][WAVES];
  const int slot = WAVES >= 4 ? 0 : (threadIdx.x >> 6) / WAVES;
  unsigned(*scratch)[WAVES] = scratch_all[slot];
  const int lane = WAVES >= 4 ? threadIdx.x : (threadIdx.x & (64 * WAVES - 1));
  const int first = lane * 8;
  int turn = 0;
  float G[CH][8], A[CH][8], B[CH][8];
  int have = -1;  // the sample that G, A, B belong to
  const int64_t row0 = ((int64_t)blockIdx.x * SLOTS + slot) * p.rows_per_group;
  // every wave of a workgroup makes the same number of turns: barriers inside (WAVES > 1) are met by all, and a wave without a row repeats the last one unwritten
  for (int r = 0; r < p.rows_per_group; ++r) {
    const int64_t row_ = row0 + r;
    if (WAVES == 1 && row_ >= p.M) break;
    const bool live = row_ < p.M;
    const int64_t row = live ? row_ : p.M - 1;
    const T* hrow = reinterpret_cast<const T*>(p.h) + row * p.ldh;
    const T* yrow = reinterpret_cast<const T*>(p.y) + row * p.ldy;
    Pack8 hv[CH], yv[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = first + i * WAVES * 512;
      hv[i] = load_piece<T>(hrow + c, p.D - c);
      if (p.y) yv[i] = load_piece<T>(yrow + c, p.D - c);
    }
    const int b = (int)(row / p.rows_per_batch);
    if (b != have) {
      have = b;
      const T* gm = reinterpret_cast<const T*>(p.gate_mod) + (int64_t)b * p.gate_stride;
      const T* sm = reinterpret_cast<const T*>(p.mod_scale) + (int64_t)b * p.mod_stride;
      const T* tm = reinterpret_cast<const T*>(p.mod_shift) + (int64_t)b * p.mod_stride;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int c = first + i * WAVES * 512, n = p.D - c;
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) G[i][e] = p.gate_table || p.gate_mod ? 0.f : 1.f, A[i][e] = 1.f, B[i][e] = 0.f;
        if (p.gate_table) {
          load_floats(p.gate_table + c, n, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) G[i][e] = f[e];
        }
        if (p.gate_mod) {
          unpack8<T>(load_piece<T>(gm + c, n), f);
#pragma unroll
          for (int e = 0; e < 8; ++e) G[i][e] += f[e];
        }
        if (p.post_weight) {
          load_floats(p.post_weight + c, n, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) G[i][e] *= f[e];
        }
        if (p.table_scale) {
          load_floats(p.table_scale + c, n, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) A[i][e] += f[e];
        }
        if (p.mod_scale) {
          unpack8<T>(load_piece<T>(sm + c, n), f);
#pragma unroll
          for (int e = 0; e < 8; ++e) A[i][e] += f[e];
        }
        if (p.pre_weight) {
          load_floats(p.pre_weight + c, n, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) A[i][e] *= f[e];
        }
        if (p.table_shift) {
          load_floats(p.table_shift + c, n, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) B[i][e] = f[e];
        }
        if (p.mod_shift) {
          unpack8<T>(load_piece<T>(tm + c, n), f);
#pragma unroll
          for (int e = 0; e < 8; ++e) B[i][e] += f[e];
        }
      }
    }
    float x[CH][8];
    if (p.y) {
      float u[CH][8], mean = 0.f, rstd = 1.f;
#pragma unroll
      for (int i = 0; i < CH; ++i) unpack8<T>(yv[i], u[i]);
      if (p.post) row_statistics<WAVES, CH>(u, p.post, first, p.D, p.eps, scratch, turn, mean, rstd);
      T* ho = reinterpret_cast<T*>(p.h_out) + row * p.ldho;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int c = first + i * WAVES * 512;
        unpack8<T>(hv[i], x[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = c + e < p.D ? p.resid_scale * x[i][e] + (u[i][e] - mean) * rstd * G[i][e] : 0.f;
        if (live) store_piece<T>(ho + c, pack8<T>(x[i]), p.D - c);
      }
    } else {
#pragma unroll
      for (int i = 0; i < CH; ++i) unpack8<T>(hv[i], x[i]);
    }
    if (p.pre == NORM_NONE) continue;
    float mean, rstd;
    row_statistics<WAVES, CH>(x, p.pre, first, p.D, p.eps, scratch, turn, mean, rstd);
    Pack8 nv[CH];
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = first + i * WAVES * 512;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] = c + e < p.D ? (x[i][e] - mean) * rstd * A[i][e] + B[i][e] : 0.f;
      nv[i] = pack8<T>(x[i]);
      m = max_bits(m, nv[i]);
    }
    if (p.q) {
      const unsigned bits = row_all<WAVES>(fold_bits(m), MaxOp{}, scratch, turn);
      const Int8Scale k = int8_scale<T>(bits);
      if (live && lane == 0) p.q_scale[row] = k.s;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int c = first + i * WAVES * 512;
        unpack8<T>(nv[i], x[i]);
        if (live) store_int8_piece(p.q + row * p.ldq + c, int8_piece(x[i], k), p.D - c);
      }
    } else {
      T* no = reinterpret_cast<T*>(p.n_out) + row * p.ldn;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int c = first + i * WAVES * 512;
        if (live) store_piece<T>(no + c, nv[i], p.D - c);
      }
    }
  }
}

struct QuantizeArgs {
  const void* x;
  int8_t* q;
  float* scale;
  int64_t ldx, ldq;
  int M, K;
};

// One row per WAVES waves, the whole row in registers between the maximum and the rounding: read once.
template <typename T, int WAVES, int CH>
__global__ __launch_bounds__(WAVES > 4 ? WAVES * 64 : 256) void quantize_rows_kernel(const QuantizeArgs p) {
  constexpr int SLOTS = WAVES >= 4 ? 1 : 4 / WAVES;
  __shared__ unsigned scratch_all[SLOTS][2][WAVES];
  const int slot = WAVES >= 4 ? 0 : (threadIdx.x >> 6) / WAVES;
  const int lane = WAVES >= 4 ? threadIdx.x : (threadIdx.x & (64 * WAVES - 1));
  const int64_t row_ = (int64_t)blockIdx.x * SLOTS + slot;
  const bool live = row_ < p.M;
  const int64_t row = live ? row_ : p.M - 1;
  const T* xrow = reinterpret_cast<const T*>(p.x) + row * p.ldx;
  int turn = 0;
  Pack8 v[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = (lane + i * WAVES * 64) * 8;
    v[i] = load_piece<T>(xrow + c, p.K - c);
  }
  u16x2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < CH; ++i) m = max_bits(m, v[i]);
  const unsigned bits = row_all<WAVES>(fold_bits(m), MaxOp{}, scratch_all[slot], turn);
  const Int8Scale k = int8_scale<T>(bits);
  if (!live) return;
  if (lane == 0) p.scale[row] = k.s;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = (lane + i * WAVES * 64) * 8;
    float x[8];
    unpack8<T>(v[i], x);
    store_int8_piece(p.q + row * p.ldq + c, int8_piece(x, k), p.K - c);
  }
}

}  // namespace ecad
