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

// Rows a workgroup works on at a time: four where a row is one wave's, else one (waves of a row meet at barriers, and rows end at different turns).
constexpr int row_slots(int waves) { return waves == 1 ? 4 : 1; }

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

// Layer: takes the mean off the values of a row that is spread over WAVES waves, CH pieces per lane.  Returns 1 / sqrt(mean square + eps).  Pieces and lanes beyond the row
// hold zeros before (and less the mean behind: whoever multiplies them does so with zeros).  RAGGED: the row's last piece is not whole.
template <int WAVES, int CH, bool RAGGED>
ECAD_DEV float row_statistics(float (&x)[CH][8], int kind, int first, int D, float inv_d, float eps, unsigned (*scratch)[WAVES], int& turn) {
  if (kind == NORM_LAYER) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += x[i][e];
    const float mean = row_all<WAVES>(sum, AddOp{}, scratch, turn) * inv_d;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] -= mean;
  }
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int left = D - (first + i * WAVES * 512);
    float part = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = RAGGED && e >= left ? 0.f : x[i][e];
      part += d * d;
    }
    sq += left > 0 ? part : 0.f;
  }
  return 1.0f / sqrtf(row_all<WAVES>(sq, AddOp{}, scratch, turn) * inv_d + eps);
}

template <typename T, bool RAGGED> ECAD_DEV void row_store(T* p, const Pack8& v, int left) {
  if constexpr (RAGGED) store_piece<T>(p, v, left);
  else if (left > 0) reinterpret_cast<Bytes16*>(p)->u = v.u;
}

// A row on WAVES waves, CH pieces of eight elements per lane; every wave (or workgroup of a wider row) takes rows_per_group consecutive rows, the next one's
// loads in flight while one is worked on.  The channel vectors g, 1 + s, t of a sample stay in registers from row to row: read anew for every row they are up to
// 26 bytes per element out of L2 against the 8 that the rows themselves move.  They are zero beyond the row, and with them everything that is computed there.
// HOLD false (rows of more than 8192 values on 16 waves, whose lanes have 128 registers): read anew all the same, and from 16384 values on nothing is in flight ahead.
// Bound by memory: 8 bytes per value (7 with 8-bit rows out), at the 5.15 TB/s of a large copy 14.7 us for 8192 x 1152 (19.0 measured, a launch being 1.9 of them),
// 104 us for 16384 x 4096 (109), 58.6 us for 32768 x 1152 (56.3: 5.4 TB/s, part of it from the last-level cache), 52 us for 4096 x 8192 (52.4).  Rows beyond 8192 values:
// 2048 x 16384 79 us (3.4 TB/s), 2048 x 32768 156 us (3.4): one row per CU at a time, and the channel vectors out of L2 for each.  To 8-bit rows 4096 x 1152 15.8 us of 6.4
// (two rows a wave: ramp and two rows' latency).  Few rows: 5 x 1153 5.5 us: a launch, the loads of the row and its vectors, four meetings of the row's waves.
// (Times here and in the other headers: medians of a kernel trace, the same data again and again; profiles/operators_kernel_stats.csv.)
template <typename T, int WAVES, int CH, bool RAGGED, bool HOLD>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) void gate_norm_kernel(const GateNormArgs p) {
  constexpr int SLOTS = row_slots(WAVES);
  constexpr bool AHEAD = HOLD || CH <= 2;  // the next row's loads are in flight while one is worked on
  __shared__ unsigned scratch[2][WAVES];  // (one wave a row: not used)
  const int slot = WAVES == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const int lane = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
  int first = lane * 8;
  int turn = 0;
  float G[HOLD ? CH : 1][8], A[HOLD ? CH : 1][8], B[HOLD ? CH : 1][8];
  int have = -1;  // the sample that G, A, B belong to
  const float inv_d = 1.0f / (float)p.D;
  const int64_t row0 = ((int64_t)blockIdx.x * SLOTS + slot) * p.rows_per_group;
  // rows_per_group and M are the same for all waves of a row: they leave the loop together (the barriers inside are a row's own where WAVES > 1)
  const int64_t end = row0 + p.rows_per_group < p.M ? row0 + p.rows_per_group : p.M;
  Pack8 hv[CH], yv[CH];
  auto fetch = [&](int64_t row) {
    const T* hrow = reinterpret_cast<const T*>(p.h) + row * p.ldh;
    const T* yrow = reinterpret_cast<const T*>(p.y) + row * p.ldy;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = first + i * WAVES * 512;
      hv[i] = row_load<T, RAGGED>(hrow, c, p.D);
      if (p.y) yv[i] = row_load<T, RAGGED>(yrow, c, p.D);
    }
  };
  if (AHEAD && row0 < end) fetch(row0);
  for (int64_t row = row0; row < end; ++row) {
    // one piece after the other, its addresses made for it: ahead of the loop and side by side they took 200 registers that are not there (2048 x 32768: 555 us)
    auto next_piece = [&]() {
      if constexpr (!HOLD) {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" : "+v"(first));
      }
    };
    next_piece();
    if constexpr (!AHEAD) fetch(row);
    const int b = (int)((unsigned)row / (unsigned)p.rows_per_batch);
    // the vectors of piece i: the gate's (what & 1) or scale and shift (what & 2).  All loads first: each is behind a branch on its pointer, and combined one by one
    // they would wait for each other (eight round trips to memory in front of the first row: 5 of the 8.5 us of a call with five rows)
    auto channels = [&](int i, int at, int what) {
      const int c = first + i * WAVES * 512, n = p.D - c;
      float gt[8], pw[8], st[8], ew[8], ht[8];
      Pack8 gm, sm, hm;
      auto table = [&](const float* v, float (&f)[8]) {
        if (!v) return;
        if constexpr (RAGGED) {
          load_floats(v + c, n, f);
        } else if (n > 0) {
          load_floats(v + c, 8, f);
        }
      };
      auto mod = [&](const void* base, int64_t stride, Pack8& f) {
        if (base) f = row_load<T, RAGGED>(reinterpret_cast<const T*>(base) + (int64_t)b * stride, c, p.D);
      };
      if (what & 1) table(p.gate_table, gt), mod(p.gate_mod, p.gate_stride, gm), table(p.post_weight, pw);
      if (what & 2) table(p.table_scale, st), mod(p.mod_scale, p.mod_stride, sm), table(p.pre_weight, ew), table(p.table_shift, ht), mod(p.mod_shift, p.mod_stride, hm);
      float f[8];
      if (what & 1) {
#pragma unroll
        for (int e = 0; e < 8; ++e) G[at][e] = p.gate_table ? gt[e] : (p.gate_mod ? 0.f : 1.f);
        unpack8<T>(row_piece<RAGGED>(gm, c, p.D), f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (p.gate_mod) G[at][e] += f[e];
          if (p.post_weight) G[at][e] *= pw[e];
          if (e >= n) G[at][e] = 0.f;
        }
      }
      if (what & 2) {
        unpack8<T>(row_piece<RAGGED>(sm, c, p.D), f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          A[at][e] = p.table_scale ? 1.f + st[e] : 1.f;
          if (p.mod_scale) A[at][e] += f[e];
          if (p.pre_weight) A[at][e] *= ew[e];
          if (e >= n) A[at][e] = 0.f;
        }
        unpack8<T>(row_piece<RAGGED>(hm, c, p.D), f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          B[at][e] = p.table_shift ? ht[e] : 0.f;
          if (p.mod_shift) B[at][e] += f[e];
          if (e >= n) B[at][e] = 0.f;
        }
      }
    };
    if (HOLD && b != have) {
      have = b;
#pragma unroll
      for (int i = 0; i < CH; ++i) channels(i, i, 3);
    }
    float x[CH][8];
    auto unpack_h = [&](int i) { unpack8<T>(row_piece<RAGGED>(hv[i], first + i * WAVES * 512, p.D), x[i]); };
    if (AHEAD || !p.y) {
#pragma unroll
      for (int i = 0; i < CH; ++i) unpack_h(i);
    }
    if (p.y) {
      float u[CH][8];
#pragma unroll
      for (int i = 0; i < CH; ++i) unpack8<T>(row_piece<RAGGED>(yv[i], first + i * WAVES * 512, p.D), u[i]);
      if (AHEAD && row + 1 < end) fetch(row + 1);
      if (p.post) {
        const float rstd = row_statistics<WAVES, CH, RAGGED>(u, p.post, first, p.D, inv_d, p.eps, scratch, turn);
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) u[i][e] *= rstd;
      }
      T* ho = reinterpret_cast<T*>(p.h_out) + row * p.ldho;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int c = first + i * WAVES * 512, at = HOLD ? i : 0;
        if constexpr (!HOLD) next_piece();
        if constexpr (!AHEAD) unpack_h(i);
        if constexpr (!HOLD) channels(i, 0, 1);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = __builtin_fmaf(u[i][e], G[at][e], p.resid_scale * x[i][e]);
        row_store<T, RAGGED>(ho + c, pack8<T>(x[i]), p.D - c);
      }
    } else if (AHEAD && row + 1 < end) {
      fetch(row + 1);
    }
    if (p.pre == NORM_NONE) continue;
    const float rstd = row_statistics<WAVES, CH, RAGGED>(x, p.pre, first, p.D, inv_d, p.eps, scratch, turn);
    Pack8 nv[CH];
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int at = HOLD ? i : 0;
      if constexpr (!HOLD) next_piece(), channels(i, 0, 2);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] = __builtin_fmaf(x[i][e] * rstd, A[at][e], B[at][e]);
      nv[i] = pack8<T>(x[i]);
      if constexpr (!HOLD) asm volatile("" : "+v"(nv[i].u));  // now, not where it is stored
    }
    if (p.q) {
#pragma unroll
      for (int i = 0; i < CH; ++i) m = max_bits(m, nv[i]);
      const Int8Scale k = int8_scale<T>(__builtin_amdgcn_readfirstlane(row_all<WAVES>(fold_bits(m), MaxOp{}, scratch, turn)));
      if (lane == 0) p.q_scale[row] = k.s;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        next_piece();
        const int c = first + i * WAVES * 512;
        unpack8<T>(nv[i], x[i]);
        store_int8_piece<RAGGED>(p.q + row * p.ldq + c, int8_piece(x[i], k), p.D - c);
      }
    } else {
      T* no = reinterpret_cast<T*>(p.n_out) + row * p.ldn;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        next_piece();
        const int c = first + i * WAVES * 512;
        row_store<T, RAGGED>(no + c, nv[i], p.D - c);
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

// One row per WAVES waves, the whole row in registers between the maximum and the rounding: read once.  Bound by memory, 3 bytes per value: 8192 x 4608 19.2 us
// (5.9 TB/s, part of it from the last-level cache; a copy moves 5.15), 8192 x 1152 7.2 us (3.9 TB/s with its launch), 601 x 4001 4.8 us.
template <typename T, int WAVES, int CH, bool RAGGED>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) void quantize_rows_kernel(const QuantizeArgs p) {
  __shared__ unsigned scratch[2][WAVES];
  const int lane = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
  const int64_t row = (int64_t)blockIdx.x * row_slots(WAVES) + (WAVES == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
  if (row >= p.M) return;  // whole workgroups, or waves that share nothing
  const T* xrow = reinterpret_cast<const T*>(p.x) + row * p.ldx;
  int turn = 0;
  Pack8 v[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    v[i] = row_load<T, RAGGED>(xrow, (lane + i * WAVES * 64) * 8, p.K);
  }
  u16x2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    v[i] = row_piece<RAGGED>(v[i], (lane + i * WAVES * 64) * 8, p.K);
    m = max_bits(m, v[i]);
  }
  const Int8Scale k = int8_scale<T>(__builtin_amdgcn_readfirstlane(row_all<WAVES>(fold_bits(m), MaxOp{}, scratch, turn)));
  if (lane == 0) p.scale[row] = k.s;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = (lane + i * WAVES * 64) * 8;
    float x[8];
    unpack8<T>(v[i], x);
    store_int8_piece<RAGGED>(p.q + row * p.ldq + c, int8_piece(x, k), p.K - c);
  }
}

}  // namespace ecad
