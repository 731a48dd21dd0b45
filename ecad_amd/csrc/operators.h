// operators.h -- host interface of operators.hip (the single-op entry points of an 8-bit transformer block): argument records and launch functions.
// Every function checks its arguments, launches on ctx.stream and returns an ECAD_* code; the message of a refusal is in st.msg.  They allocate nothing, hold
// nothing between calls and wait for nothing, so they may be captured into a graph and called from several streams at once.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ecad {

struct OpCtx {
  int dtype;  // ECAD_DTYPE_F16 | ECAD_DTYPE_BF16: the storage type of x, y, h, out, resid and the modulations
  int num_cus;
  hipStream_t stream;
};

struct OpStatus {
  char msg[320];
};

// q[i][:] = rint(x[i][:] / s_i), s_i = max|x_i| / 127 in fp32
struct QuantizeCall {
  const void* x;
  int64_t ldx;
  int8_t* q;
  int64_t ldq;
  float* scale;
  int M, K;
};

// out = epi(sa[m] sw[n] sum_k A[m][k] W[n][k] + bias[n]); epi 3: out (may be null), resid_out = resid + (gate_table + gate_mod[m / rows_per_batch]) * out
struct Int8GemmCall {
  const int8_t* A;
  int64_t lda;
  const float* sa;
  const int8_t* W;
  int64_t ldw;
  const float* sw;
  const float* bias;
  void* out;
  int64_t ldo;
  const void* resid;
  int64_t ldr;
  void* resid_out;
  int64_t ldro;
  const float* gate_table;
  const void* gate_mod;
  int64_t gate_stride;
  int M, N, K, epi, rows_per_batch, kernel;
};

struct GateNormCall {
  const void* h;
  int64_t ldh;
  const void* y;  // null: h' = h, nothing written to h_out
  int64_t ldy;
  void* h_out;
  int64_t ldho;
  void* n_out;  // null with q, or with pre 0
  int64_t ldn;
  int8_t* q;  // 8-bit rows of n instead of n
  int64_t ldq;
  float* q_scale;
  const float* post_weight;  // [D] or null
  const float* pre_weight;
  const float* gate_table;
  const void* gate_mod;
  int64_t gate_stride;
  const float* table_shift;
  const float* table_scale;
  const void* mod_shift;
  const void* mod_scale;
  int64_t mod_stride;
  int M, D, rows_per_batch, post, pre;
  float resid_scale, eps;
};

struct RopeTableCall {
  const void* positions;  // [S][axes] int32 or fp32
  int positions_float;
  const int32_t* axes_dims;  // host
  int axes, S, scaling;
  float* table;  // [S][pairs][2] (cos, sin)
  double theta, factor, original_length, beta_fast, beta_slow;
};

struct RopeHeads {
  const void* x;
  void* out;
  int64_t sb, ss, sh;     // element strides of x by sample, token, head; the elements of a head are contiguous
  int64_t ob, os, oh;
  int H;
};

struct RopeCall {
  RopeHeads q, k;  // k.H == 0: queries only
  const float* table;
  const int32_t* index;  // null: row = token
  int64_t index_stride;  // between samples; 0: the same rows for every sample
  int B, S, D, rot, table_rows, half, inverse;
};

int op_num_cus(int device) noexcept;
int op_quantize_int8(const OpCtx& ctx, const QuantizeCall& c, OpStatus& st) noexcept;
int op_gemm_int8(const OpCtx& ctx, const Int8GemmCall& c, OpStatus& st) noexcept;
int op_gate_norm(const OpCtx& ctx, const GateNormCall& c, OpStatus& st) noexcept;
int op_rope_table(const OpCtx& ctx, const RopeTableCall& c, OpStatus& st) noexcept;
int op_rope(const OpCtx& ctx, const RopeCall& c, OpStatus& st) noexcept;

}  // namespace ecad
