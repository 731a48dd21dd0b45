// operators.h -- host interface of operators.hip (the single-op entry points of an 8-bit transformer block): argument records and launch functions.
// Every function checks its arguments, launches on ctx.stream and returns an ECAD_* code; the message of a refusal is in st.msg.  They allocate nothing, hold
// nothing between calls and wait for nothing, so they may be captured into a graph and called from several streams at once.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ecad_hip.h"

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

struct RopeTableCall {
  const void* positions;  // [S][axes] int32 or fp32
  int positions_float;
  const int32_t* axes_dims;  // host
  int axes, S, scaling;
  float* table;  // [S][pairs][2] (cos, sin)
  double theta, factor, original_length, beta_fast, beta_slow;
};

int op_num_cus(int device) noexcept;
int op_quantize_int8(const OpCtx& ctx, const QuantizeCall& c, OpStatus& st) noexcept;
int op_gemm_int8(const OpCtx& ctx, const EcadInt8Gemm& c, OpStatus& st) noexcept;
int op_gate_norm(const OpCtx& ctx, const EcadGateNorm& c, OpStatus& st) noexcept;
int op_rope_table(const OpCtx& ctx, const RopeTableCall& c, OpStatus& st) noexcept;
int op_rope(const OpCtx& ctx, const EcadRope& c, OpStatus& st) noexcept;

}  // namespace ecad
