// row_ops.h -- what the row kernels of operators.hip share: 8-element pieces at any element alignment, sums and maxima over a wave or a workgroup, and the exact
// 8-bit rounding.
#pragma once
#include "common.h"

namespace ecad {

// 16 bytes at the alignment of one 16-bit element: rows of odd width or stride keep their wide accesses (global memory takes them at any address here).
struct __attribute__((packed, aligned(2))) Bytes16 {
  u32x4 u;
};
struct __attribute__((packed, aligned(2))) Bytes8 {
  u32x2 u;
};
struct __attribute__((packed, aligned(4))) Floats4 {
  f32x4 f;
};

// elements [0, n) of a piece of eight, the others zero; n >= 8: the whole piece
template <typename T> ECAD_DEV Pack8 load_piece(const T* p, int n) {
  Pack8 v;
  if (n >= 8) {
    v.u = reinterpret_cast<const Bytes16*>(p)->u;
  } else {
    v.u = (u32x4){0, 0, 0, 0};
    const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) v.s[e] = (short)s[e];
  }
  return v;
}
template <typename T> ECAD_DEV void store_piece(T* p, const Pack8& v, int n) {
  if (n >= 8) {
    reinterpret_cast<Bytes16*>(p)->u = v.u;
  } else {
    unsigned short* d = reinterpret_cast<unsigned short*>(p);
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) d[e] = (unsigned short)v.s[e];
  }
}
ECAD_DEV void load_floats(const float* p, int n, float (&f)[8]) {
  if (n >= 8) {
    const f32x4 a = reinterpret_cast<const Floats4*>(p)->f, b = reinterpret_cast<const Floats4*>(p + 4)->f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = a[e], f[4 + e] = b[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = e < n ? p[e] : 0.f;
  }
}

// ---- over the 64 lanes, in the vector unit alone (a shuffle is a round trip through the LDS queue): neighbours by DPP, 16-lane rows and halves by the lane swaps
template <int CTRL, typename V> ECAD_DEV V dpp(V v) { return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true)); }
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_HALF_MIRROR = 0x141, DPP_MIRROR = 0x140;

template <typename V> ECAD_DEV void swap_rows16(V& a, V& b) { asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b)); }
template <typename V> ECAD_DEV void swap_rows32(V& a, V& b) { asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b)); }

template <typename V, typename F> ECAD_DEV V wave_all(V v, F f) {
  v = f(v, dpp<DPP_XOR1>(v));
  v = f(v, dpp<DPP_XOR2>(v));
  v = f(v, dpp<DPP_HALF_MIRROR>(v));
  v = f(v, dpp<DPP_MIRROR>(v));
  V a = v, b = v;
  swap_rows16(a, b);
  a = f(a, b);
  b = a;
  swap_rows32(a, b);
  return f(a, b);
}
struct AddOp {
  ECAD_DEV float operator()(float a, float b) const { return a + b; }
};
struct MaxOp {
  ECAD_DEV unsigned operator()(unsigned a, unsigned b) const { return a > b ? a : b; }
};

// over the WAVES waves that share a row, every wave gets the same value; `turn` alternates two rows of the scratch, so that one barrier per use is enough
template <int WAVES, typename V, typename F> ECAD_DEV V row_all(V v, F f, unsigned (*scratch)[WAVES], int& turn) {
  v = wave_all(v, f);
  if constexpr (WAVES > 1) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) scratch[turn][wave] = __builtin_bit_cast(unsigned, v);
    __syncthreads();
    v = __builtin_bit_cast(V, scratch[turn][0]);
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v = f(v, __builtin_bit_cast(V, scratch[turn][w]));
    turn ^= 1;
  }
  return v;
}

// largest magnitude of a packed piece, as the bits of the 16-bit type: with the sign off they order as the values do, infinity above every number and NaN above
// infinity, so the maximum of the bits (two elements per instruction) also says whether the row holds one
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
ECAD_DEV u16x2 max_bits(u16x2 m, const Pack8& p) {
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, p.u[i] & 0x7fff7fffu));
  return m;
}
ECAD_DEV unsigned fold_bits(u16x2 m) { return m[0] > m[1] ? m[0] : m[1]; }
template <typename T> ECAD_DEV float bits_value(unsigned b) { return (float)__builtin_bit_cast(T, (unsigned short)b); }

// ---- 8-bit rows.  s = max|x| / 127 rounded to fp32 IS the scale; q = the integer nearest to x / s in exact arithmetic, ties to the even one.  inv = 1 / s puts the
// quotient within 1e-5 of the true one, so only a value next to a border can be on the wrong side; its remainder x - n s is exact in fp32 (both are multiples of
// the last place of the smaller one and it is below s) and decides.  A row with an infinity or a NaN has scale NaN and zeros: its products are NaN, not numbers.
constexpr float INT8_MAX_F = 127.0f;
constexpr float INT8_TINY = 1e-30f;  // below: 1 / s could leave the range of fp32, quotients are divided

struct Int8Scale {
  float s, inv, half;
  bool bad, tiny;
};
template <typename T> ECAD_DEV Int8Scale int8_scale(unsigned max_magnitude_bits) {
  const float amax = bits_value<T>(max_magnitude_bits);
  Int8Scale r;
  r.bad = !(amax < __builtin_inff());
  r.tiny = amax < INT8_TINY;
  r.s = r.bad ? __builtin_nanf("") : __fdiv_rn(amax, INT8_MAX_F);
  r.inv = r.bad || r.tiny ? 0.f : __fdiv_rn(1.0f, r.s);
  r.half = 0.5f * r.s;
  return r;
}
ECAD_DEV int int8_round(float x, const Int8Scale& k) {
  float n = rintf(x * k.inv);
  const float d = __builtin_fmaf(-n, k.s, x);
  if (fabsf(d) >= k.half) {  // on or beyond the border
    const float step = d > 0.f ? 1.f : -1.f;
    if (fabsf(d) > k.half || ((int)n & 1)) n += step;
  }
  return (int)n;
}
// rows whose largest value is below INT8_TINY (bf16 only): the division itself, in 64 bits
ECAD_DEV int int8_round_tiny(float x, const Int8Scale& k) { return k.s > 0.f ? (int)fmin(fmax(rint((double)x / (double)k.s), -127.0), 127.0) : 0; }

ECAD_DEV unsigned pack_bytes(int a, int b, int c, int d) { return (unsigned)(a & 255) | (unsigned)(b & 255) << 8 | (unsigned)(c & 255) << 16 | (unsigned)d << 24; }

// eight values of a row to their 8-bit piece (the branches are the row's: the same for all its lanes)
ECAD_DEV u32x2 int8_piece(const float (&x)[8], const Int8Scale& k) {
  int n[8];
  if (k.bad) return (u32x2){0, 0};
  if (!k.tiny) {
#pragma unroll
    for (int e = 0; e < 8; ++e) n[e] = int8_round(x[e], k);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) n[e] = int8_round_tiny(x[e], k);
  }
  return (u32x2){pack_bytes(n[0], n[1], n[2], n[3]), pack_bytes(n[4], n[5], n[6], n[7])};
}
ECAD_DEV void store_int8_piece(int8_t* p, u32x2 v, int n) {  // rows of 8-bit values start on 16 bytes
  if (n >= 8) {
    *reinterpret_cast<u32x2*>(p) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) p[e] = (int8_t)(v[e >> 2] >> (8 * (e & 3)));
  }
}

}  // namespace ecad
