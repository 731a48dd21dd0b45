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
// The piece at column c of a row of D elements, zeros beyond its end, in two steps: the load, and behind it (where the piece is used: the load stays in flight until
// then) what makes it whole.  RAGGED: the row's last piece is not whole; where the row has eight elements the last eight are read in its place and shifted, without
// branches.  The elements shifted out belong to the piece before: what another lane may be writing to them in place does not matter.
template <typename T, bool RAGGED> ECAD_DEV Pack8 row_load(const T* row, int c, int D) {
  Pack8 v;
  if constexpr (!RAGGED) {
    v.u = (u32x4){0, 0, 0, 0};
    if (c < D) v.u = reinterpret_cast<const Bytes16*>(row + c)->u;
  } else if (D < 8) {
    v = load_piece<T>(row + c, D - c);
  } else {
    v.u = reinterpret_cast<const Bytes16*>(row + (c < D - 8 ? c : D - 8))->u;
  }
  return v;
}
template <bool RAGGED> ECAD_DEV Pack8 row_piece(const Pack8& raw, int c, int D) {
  if constexpr (!RAGGED) return raw;
  const int s = D < 8 || c < D - 8 ? 0 : c - (D - 8);
  unsigned a = raw.u[0], b = raw.u[1], d = raw.u[2], e = raw.u[3];
  a = s & 4 ? d : a, b = s & 4 ? e : b, d = s & 4 ? 0u : d, e = s & 4 ? 0u : e;
  a = s & 2 ? b : a, b = s & 2 ? d : b, d = s & 2 ? e : d, e = s & 2 ? 0u : e;
  a = s & 1 ? (a >> 16 | b << 16) : a, b = s & 1 ? (b >> 16 | d << 16) : b, d = s & 1 ? (d >> 16 | e << 16) : d, e = s & 1 ? e >> 16 : e;
  const bool none = s >= 8;
  Pack8 v;
  v.u = (u32x4){none ? 0u : a, none ? 0u : b, none ? 0u : d, none ? 0u : e};
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
constexpr float INT8_TINY = 1e-30f;         // below: 1 / s could leave the range of fp32, quotients are divided
constexpr float INT8_MAGIC = 12582912.0f;   // 1.5 2^23: adding it rounds to an integer (ties to even) and leaves that integer's two's complement in the low bits

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
// rows whose largest value is below INT8_TINY (bf16 only): the division itself, in 64 bits
ECAD_DEV float int8_round_tiny(float x, const Int8Scale& k) { return k.s > 0.f ? (float)fmin(fmax(rint((double)x / (double)k.s), -127.0), 127.0) : 0.f; }

// low bytes of four registers into one
ECAD_DEV unsigned gather_bytes(const float* m) {
  const unsigned lo = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, m[1]), __builtin_bit_cast(unsigned, m[0]), 0x0c0c0400u);
  const unsigned hi = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, m[3]), __builtin_bit_cast(unsigned, m[2]), 0x0c0c0400u);
  return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

// eight values of a row to their 8-bit piece (bad and tiny are the row's: the same for all its lanes)
ECAD_DEV u32x2 int8_piece(const float (&x)[8], const Int8Scale& k) {
  float m[8];
  if (k.bad) return (u32x2){0, 0};
  if (!k.tiny) {
    float worst = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      m[e] = __builtin_fmaf(x[e], k.inv, INT8_MAGIC);
      worst = fmaxf(worst, fabsf(__builtin_fmaf(INT8_MAGIC - m[e], k.s, x[e])));
    }
    if (worst >= k.half) {  // one of the eight on or beyond the border
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = __builtin_fmaf(INT8_MAGIC - m[e], k.s, x[e]), step = d > 0.f ? 1.f : -1.f;
        const bool other = fabsf(d) > k.half || (fabsf(d) == k.half && (__builtin_bit_cast(unsigned, m[e]) & 1));
        m[e] += other ? step : 0.f;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) m[e] = int8_round_tiny(x[e], k) + INT8_MAGIC;
  }
  return (u32x2){gather_bytes(m), gather_bytes(m + 4)};
}
template <bool RAGGED> ECAD_DEV void store_int8_piece(int8_t* p, u32x2 v, int n) {  // rows of 8-bit values start on 16 bytes
  if (n >= (RAGGED ? 8 : 1)) {
    *reinterpret_cast<u32x2*>(p) = v;
  } else if (RAGGED) {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) p[e] = (int8_t)(v[e >> 2] >> (8 * (e & 3)));
  }
}

}  // namespace ecad
