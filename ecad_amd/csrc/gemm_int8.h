// gemm_int8.h -- 8-bit integer products with a scale per row (token) and per column (output channel):
//
//   o[m][n] = act(sa[m] sw[n] sum_k A[m][k] W[n][k] + bias[n]),   epilogue 3: resid'[m][n] = resid[m][n] + (gt[n] + gm[sample][n]) T(o[m][n])
//
// The sums are whole numbers in 32 bits (K < 2^17: 127^2 K < 2^31), so no order of K changes them and every kernel here gives the same bits.  The scales
// (the token's first: their own product could leave the normal range of fp32 where the result does not), the bias, the activation and the gate are fp32; o is rounded once to the storage type, and the residual takes the rounded o (it is what a cache of
// the sub-layer holds and replays).  A row whose scale is NaN comes out NaN.
//
// Operands: rows of 8-bit integers on 16 bytes, any M, N, K.  The last 16-byte piece of a row may reach past column K: it stays inside the aligned 16 bytes that
// hold a value of the row, and the bytes behind K are masked on the W side (zero times anything is zero).
#pragma once
#include "gemm_int8_asm.h"
#include "row_ops.h"

namespace ecad {

typedef int i32x4 __attribute__((ext_vector_type(4)));

enum Int8Epi { I8_BIAS = 0, I8_GELU = 1, I8_SILU = 2, I8_RESID = 3 };

struct Int8GemmArgs {
  const int8_t* A;
  const int8_t* W;
  const float* sa;
  const float* sw;
  const float* bias;
  void* out;
  const void* resid;
  void* resid_out;
  const float* gate_table;
  const void* gate_mod;
  int64_t lda, ldw, ldo, ldr, ldro, gate_stride;
  int M, N, K, rows_per_batch;
};

ECAD_DEV i32x4 mfma_i8(const Pack8& a, const Pack8& b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a.u), __builtin_bit_cast(i32x4, b.u), c, 0, 0, 0);
}

// 16 bytes per lane from base + off (32-bit lane offsets, uniform base) to LDS at lds_off + 16 lane.  In asm, as glds16_raw: the kernel owns the waits.
ECAD_DEV void lds_dma16(const void* base, unsigned off, unsigned lds_off) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0" : "=&s"(keep) : "v"(off), "s"(base), "s"(lds_off) : "memory");
}

// keeps the first n bytes of a 16-byte piece
ECAD_DEV void keep_bytes(Pack8& p, int n) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int left = n - 4 * d;
    p.u[d] = left >= 4 ? p.u[d] : (left <= 0 ? 0u : p.u[d] & ((1u << (8 * left)) - 1u));
  }
}

// The fp32 value before its rounding to the storage type, in every kernel the same: without the pin the compiler may fuse the last fma with the conversion
// (v_fma_mixlo_f16, one rounding instead of two) in one kernel and not in another.
ECAD_DEV float pinned(float v) {
  asm("" : "+v"(v));
  return v;
}
// XCD-aware order: workgroups b, b + 8, ... share an XCD and get a run of neighbouring tiles, walked in strips of four tile rows, so that the tiles in flight on one
// L2 share their A and W rows
ECAD_DEV void int8_tile_of(int bid, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int total = tiles_m * tiles_n;
  const int q = total >> 3, r = total & 7, xcd = bid & 7, idx = bid >> 3;
  bid = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
  const int strip = bid / (4 * tiles_n), in = bid - strip * 4 * tiles_n;
  const int rows = tiles_m - 4 * strip < 4 ? tiles_m - 4 * strip : 4;
  tn = in / rows;
  tm = 4 * strip + in - tn * rows;
}

template <int EPI> ECAD_DEV float int8_act(float v) {
  v = pinned(v);
  if constexpr (EPI == I8_GELU) v = pinned(gelu_tanh(v));
  if constexpr (EPI == I8_SILU) v = pinned(silu(v));
  return v;
}

// Epilogue of a tile from its accumulators: lane (l15, g) of a wave holds row m = 16 i + l15, columns 16 j + 4 g .. + 3 of fragment (i, j) of the wave's block at
// (wm0, wn0) of the tile.
// holds: this wave has sums (the others of a tile that is split along K help to write it out).
//   Whole tiles of 16-byte rows without a residual leave straight from the registers: two neighbouring fragments swap halves between lane rows, so a lane ends with
//   eight consecutive columns -- one 16-byte store per pair, 64 contiguous bytes of each of 16 rows -- and LDS stays free.
//   Everything else goes through a row-major tile in LDS (the ring is done with) and leaves in a rolled loop of 16-byte pieces of rows: the residual's reads are
//   contiguous, and edges need one piece of code instead of one per fragment.  (The accumulators can only be named by constants, so whatever stands beside them is
//   unrolled 64 times: with the edges in there the kernel was 250 KB of code and spent 30 us of a 37 us one-round launch fetching it.)
template <typename T, int BM, int BN, int FM, int FN, int NT, int EPI, typename AccFn>
ECAD_DEV void int8_epilogue(const Int8GemmArgs& p, char* smem, int m0, int n0, int wm0, int wn0, bool holds, AccFn&& acc) {
  constexpr int CS = BN + 8;  // row stride of the tile in LDS: 16-byte rows, four banks apart
  const int lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4;
  const bool direct = EPI != I8_RESID && m0 + BM <= p.M && n0 + BN <= p.N && p.ldo % 8 == 0 && ((uintptr_t)p.out & 15) == 0;
  float sa[FM];
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = m0 + wm0 + 16 * i + l15;
    sa[i] = p.sa[m < p.M ? m : p.M - 1];
  }
  auto columns = [&](const float* v, int n) {
    if (n + 3 < p.N) return reinterpret_cast<const Floats4*>(v + n)->f;
    f32x4 f = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 3; ++r)
      if (n + r < p.N) f[r] = v[n + r];
    return f;
  };
  auto packed = [&](auto ic, auto jc, const f32x4& sw, const f32x4& bias) {
    const i32x4 a = acc(ic, jc);
    float o[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = int8_act<EPI>(__builtin_fmaf((float)a[r] * sa[decltype(ic)::value], sw[r], bias[r]));
    return (u32x2){pack2<T>(o[0], o[1]), pack2<T>(o[2], o[3])};
  };
  if (direct) {
    if (!holds) return;
    T* row = reinterpret_cast<T*>(p.out) + (int64_t)(m0 + wm0 + l15) * p.ldo + n0 + wn0;
    static_for<(FN + 1) / 2>([&](auto jh) {
      constexpr int j = 2 * decltype(jh)::value, j1 = j + 1 < FN ? j + 1 : j;
      const int n = n0 + wn0 + 16 * j + 4 * g;
      const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
      const f32x4 sw0 = columns(p.sw, n), b0 = p.bias ? columns(p.bias, n) : zero;
      const f32x4 sw1 = columns(p.sw, n + 16 * (j1 - j)), b1 = p.bias ? columns(p.bias, n + 16 * (j1 - j)) : zero;
      static_for<FM>([&](auto ic) {
        T* at = row + (int64_t)(16 * decltype(ic)::value) * p.ldo + 16 * j;
        const u32x2 lo = packed(ic, std::integral_constant<int, j>{}, sw0, b0);
        if constexpr (j1 > j) {
          const u32x2 hi = packed(ic, std::integral_constant<int, j1>{}, sw1, b1);
          unsigned a0 = lo[0], a1 = lo[1], c0 = hi[0], c1 = hi[1];
          swap_rows16(a0, c0);
          swap_rows16(a1, c1);
          *reinterpret_cast<u32x4*>(at + 16 * (g & 1) + 8 * (g >> 1)) = (u32x4){a0, a1, c0, c1};
        } else {
          *reinterpret_cast<u32x2*>(at + 4 * g) = lo;
        }
      });
    });
    return;
  }
  // the rolled loop in batches of U pieces a thread: a batch's residual and gates are requested before the batch in front of it is worked on, the first one before
  // the sums are staged (one piece at a time each read was waited for behind the write of the piece before: 8192 x 1152 x 4608 52.5 us)
  constexpr int CPR = BN / 8, PIECES = BM * CPR / NT, U = PIECES % 6 == 0 ? 6 : (PIECES % 4 == 0 ? 4 : PIECES);
  static_assert(BM * CPR % NT == 0 && PIECES % U == 0, "whole batches");
  struct Batch {
    Pack8 h[U], gm[U];
    float gt[U][8];
  };
  auto where = [&](int b, int u, int& r, int& c) {
    const int it = (b * U + u) * NT + (int)threadIdx.x;
    r = it / CPR, c = (it - r * CPR) * 8;
  };
  auto request = [&](int b, Batch& x) {
    if constexpr (EPI == I8_RESID) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        int r, c;
        where(b, u, r, c);
        const int m = m0 + r, n = n0 + c, left = p.N - n;
        if (m >= p.M || left <= 0) continue;
        x.h[u] = load_piece<T>(reinterpret_cast<const T*>(p.resid) + (int64_t)m * p.ldr + n, left);
        if (p.gate_table) load_floats(p.gate_table + n, left, x.gt[u]);
        if (p.gate_mod) x.gm[u] = load_piece<T>(reinterpret_cast<const T*>(p.gate_mod) + (int64_t)(m / p.rows_per_batch) * p.gate_stride + n, left);
      }
    }
  };
  T* tile = reinterpret_cast<T*>(smem);
  Batch batch;
  request(0, batch);
  if (holds) static_for<FN>([&](auto jc) {
    constexpr int j = decltype(jc)::value;
    const int n = n0 + wn0 + 16 * j + 4 * g;
    const f32x4 sw = columns(p.sw, n), bias = p.bias ? columns(p.bias, n) : (f32x4){0.f, 0.f, 0.f, 0.f};
    static_for<FM>([&](auto ic) { *reinterpret_cast<u32x2*>(tile + (wm0 + 16 * decltype(ic)::value + l15) * CS + wn0 + 16 * j + 4 * g) = packed(ic, jc, sw, bias); });
  });
  __syncthreads();
  for (int b = 0; b < PIECES / U; ++b) {
    const Batch now = batch;
    if (b + 1 < PIECES / U) request(b + 1, batch);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      int r, c;
      where(b, u, r, c);
      const int m = m0 + r, n = n0 + c, left = p.N - n;
      if (m >= p.M || left <= 0) continue;
      const Pack8 v = lds_read16(tile + r * CS + c);
      if (EPI != I8_RESID || p.out) store_piece<T>(reinterpret_cast<T*>(p.out) + (int64_t)m * p.ldo + n, v, left);
      if constexpr (EPI == I8_RESID) {
        float o[8], h[8], gm[8];
        unpack8<T>(v, o);
        unpack8<T>(now.h[u], h);
        unpack8<T>(now.gm[u], gm);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float gate = p.gate_table ? now.gt[u][e] : (p.gate_mod ? 0.f : 1.f);
          if (p.gate_mod) gate += gm[e];
          h[e] = pinned(__builtin_fmaf(gate, o[e], h[e]));
        }
        store_piece<T>(reinterpret_cast<T*>(p.resid_out) + (int64_t)m * p.ldro + n, pack8<T>(h), left);
      }
    }
  }
}
constexpr int int8_lds_bytes(int bm, int bn, int stages) {
  const int ring = stages * (bm + bn) * 128, tile = bm * (bn + 8) * 2;
  return ring > tile ? ring : tile;
}

// BM x BN tile on WM x WN waves, KW such groups along K.  A step is 128 bytes of K per row for every group: pieces of eight rows (1 KiB) travel straight to LDS, 16-byte
// chunks XOR-swizzled by (row >> 1) & 7 on the source side, so that the fragment reads (16 rows x 16 bytes) meet every bank once.  One barrier per step, STAGES steps in
// a ring.  KW > 1 is for products of few tiles, whose time is the number of steps: the groups' sums meet in LDS (whole numbers: the same bits).
// Bound by the latency of a step where tiles are few (601 x 1111 x 4001: 180 tiles, 16 steps of two, 12.0 us, 13.1 with SiLU; 1024 x 1152 x 1152: 8.0 us), by the LDS pieces'
// issue where they are many (8192 x 4608 x 1152: 67 us on 128 x 128 tiles, 1290 TOP/s; the wide kernels below take those).  One workgroup walks all of K for its tile: 512 x 1152
// x 4608 is 144 of them on 256 CUs (11.9 us of 2.3), 64 x 4096 x 8192 64 (18.5 of 6.5).
template <typename T, int BM, int BN, int WM, int WN, int KW, int STAGES, int EPI>
__global__ __launch_bounds__(WM * WN * KW * 64, 2) void gemm_int8_kernel(const Int8GemmArgs p) {
  constexpr int NG = WM * WN, NW = NG * KW, FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr int A_BYTES = BM * 128, GROUP_BYTES = (BM + BN) * 128, STAGE_BYTES = KW * GROUP_BYTES;
  constexpr int PPG = (BM + BN) / 8, PPW = KW * PPG / NW;  // pieces per group and step, per wave
  static_assert(KW * PPG % NW == 0, "whole pieces per wave");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kg = wave / NG, wm = wave % NG % WM, wn = wave % NG / WM;
  const int l15 = lane & 15, g = lane >> 4;
  int tm, tn;
  int8_tile_of(blockIdx.x, (p.M + BM - 1) / BM, (p.N + BN - 1) / BN, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const char* a_tile = reinterpret_cast<const char*>(p.A) + (int64_t)m0 * p.lda;
  const char* w_tile = reinterpret_cast<const char*>(p.W) + (int64_t)n0 * p.ldw;
  const unsigned lds = __builtin_amdgcn_readfirstlane(lds_offset(smem));

  unsigned row_off[PPW], chunk[PPW], dst[PPW];  // lane offset of the row; of its 16-byte chunk within the step; LDS place of the piece
  const char* base[PPW];
#pragma unroll
  for (int i = 0; i < PPW; ++i) {
    const int at = wave * PPW + i, group = at / PPG, piece = at % PPG;
    const bool of_a = piece < BM / 8;
    const int r = (of_a ? piece : piece - BM / 8) * 8 + (lane >> 3);
    const int rows = of_a ? p.M - m0 : p.N - n0;
    row_off[i] = (unsigned)(r < rows ? r : rows - 1) * (unsigned)(of_a ? p.lda : p.ldw);
    chunk[i] = (unsigned)(group * 128) + (unsigned)(((lane & 7) ^ ((r >> 1) & 7)) * 16);
    dst[i] = __builtin_amdgcn_readfirstlane(at * 1024);
    base[i] = of_a ? a_tile : w_tile;
  }
  const int nk = (p.K + 128 * KW - 1) / (128 * KW);
  auto issue = [&](int kt, int slot) {  // chunks behind the end of K read the start of their row instead (masked below)
#pragma unroll
    for (int i = 0; i < PPW; ++i) {
      const unsigned k = (unsigned)kt * (128 * KW) + chunk[i];
      lds_dma16(base[i], row_off[i] + (k < (unsigned)p.K ? k : 0u), lds + slot * STAGE_BYTES + dst[i]);
    }
  };

  i32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = (i32x4){0, 0, 0, 0};
  const int swz = (l15 >> 1) & 7;
  const int a_row = kg * GROUP_BYTES + (wm * (BM / WM) + l15) * 128, w_row = kg * GROUP_BYTES + A_BYTES + (wn * (BN / WN) + l15) * 128;
  auto step = [&](int slot, int left, auto last) {
    const char* st = smem + slot * STAGE_BYTES;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      Pack8 af[FM], wf[FN];
      const int at = ((4 * s + g) ^ swz) * 16;
#pragma unroll
      for (int i = 0; i < FM; ++i) af[i] = lds_read16(st + a_row + i * 2048 + at);
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        wf[j] = lds_read16(st + w_row + j * 2048 + at);
        if constexpr (decltype(last)::value) keep_bytes(wf[j], left - (4 * s + g) * 16);
      }
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int i = 0; i < FM; ++i) acc[i][j] = mfma_i8(wf[j], af[i], acc[i][j]);
    }
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
    if (s < nk) issue(s, s);
  int slot = 0;
  for (int kt = 0; kt < nk; ++kt) {
    // this wave's pieces of step kt have landed (later ones may be in flight), its reads of the slot that is filled next are done; the barrier says so for all waves
    if (STAGES > 2 && kt + STAGES - 2 < nk) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(PPW * (STAGES - 2)) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (kt + STAGES - 1 < nk) issue(kt + STAGES - 1, slot == 0 ? STAGES - 1 : slot - 1);
    const int left = p.K - (kt * KW + kg) * 128;
    if (left >= 128) step(slot, left, std::false_type{});
    else step(slot, left, std::true_type{});
    slot = slot + 1 == STAGES ? 0 : slot + 1;
  }
  __syncthreads();
  if constexpr (KW > 1) {  // the other groups' sums to the first one
    i32x4* part = reinterpret_cast<i32x4*>(smem) + (wave % NG) * 64 + lane;
    constexpr int FRAGS = FM * FN;
    if (kg > 0) {
#pragma unroll
      for (int f = 0; f < FRAGS; ++f) part[((kg - 1) * FRAGS + f) * NG * 64] = acc[f / FN][f % FN];
    }
    __syncthreads();
    if (kg == 0) {
#pragma unroll
      for (int f = 0; f < FRAGS; ++f)
#pragma unroll
        for (int k = 0; k < KW - 1; ++k) acc[f / FN][f % FN] += part[(k * FRAGS + f) * NG * 64];
    }
    __syncthreads();
  }
  int8_epilogue<T, BM, BN, FM, FN, NW * 64, EPI>(p, smem, m0, n0, wm * (BM / WM), wn * (BN / WN), kg == 0, [&](auto ic, auto jc) -> i32x4 { return acc[decltype(ic)::value][decltype(jc)::value]; });
}

// The same product on one wave per SIMD, 256 x BN tiles on four waves: the K loop over whole stages is one hand-placed asm statement (gemm_int8_asm.h, generated by
// scripts/gen_gemm_i8.py) that leaves the accumulators in AGPRs.  hipcc knows those only as clobbers of the statement: everything that touches them afterwards is asm
// too, and the build fails if the compiler uses one before the last is read (scripts/audit_agpr.py).
// As the clock allows: 8192 x 8192 x 4096 209 to 241 us (2280 to 2630 TOP/s; a library's 8192^3: 2330); 8192 x 1152 x 4608 41 to 47 us (1850 to 2110), 56 with the gated
// residual; 8192 x 4608 x 1152 56 to 63 us (1370 to 1560), 61 with GELU; 4096 x 3456 x 1152 23.4 to 25.9 us (1260 to 1390).  Bound by the stream of operands into LDS: a piece
// holds its wave 60 to 180 cycles, and a stage of the 256 x 144 tile takes 1 us with 0.5 us of matrix instructions in it (their pipe is busy 36 % of a CU's cycles at K 1152, 40 %
// at 4608); then by what every round of tiles has to itself, one workgroup being on a CU: the ring's fill and the epilogue.  8192 x 4608 x 1152 is 512 tiles of 256 x 288, two
// rounds of nine stages; by the constants of choose_int8 8 us of a round's 25 are outside its K loop.  8192 x 1152 x 4608 is 256 tiles of 256 x 144, one round.
template <int BN> struct Int8Wide {
  static constexpr bool tall = BN == 144;                      // waves stacked 4 x 1 (64 x 144 each), else 2 x 2 (128 x BN / 2)
  static constexpr int FM = tall ? 4 : 8, FN = tall ? 9 : BN / 32, stages = tall ? 3 : 2;
  static constexpr int fewest = tall ? GEMM_I8_PERIOD_144 : (BN == 256 ? GEMM_I8_PERIOD_256 : GEMM_I8_PERIOD_288);  // stages
  static constexpr bool ninth = BN == 288;                     // the ninth column of fragments in registers of the caller
  static constexpr int agpr(int i, int j) { return 4 * ((tall ? 9 : 8) * i + j); }
};

template <int R> ECAD_DEV i32x4 agpr_read() {
  i32x4 v;
  asm volatile("v_accvgpr_read_b32 %0, a%c4\n\tv_accvgpr_read_b32 %1, a%c5\n\tv_accvgpr_read_b32 %2, a%c6\n\tv_accvgpr_read_b32 %3, a%c7"
               : "=v"(v[0]), "=v"(v[1]), "=v"(v[2]), "=v"(v[3])
               : "i"(R), "i"(R + 1), "i"(R + 2), "i"(R + 3));
  return v;
}
template <int R> ECAD_DEV void agpr_mfma(const Pack8& w, const Pack8& a) {
  asm volatile("v_mfma_i32_16x16x64_i8 a[%c2:%c3], %0, %1, a[%c2:%c3]" : : "v"(w.u), "v"(a.u), "i"(R), "i"(R + 3));
}

ECAD_DEV void vgpr_mfma(i32x4& c, const Pack8& w, const Pack8& a) { asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+v"(c) : "v"(w.u), "v"(a.u)); }
ECAD_DEV void settle(Pack8& p) { asm volatile("s_nop 4" : "+v"(p.u)); }  // between a vector write and an asm statement that multiplies with it

template <typename T, int BN, int EPI>
__global__ __launch_bounds__(256) void gemm_int8_wide_kernel(const Int8GemmArgs p) {
  typedef Int8Wide<BN> G;
  constexpr int BM = 256, FM = G::FM, FN = G::FN;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4;
  const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm0 = G::tall ? 64 * wave : 128 * (wave & 1), wn0 = G::tall ? 0 : BN / 2 * (wave >> 1);
  int tm, tn;
  int8_tile_of(blockIdx.x, (p.M + BM - 1) / BM, (p.N + BN - 1) / BN, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const int8_t* ap = p.A + (int64_t)m0 * p.lda;
  const int8_t* wp = p.W + (int64_t)n0 * p.ldw;
  const unsigned ra = p.M - m0 < BM ? p.M - m0 - 1 : BM - 1, rw = p.N - n0 < BN ? p.N - n0 - 1 : BN - 1;
  i32x4 c8[8];
  if constexpr (G::ninth) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c8[i] = (i32x4){0, 0, 0, 0};
  }
  {
    const unsigned stages = (unsigned)p.K >> 7, rsa = (unsigned)p.lda, rsw = (unsigned)p.ldw, lds = __builtin_amdgcn_readfirstlane(lds_offset(smem)), zero = 1;
    const unsigned trips = stages / G::fewest - 1, rem = stages % G::fewest;
    if constexpr (BN == 256) { GEMM_I8_ASM_256(ap, wp, rsa, rsw, ra, rw, trips, rem, lds, wave, zero); }
    else if constexpr (BN == 144) { GEMM_I8_ASM_144(ap, wp, rsa, rsw, ra, rw, trips, rem, lds, wave, zero); }
    else { GEMM_I8_ASM_288(ap, wp, rsa, rsw, ra, rw, trips, rem, lds, wave, zero, c8); }
  }
  if (p.K & 127) {  // K behind the last whole stage: fragments straight from memory (a wave's own rows and columns), two matrix instructions per accumulator
    const int k0 = p.K & ~127;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      Pack8 a[FM], w[FN];
      const int k = k0 + 64 * s + 16 * g, left = p.K - k;
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const unsigned r = wm0 + 16 * i + l15;
        a[i].u = (u32x4){0, 0, 0, 0};
        if (left > 0) a[i] = gload16(ap + (int64_t)(r < ra ? r : ra) * p.lda + k);
      }
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const unsigned r = wn0 + 16 * j + l15;
        w[j].u = (u32x4){0, 0, 0, 0};
        if (left > 0) w[j] = gload16(wp + (int64_t)(r < rw ? r : rw) * p.ldw + k);
        keep_bytes(w[j], left);
      }
      static_for<FN>([&](auto jc) {
        settle(w[decltype(jc)::value]);
        static_for<FM>([&](auto ic) {
          constexpr int i = decltype(ic)::value, j = decltype(jc)::value;
          if constexpr (j < 8 || G::tall) agpr_mfma<G::agpr(i, j)>(w[j], a[i]);
          else vgpr_mfma(c8[i], w[j], a[i]);
        });
      });
    }
    // and the accumulators are read next, the ninth column's by ordinary instructions: tied to the wait by the operands
    if constexpr (G::ninth)
      asm volatile("s_nop 15\n\ts_nop 7" : "+v"(c8[0]), "+v"(c8[1]), "+v"(c8[2]), "+v"(c8[3]), "+v"(c8[4]), "+v"(c8[5]), "+v"(c8[6]), "+v"(c8[7]));
    else
      asm volatile("s_nop 15\n\ts_nop 7");
  }
  int8_epilogue<T, BM, BN, FM, FN, 256, EPI>(p, smem, m0, n0, wm0, wn0, true, [&](auto ic, auto jc) -> i32x4 {
    constexpr int i = decltype(ic)::value, j = decltype(jc)::value;
    if constexpr (j < 8 || G::tall) return agpr_read<G::agpr(i, j)>();
    else return c8[i];
  });
}

// Few rows (M <= 16 FM): the time is the reading of W.  A workgroup owns 16 columns; its waves take turns along K in steps of 64 bytes per row, operands go
// straight to registers in the matrix instruction's layout (each W byte is used by one wave only: nothing to share through LDS), several steps in flight; the waves'
// sums meet in LDS.  8 x 6912 x 1152 (8 MB) 4.5 us, 8 x 4096 x 8192 (33.5 MB) 9.4 us: 3.6 TB/s with the launch and the first loads' latency in it.  Narrow weights are
// bound by the CUs that have no columns: 1152 are 72 workgroups on 256 CUs, 5.3 MB in 5.7 to 6.5 us at 8 rows and 8.1 to 8.9 at 32.
template <typename T, int FM, int NW, int EPI>
__global__ __launch_bounds__(NW * 64) void gemm_int8_rows_kernel(const Int8GemmArgs p) {
  __shared__ int part[NW][FM * 256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int8_t* wp = p.W + (int64_t)(n0 + l15 < p.N ? n0 + l15 : p.N - 1) * p.ldw;
  const int8_t* ap[FM];
#pragma unroll
  for (int i = 0; i < FM; ++i) ap[i] = p.A + (int64_t)(16 * i + l15 < p.M ? 16 * i + l15 : p.M - 1) * p.lda;
  i32x4 acc[FM];
#pragma unroll
  for (int i = 0; i < FM; ++i) acc[i] = (i32x4){0, 0, 0, 0};
  constexpr int U = 4;
  int k = wave * 64 + 16 * g;  // this lane's first byte; the wave's steps lie NW * 64 apart
  for (; k - 16 * g + (U - 1) * NW * 64 + 64 <= p.K; k += U * NW * 64) {
    Pack8 w[U], a[U][FM];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w[u] = gload16(wp + k + u * NW * 64);
#pragma unroll
      for (int i = 0; i < FM; ++i) a[u][i] = gload16(ap[i] + k + u * NW * 64);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < FM; ++i) acc[i] = mfma_i8(w[u], a[u][i], acc[i]);
  }
  for (; k - 16 * g < p.K; k += NW * 64) {
    Pack8 w, a[FM];
    w.u = (u32x4){0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < FM; ++i) a[i].u = (u32x4){0, 0, 0, 0};
    if (k < p.K) {
      w = gload16(wp + k);
      keep_bytes(w, p.K - k);
#pragma unroll
      for (int i = 0; i < FM; ++i) a[i] = gload16(ap[i] + k);
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) acc[i] = mfma_i8(w, a[i], acc[i]);
  }
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) part[wave][i * 256 + l15 * 16 + 4 * g + r] = acc[i][r];
  __syncthreads();
  for (int it = threadIdx.x; it < FM * 256; it += NW * 64) {
    const int m = it >> 4, n = n0 + (it & 15);
    if (m >= p.M || n >= p.N) continue;
    int sum = part[0][it];
#pragma unroll
    for (int w = 1; w < NW; ++w) sum += part[w][it];
    const float o = int8_act<EPI>(__builtin_fmaf((float)sum * p.sa[m], p.sw[n], p.bias ? p.bias[n] : 0.f));
    const float rounded = round_elem<T>(o);
    if (EPI != I8_RESID || p.out) reinterpret_cast<T*>(p.out)[(int64_t)m * p.ldo + n] = (T)o;
    if constexpr (EPI == I8_RESID) {
      float gate = p.gate_table ? p.gate_table[n] : (p.gate_mod ? 0.f : 1.f);
      if (p.gate_mod) gate += (float)reinterpret_cast<const T*>(p.gate_mod)[(int64_t)(m / p.rows_per_batch) * p.gate_stride + n];
      reinterpret_cast<T*>(p.resid_out)[(int64_t)m * p.ldro + n] = (T)pinned(__builtin_fmaf(gate, rounded, (float)reinterpret_cast<const T*>(p.resid)[(int64_t)m * p.ldr + n]));
    }
  }
}

}  // namespace ecad
