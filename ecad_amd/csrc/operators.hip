// operators.hip -- the single-op entry points of an 8-bit transformer block (operators.h): argument checks and launches of row_ops.h, gate_norm.h, rope.h and
// gemm_int8.h.  A unit of its own, compiled without -ffast-math: the 8-bit rounding needs the divisions and remainders it writes down.
#include "operators.h"

#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include <atomic>

#include "gate_norm.h"
#include "gemm_int8.h"
#include "rope.h"

namespace ecad {
namespace {

int refuse(OpStatus& st, int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(st.msg, sizeof st.msg, fmt, ap);
  va_end(ap);
  return code;
}

int launched(OpStatus& st, const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? ECAD_OK : refuse(st, ECAD_E_HIP, "%s: launch failed: %s", what, hipGetErrorString(e));
}

// threads of a launch are counted in 32 bits
bool fits(int64_t blocks, int threads) { return blocks <= 0x7fffffff && blocks * threads <= 0xffffffffll; }

bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// more than 64 KiB of LDS has to be asked for once per kernel and device
int allow_lds(std::atomic<uint64_t>& done, const void* kernel, int bytes, OpStatus& st) {
  int dev = 0;
  if (bytes <= 65536) return ECAD_OK;
  if (hipGetDevice(&dev) == hipSuccess && dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return ECAD_OK;
  const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return refuse(st, ECAD_E_HIP, "LDS of %d bytes refused: %s", bytes, hipGetErrorString(e));
  if (dev < 64) done.fetch_or((uint64_t)1 << dev, std::memory_order_relaxed);
  return ECAD_OK;
}

// ---- memory that an argument covers: sizes and strides (bytes), outermost first, the elements of the last dimension dense ----------------------------------------

struct Region {
  const char* p;
  int64_t n[4], step[4];
  int64_t bytes;  // of the dense innermost part
  bool empty() const {
    if (!p || bytes <= 0) return true;
    for (int64_t x : n)
      if (x == 0) return true;
    return false;
  }
  int64_t reach() const {
    int64_t r = bytes;
    for (int i = 0; i < 4; ++i) r += (n[i] - 1) * step[i];
    return r;
  }
};
Region matrix(const void* p, int64_t rows, int64_t width, int64_t stride, int64_t size) { return {(const char*)p, {1, 1, 1, rows}, {0, 0, 0, stride * size}, width * size}; }
Region vector(const void* p, int64_t n, int64_t size) { return matrix(p, 1, n, 0, size); }

// every element of an output has memory of its own
bool distinct(const Region& r) {
  int64_t n[4], step[4];
  int d = 0;
  for (int i = 0; i < 4; ++i)
    if (r.n[i] > 1) {  // insertion by stride
      int j = d++;
      for (; j > 0 && step[j - 1] > r.step[i]; --j) n[j] = n[j - 1], step[j] = step[j - 1];
      n[j] = r.n[i], step[j] = r.step[i];
    }
  int64_t need = r.bytes;
  for (int i = 0; i < d; ++i) {
    if (step[i] < need) return false;
    need += step[i] * (n[i] - 1);
  }
  return true;
}

// Whether two regions may share memory.  Where all the strides of both that are not inside a row are multiples of that row's length (columns of one buffer), the
// bytes that each takes of the row decide.
bool meet(const Region& a, const Region& b) {
  if (a.empty() || b.empty() || a.p + a.reach() <= b.p || b.p + b.reach() <= a.p) return false;
  for (int i = 0; i < 4; ++i) {
    const int64_t row = a.step[i];
    if (a.n[i] < 2 || row <= 0) continue;
    auto inner = [&](const Region& r) {
      int64_t x = r.bytes;
      for (int j = 0; j < 4; ++j)
        if (r.n[j] > 1 && r.step[j] % row) x += (r.n[j] - 1) * r.step[j];
      return x;
    };
    const int64_t gap = ((b.p - a.p) % row + row) % row;
    if (gap >= inner(a) && gap + inner(b) <= row) return false;
  }
  return true;
}

template <size_t N> bool meets_any(const Region& out, const Region (&others)[N]) {
  for (const Region& r : others)
    if (meet(out, r)) return true;
  return false;
}

constexpr int MAX_ROW = 32768;       // widest row that the norms hold in registers (1024 lanes x 4 pieces)
constexpr int MAX_INT8_K = 131071;   // 128^2 K stays below 2^31

// ---- 8-bit rows ----------------------------------------------------------------------------------------------------------------------------------------------

template <typename T, int WAVES, int CH> int launch_quantize(const OpCtx& ctx, const QuantizeArgs& whole, OpStatus& st) {
  constexpr int slots = row_slots(WAVES), threads = WAVES == 1 ? 256 : WAVES * 64;
  constexpr int64_t most = 0xffffffffll / threads * slots < 0x7fffffff ? 0xffffffffll / threads * slots : 0x7fffffff;  // rows of one launch
  for (int64_t row = 0; row < whole.M; row += most) {
    QuantizeArgs a = whole;
    a.x = reinterpret_cast<const T*>(whole.x) + row * whole.ldx;
    a.q += row * whole.ldq;
    a.scale += row;
    a.M = (int)(whole.M - row < most ? whole.M - row : most);
    const dim3 grid((unsigned)(((int64_t)a.M + slots - 1) / slots));
    if (a.K % 8) hipLaunchKernelGGL((quantize_rows_kernel<T, WAVES, CH, true>), grid, dim3(threads), 0, ctx.stream, a);
    else hipLaunchKernelGGL((quantize_rows_kernel<T, WAVES, CH, false>), grid, dim3(threads), 0, ctx.stream, a);
  }
  return launched(st, "quantize_int8");
}
template <typename T> int quantize_t(const OpCtx& ctx, const QuantizeArgs& a, OpStatus& st) {
  const int pieces = (a.K + 7) / 8;
  if (pieces <= 64) return launch_quantize<T, 1, 1>(ctx, a, st);
  if (pieces <= 128) return launch_quantize<T, 1, 2>(ctx, a, st);
  if (pieces <= 192) return launch_quantize<T, 1, 3>(ctx, a, st);
  if (pieces <= 256) return launch_quantize<T, 4, 1>(ctx, a, st);
  if (pieces <= 512) return launch_quantize<T, 4, 2>(ctx, a, st);
  if (pieces <= 768) return launch_quantize<T, 4, 3>(ctx, a, st);
  if (pieces <= 1024) return launch_quantize<T, 4, 4>(ctx, a, st);
  if (pieces <= 2048) return launch_quantize<T, 8, 4>(ctx, a, st);
  if (pieces <= 4096) return launch_quantize<T, 16, 4>(ctx, a, st);
  return launch_quantize<T, 16, 16>(ctx, a, st);
}

// ---- norms ---------------------------------------------------------------------------------------------------------------------------------------------------

template <typename T, int WAVES, int CH, bool HOLD = true> int launch_norm(const OpCtx& ctx, GateNormArgs& a, int per_cu, OpStatus& st) {
  // Rows in turn: a lane keeps the channel vectors and has the next row's loads in flight while it works on one.  per_cu: rows that a CU works on at a time (what its
  // registers hold: 115 / 165 / 230 of 512 per lane at one / two / three pieces); every wave gets at least one row.  One wave a row, three pieces: 8 was the
  // best of 4, 8, 12, 16, 24 and 32 at 8192 and 32768 rows of 1152.
  const int slots = row_slots(WAVES);
  const int64_t at_once = (int64_t)ctx.num_cus * per_cu;
  a.rows_per_group = (int)((a.M + at_once - 1) / at_once);
  const dim3 grid((unsigned)(((int64_t)a.M + (int64_t)slots * a.rows_per_group - 1) / ((int64_t)slots * a.rows_per_group))), block(WAVES == 1 ? 256 : WAVES * 64);
  if (a.D % 8) hipLaunchKernelGGL((gate_norm_kernel<T, WAVES, CH, true, HOLD>), grid, block, 0, ctx.stream, a);
  else hipLaunchKernelGGL((gate_norm_kernel<T, WAVES, CH, false, HOLD>), grid, block, 0, ctx.stream, a);
  return launched(st, "gate_norm");
}
template <typename T> int gate_norm_t(const OpCtx& ctx, GateNormArgs& a, OpStatus& st) {
  const int pieces = (a.D + 7) / 8;
  if (pieces <= 64) return launch_norm<T, 1, 1>(ctx, a, 20, st);
  if (pieces <= 128) return launch_norm<T, 2, 1>(ctx, a, 10, st);
  // three waves a row / one: 1152 values 5 rows 4.0 / 5.9 us, 2048 rows 8.1 / 9.3, 4096 rows 13.2 / 12.1, 32768 rows 75 / 55; 1032 values 4.0 / 6.0, 8.3 / 9.5, 13.0 / 12.1,
  // 64 / 62; 1536 values 4.1 / 6.0, 8.5 / 9.7, 13.5 / 12.7, 100 / 86
  if (pieces <= 192) return a.M <= 8 * ctx.num_cus ? launch_norm<T, 3, 1>(ctx, a, 6, st) : launch_norm<T, 1, 3>(ctx, a, 8, st);
  if (pieces <= 256) return launch_norm<T, 4, 1>(ctx, a, 5, st);
  if (pieces <= 512) return launch_norm<T, 8, 1>(ctx, a, 2, st);
  if (pieces <= 1024) return launch_norm<T, 8, 2>(ctx, a, 1, st);
  if (pieces <= 2048) return launch_norm<T, 16, 2, false>(ctx, a, 1, st);
  return launch_norm<T, 16, 4, false>(ctx, a, 1, st);
}

// ---- products ------------------------------------------------------------------------------------------------------------------------------------------------

int64_t tiles_of(const Int8GemmArgs& a, int bm, int bn) { return ((int64_t)a.M + bm - 1) / bm * (((int64_t)a.N + bn - 1) / bn); }

int launch_int8(const OpCtx& ctx, const Int8GemmArgs& a, OpStatus& st, std::atomic<uint64_t>& done, void (*kernel)(const Int8GemmArgs), int bm, int bn, int threads, int bytes) {
  const int rc = allow_lds(done, (const void*)kernel, bytes, st);
  if (rc) return rc;
  const int64_t tiles = tiles_of(a, bm, bn);
  if (!fits(tiles, threads)) return refuse(st, ECAD_E_UNSUPPORTED, "gemm_int8: %lld tiles are more than one launch takes", (long long)tiles);
  hipLaunchKernelGGL(kernel, dim3((unsigned)tiles), dim3(threads), bytes, ctx.stream, a);
  return launched(st, "gemm_int8");
}
template <typename T, int EPI, int BM, int BN, int WM, int WN, int KW, int STAGES> int launch_tile(const OpCtx& ctx, const Int8GemmArgs& a, OpStatus& st) {
  static std::atomic<uint64_t> done{0};
  return launch_int8(ctx, a, st, done, gemm_int8_kernel<T, BM, BN, WM, WN, KW, STAGES, EPI>, BM, BN, WM * WN * KW * 64, int8_lds_bytes(BM, BN, STAGES * KW));
}
template <typename T, int EPI, int BN> int launch_wide(const OpCtx& ctx, const Int8GemmArgs& a, OpStatus& st) {
  static std::atomic<uint64_t> done{0};
  if (a.K / 128 < Int8Wide<BN>::fewest) return refuse(st, ECAD_E_UNSUPPORTED, "gemm_int8: the 256 x %d kernel needs K of at least %d, got %d", BN, Int8Wide<BN>::fewest * 128, a.K);
  return launch_int8(ctx, a, st, done, gemm_int8_wide_kernel<T, BN, EPI>, 256, BN, 256, int8_lds_bytes(256, BN, Int8Wide<BN>::stages));
}

// Which kernel: the one with the smallest estimated time, rounds of the tiles it needs over the chip times (what a round costs outside the K loop + its K stages), in
// microseconds; a stage costs more the fuller the chip is (operands from L2, and the clock under load).  The pick is the fastest kernel at 18 of the 19 shapes of more than
// 32 rows in profiles/operators_kernel_choice.csv (8000 x 500 x 3000: 21 % off).  Some of them, us, plain epilogue:
//                        64 x 64   64 x 64, K over two   128 x 128   256 x 144   256 x 256   256 x 288
//   512 x 4608 x 1152     12.7        15.6                12.3        14.1        17.9        20.5
//   512 x 1152 x 4608     16.8        11.9                31.2        29.4        42.6        45.9
//   601 x 1111 x 4001     16.1        12.0                29.9        32.0        45.3        50.9
//   1024 x 1152 x 1152     8.0        11.7                11.8        13.4        19.3        19.6
//   2048 x 4608 x 1152    32.9        46.7                26.1        18.1        21.3        24.3
//   4096 x 3456 x 1152    48.0        69.8                30.3        31.0        23.4        25.7
//   8000 x 500 x 3000     30.0        35.8                27.0        32.7        48.6        50.8
//   8192 x 4608 x 1152   113.9       171.9                67.4        66.7        66.4        63.4
//   8192 x 1152 x 4608    92.9       102.4                72.9        41.2        51.1        54.9
//   8192 x 8192 x 4096   542         615                 299         269         209         227
int choose_int8(const OpCtx& ctx, const Int8GemmArgs& a) {
  struct Tile {
    int id, bm, bn, per_cu, fewest;
    double round, stage, full, least;  // a stage: stage + full * (share of the chip in use), at least `least`
  };
  static const Tile tiles[] = {{ECAD_I8_K_TILE64, 64, 64, 2, 0, 2.0, 0.42, 0.06, 0},
                               {ECAD_I8_K_TILE64_K2, 64, 64, 1, 0, 2.2, 0.25, 0.06, 0},
                               {ECAD_I8_K_TILE128, 128, 128, 2, 0, 2.6, 0.75, 0.4, 0},
                               {ECAD_I8_K_TILE144, 256, 144, 1, Int8Wide<144>::fewest, 7.0, 0.62, 0.25, 0},
                               {ECAD_I8_K_TILE256, 256, 256, 1, Int8Wide<256>::fewest, 7.0, 0.5, 1.1, 1.1},
                               {ECAD_I8_K_TILE288, 256, 288, 1, Int8Wide<288>::fewest, 8.0, 0.5, 1.35, 1.2}};
  // few-rows kernel / best tile: 32 rows 6912 x 1152 5.8 us / 6.2, 1152 x 4608 8.1 / 11.2, 4096 x 8192 13.3 / 18.2; 64 rows (a form of it that is not kept) 7.6 / 6.2, 12.2 / 11.6,
  // 21.0 / 18.5
  if (a.M <= 32 && fits(((int64_t)a.N + 15) / 16, 1024)) return ECAD_I8_K_ROWS;
  const int stages = (a.K + 127) / 128;
  int best = ECAD_I8_K_TILE64;
  double least = 1e300;
  for (const Tile& t : tiles) {
    const int64_t n = tiles_of(a, t.bm, t.bn);
    if (a.K / 128 < t.fewest || !fits(n, t.id == ECAD_I8_K_TILE64_K2 ? 512 : 256)) continue;
    const int64_t at_once = (int64_t)t.per_cu * ctx.num_cus, rounds = (n + at_once - 1) / at_once;
    const double stage = t.stage + t.full * (double)n / (double)(rounds * at_once);
    const double us = (double)rounds * (t.round + (stage > t.least ? stage : t.least) * stages);
    if (us < least) least = us, best = t.id;
  }
  return best;
}

template <typename T, int EPI> int gemm_int8_t(const OpCtx& ctx, const Int8GemmArgs& a, int kernel, OpStatus& st) {
  if (kernel == ECAD_I8_K_ROWS && a.M > 32) return refuse(st, ECAD_E_UNSUPPORTED, "gemm_int8: the few-rows kernel takes up to 32 rows, got %d", a.M);
  switch (kernel == ECAD_I8_K_AUTO ? choose_int8(ctx, a) : kernel) {
    case ECAD_I8_K_ROWS: {
      const dim3 grid((unsigned)(((int64_t)a.N + 15) / 16));
      if (!fits(grid.x, 1024)) return refuse(st, ECAD_E_UNSUPPORTED, "gemm_int8: %d columns are more than one launch of the few-rows kernel takes", a.N);
      // few workgroups: more of K in flight at a time.  Sixteen waves / eight, 8 rows: 1152 x 4608 5.6 us / 5.7, 4096 x 8192 8.1 / 8.9, 6912 x 1152 4.3 / 4.3; 8208 x 1152 5.0 / 4.6,
      // 16384 x 1152 7.1 / 6.2
      const bool narrow = (int64_t)grid.x < 2 * (int64_t)ctx.num_cus;
      if (a.M <= 16 && narrow) hipLaunchKernelGGL((gemm_int8_rows_kernel<T, 1, 16, EPI>), grid, dim3(1024), 0, ctx.stream, a);
      else if (a.M <= 16) hipLaunchKernelGGL((gemm_int8_rows_kernel<T, 1, 8, EPI>), grid, dim3(512), 0, ctx.stream, a);
      else if (narrow) hipLaunchKernelGGL((gemm_int8_rows_kernel<T, 2, 16, EPI>), grid, dim3(1024), 0, ctx.stream, a);
      else hipLaunchKernelGGL((gemm_int8_rows_kernel<T, 2, 8, EPI>), grid, dim3(512), 0, ctx.stream, a);
      return launched(st, "gemm_int8");
    }
    case ECAD_I8_K_TILE64: return launch_tile<T, EPI, 64, 64, 2, 2, 1, 4>(ctx, a, st);
    case ECAD_I8_K_TILE64_K2: return launch_tile<T, EPI, 64, 64, 2, 2, 2, 4>(ctx, a, st);
    case ECAD_I8_K_TILE128: return launch_tile<T, EPI, 128, 128, 2, 2, 1, 2>(ctx, a, st);
    case ECAD_I8_K_TILE144: return launch_wide<T, EPI, 144>(ctx, a, st);
    case ECAD_I8_K_TILE256: return launch_wide<T, EPI, 256>(ctx, a, st);
    case ECAD_I8_K_TILE288: return launch_wide<T, EPI, 288>(ctx, a, st);
    default: return refuse(st, ECAD_E_INVALID, "gemm_int8: kernel %d unknown", kernel);
  }
}
template <typename T> int gemm_int8_epi(const OpCtx& ctx, const Int8GemmArgs& a, int epi, int kernel, OpStatus& st) {
  switch (epi) {
    case I8_GELU: return gemm_int8_t<T, I8_GELU>(ctx, a, kernel, st);
    case I8_SILU: return gemm_int8_t<T, I8_SILU>(ctx, a, kernel, st);
    case I8_RESID: return gemm_int8_t<T, I8_RESID>(ctx, a, kernel, st);
    default: return gemm_int8_t<T, I8_BIAS>(ctx, a, kernel, st);
  }
}

}  // namespace

int op_num_cus(int device) noexcept {
  static std::atomic<int> known[64];
  if (device >= 0 && device < 64 && known[device].load(std::memory_order_relaxed)) return known[device].load(std::memory_order_relaxed);
  int n = 0;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || n < 1) n = 256;
  if (device >= 0 && device < 64) known[device].store(n, std::memory_order_relaxed);
  return n;
}

int op_quantize_int8(const OpCtx& ctx, const QuantizeCall& c, OpStatus& st) noexcept {
  if (c.M < 0 || c.K < 1 || c.K > MAX_INT8_K) return refuse(st, ECAD_E_INVALID, "quantize_int8: %d rows of %d values (1 to %d values a row)", c.M, c.K, MAX_INT8_K);
  if (c.M == 0) return ECAD_OK;
  if (!c.x || !c.q || !c.scale) return refuse(st, ECAD_E_INVALID, "quantize_int8: NULL pointer");
  if (c.ldx < (c.M > 1 ? c.K : 0) || c.ldq < c.K || c.ldq % 16 || !aligned(c.q, 16) || !aligned(c.x, 2) || !aligned(c.scale, 4))
    return refuse(st, ECAD_E_INVALID, "quantize_int8: x rows need a stride of at least %d, 8-bit rows start on 16 bytes with a stride of a multiple of 16 (got %lld and %lld)", c.K, (long long)c.ldx,
                  (long long)c.ldq);
  const Region x = matrix(c.x, c.M, c.K, c.ldx, 2), q = matrix(c.q, c.M, c.K, c.ldq, 1), scale = vector(c.scale, c.M, 4);
  if (meet(q, x) || meet(q, scale) || meet(scale, x)) return refuse(st, ECAD_E_INVALID, "quantize_int8: an output overlaps another argument");
  const QuantizeArgs a{c.x, c.q, c.scale, c.ldx, c.ldq, c.M, c.K};
  return ctx.dtype == ECAD_DTYPE_F16 ? quantize_t<f16_t>(ctx, a, st) : quantize_t<bf16_t>(ctx, a, st);
}

int op_gemm_int8(const OpCtx& ctx, const EcadInt8Gemm& c, OpStatus& st) noexcept {
  if (c.M < 0 || c.N < 0 || c.K < 1 || c.K > MAX_INT8_K) return refuse(st, ECAD_E_INVALID, "gemm_int8: M=%d N=%d K=%d (K from 1 to %d)", c.M, c.N, c.K, MAX_INT8_K);
  if (c.epi < 0 || c.epi > 3) return refuse(st, ECAD_E_INVALID, "gemm_int8: epilogue %d unknown", c.epi);
  if (c.M == 0 || c.N == 0) return ECAD_OK;
  if (!c.A || !c.W || !c.a_scale || !c.w_scale || (c.epi != I8_RESID && !c.out)) return refuse(st, ECAD_E_INVALID, "gemm_int8: NULL pointer");
  if (c.epi == I8_RESID && (!c.resid || !c.resid_out)) return refuse(st, ECAD_E_INVALID, "gemm_int8: epilogue 3 needs resid");
  if (!aligned(c.A, 16) || !aligned(c.W, 16) || c.lda % 16 || c.ldw % 16 || c.lda < c.K || c.ldw < c.K || c.lda > (1 << 23) || c.ldw > (1 << 23))
    return refuse(st, ECAD_E_INVALID, "gemm_int8: 8-bit rows start on 16 bytes with a stride of a multiple of 16, at least %d (got %lld and %lld)", c.K, (long long)c.lda, (long long)c.ldw);
  if (!aligned(c.a_scale, 4) || !aligned(c.w_scale, 4) || !aligned(c.bias, 4) || !aligned(c.gate_table, 4) || !aligned(c.out, 2) || !aligned(c.resid, 2) || !aligned(c.resid_out, 2) || !aligned(c.gate_mod, 2))
    return refuse(st, ECAD_E_INVALID, "gemm_int8: pointers are not aligned to their type");
  if ((c.out && c.M > 1 && c.ldo < c.N) || (c.epi == I8_RESID && c.M > 1 && (c.ldr < c.N || c.ldro < c.N))) return refuse(st, ECAD_E_INVALID, "gemm_int8: row strides of the outputs are shorter than %d", c.N);
  if (c.epi == I8_RESID && c.rows_per_batch < 1) return refuse(st, ECAD_E_INVALID, "gemm_int8: rows_per_batch must be at least 1");
  const bool gated = c.epi == I8_RESID;
  if (gated && c.gate_mod_stride < 0) return refuse(st, ECAD_E_INVALID, "gemm_int8: a stride is negative");
  const int64_t samples = gated ? ((int64_t)c.M - 1) / c.rows_per_batch + 1 : 0;
  const Region out = matrix(c.out, c.M, c.N, c.ldo, 2), resid_out = matrix(gated ? c.resid_out : nullptr, c.M, c.N, c.ldro, 2), resid = matrix(gated ? c.resid : nullptr, c.M, c.N, c.ldr, 2);
  const Region in[] = {matrix(c.A, c.M, c.K, c.lda, 1), matrix(c.W, c.N, c.K, c.ldw, 1), vector(c.a_scale, c.M, 4), vector(c.w_scale, c.N, 4), vector(c.bias, c.N, 4),
                       vector(gated ? c.gate_table : nullptr, c.N, 4), matrix(gated ? c.gate_mod : nullptr, samples, c.N, c.gate_mod_stride, 2)};
  const bool in_place = gated && c.resid_out == c.resid && (c.ldr == c.ldro || c.M == 1);
  if (meets_any(out, in) || meets_any(resid_out, in) || meet(out, resid) || meet(out, resid_out) || (!in_place && meet(resid_out, resid)))
    return refuse(st, ECAD_E_INVALID, "gemm_int8: an output overlaps another argument");
  Int8GemmArgs a{};
  a.A = c.A; a.W = c.W; a.sa = c.a_scale; a.sw = c.w_scale; a.bias = c.bias; a.out = c.out; a.resid = c.resid; a.resid_out = c.resid_out; a.gate_table = c.gate_table; a.gate_mod = c.gate_mod;
  a.lda = c.lda; a.ldw = c.ldw; a.ldo = c.ldo; a.ldr = c.ldr; a.ldro = c.ldro; a.gate_stride = c.gate_mod_stride;
  a.M = c.M; a.N = c.N; a.K = c.K; a.rows_per_batch = c.rows_per_batch > 0 ? c.rows_per_batch : 1;
  return ctx.dtype == ECAD_DTYPE_F16 ? gemm_int8_epi<f16_t>(ctx, a, c.epi, c.kernel, st) : gemm_int8_epi<bf16_t>(ctx, a, c.epi, c.kernel, st);
}

int op_gate_norm(const OpCtx& ctx, const EcadGateNorm& c, OpStatus& st) noexcept {
  if (c.M < 0 || c.D < 1) return refuse(st, ECAD_E_INVALID, "gate_norm: %d rows of %d values", c.M, c.D);
  if (c.D > MAX_ROW) return refuse(st, ECAD_E_UNSUPPORTED, "gate_norm: rows of up to %d values, got %d", MAX_ROW, c.D);
  if (c.post < NORM_NONE || c.post > NORM_LAYER || c.pre < NORM_NONE || c.pre > NORM_LAYER) return refuse(st, ECAD_E_INVALID, "gate_norm: norm kinds are 0 (none), 1 (rms), 2 (layer)");
  if (!(c.eps >= 0.f) || !(fabsf(c.resid_scale) < INFINITY)) return refuse(st, ECAD_E_INVALID, "gate_norm: eps %g, residual scale %g", (double)c.eps, (double)c.resid_scale);
  if (c.rows_per_batch < 1) return refuse(st, ECAD_E_INVALID, "gate_norm: rows_per_batch must be at least 1");
  if (c.pre == NORM_NONE && (c.pre_weight || c.table_shift || c.table_scale || c.mod_shift || c.mod_scale || c.n_out || c.q))
    return refuse(st, ECAD_E_INVALID, "gate_norm: weight, modulation and output of a pre-norm that is 'none'");
  if (c.post == NORM_NONE && c.post_weight) return refuse(st, ECAD_E_INVALID, "gate_norm: weight of a post-norm that is 'none'");
  if (c.M == 0) return ECAD_OK;  // an empty y may be NULL: it says nothing about the call
  if (!c.y && (c.post != NORM_NONE || c.post_weight || c.gate_table || c.gate_mod || c.resid_scale != 1.f || c.pre == NORM_NONE))
    return refuse(st, ECAD_E_INVALID, "gate_norm: without y there is no gate, post-norm or residual scale, and the pre-norm is what is left to do");
  if (!c.h || (c.y && !c.h_out) || (c.pre != NORM_NONE && !c.n_out == !c.q) || (c.q && !c.q_scale)) return refuse(st, ECAD_E_INVALID, "gate_norm: NULL pointer, or both n and its 8-bit rows asked for");
  const int64_t least = c.M > 1 ? c.D : 0;
  if (c.ldh < least || (c.y && (c.ldy < least || c.ldho < least)) || (c.n_out && c.ldn < least)) return refuse(st, ECAD_E_INVALID, "gate_norm: a row stride is shorter than %d", c.D);
  if (c.q && (c.ldq < c.D || c.ldq % 16 || !aligned(c.q, 16) || !aligned(c.q_scale, 4))) return refuse(st, ECAD_E_INVALID, "gate_norm: 8-bit rows start on 16 bytes with a stride of a multiple of 16");
  if (!aligned(c.h, 2) || !aligned(c.y, 2) || !aligned(c.h_out, 2) || !aligned(c.n_out, 2) || !aligned(c.gate_mod, 2) || !aligned(c.mod_shift, 2) || !aligned(c.mod_scale, 2) || !aligned(c.post_weight, 4) ||
      !aligned(c.pre_weight, 4) || !aligned(c.gate_table, 4) || !aligned(c.table_shift, 4) || !aligned(c.table_scale, 4))
    return refuse(st, ECAD_E_INVALID, "gate_norm: pointers are not aligned to their type");
  if (c.gate_mod_stride < 0 || c.mod_stride < 0) return refuse(st, ECAD_E_INVALID, "gate_norm: a stride is negative");
  const int64_t samples = ((int64_t)c.M - 1) / c.rows_per_batch + 1;
  const Region h = matrix(c.h, c.M, c.D, c.ldh, 2), y = matrix(c.y, c.M, c.D, c.ldy, 2), ho = matrix(c.y ? c.h_out : nullptr, c.M, c.D, c.ldho, 2), no = matrix(c.n_out, c.M, c.D, c.ldn, 2),
               q = matrix(c.q, c.M, c.D, c.ldq, 1), qs = vector(c.q ? c.q_scale : nullptr, c.M, 4);
  const Region in[] = {vector(c.post_weight, c.D, 4), vector(c.pre_weight, c.D, 4), vector(c.gate_table, c.D, 4), vector(c.table_shift, c.D, 4), vector(c.table_scale, c.D, 4),
                       matrix(c.gate_mod, samples, c.D, c.gate_mod_stride, 2), matrix(c.mod_shift, samples, c.D, c.mod_stride, 2), matrix(c.mod_scale, samples, c.D, c.mod_stride, 2)};
  const bool h_same = c.h_out == c.h && (c.ldho == c.ldh || c.M == 1), y_same = c.y && c.n_out == c.y && (c.ldn == c.ldy || c.M == 1);
  const Region outs[] = {ho, no, q, qs};
  bool clash = (!h_same && meet(ho, h)) || meet(ho, y) || meet(no, h) || (!y_same && meet(no, y)) || meet(q, h) || meet(q, y) || meet(qs, h) || meet(qs, y) || meet(ho, no) || meet(ho, q) || meet(ho, qs) ||
               meet(q, qs);
  for (const Region& o : outs) clash = clash || meets_any(o, in);
  if (clash) return refuse(st, ECAD_E_INVALID, "gate_norm: an output overlaps another argument");
  GateNormArgs a{};
  a.h = c.h; a.y = c.y; a.h_out = c.h_out; a.n_out = c.n_out; a.q = c.q; a.q_scale = c.q_scale; a.post_weight = c.post_weight; a.pre_weight = c.pre_weight;
  a.gate_table = c.gate_table; a.table_shift = c.table_shift; a.table_scale = c.table_scale; a.gate_mod = c.gate_mod; a.mod_shift = c.mod_shift; a.mod_scale = c.mod_scale;
  a.ldh = c.ldh; a.ldy = c.ldy; a.ldho = c.ldho; a.ldn = c.ldn; a.ldq = c.ldq; a.gate_stride = c.gate_mod_stride; a.mod_stride = c.mod_stride;
  a.M = c.M; a.D = c.D; a.rows_per_batch = c.rows_per_batch; a.post = c.post; a.pre = c.pre; a.resid_scale = c.resid_scale; a.eps = c.eps;
  return ctx.dtype == ECAD_DTYPE_F16 ? gate_norm_t<f16_t>(ctx, a, st) : gate_norm_t<bf16_t>(ctx, a, st);
}

int op_rope_table(const OpCtx& ctx, const RopeTableCall& c, OpStatus& st) noexcept {
  if (c.axes < 1 || c.axes > ROPE_MAX_AXES || !c.axes_dims || c.S < 0) return refuse(st, ECAD_E_INVALID, "rope_table: %d positions on %d axes (1 to %d)", c.S, c.axes, ROPE_MAX_AXES);
  RopeTableArgs a{};
  const double two_pi = 6.283185307179586476925;
  if (!(c.theta > 0) || c.theta == INFINITY || !(c.factor > 0) || c.factor == INFINITY) return refuse(st, ECAD_E_INVALID, "rope_table: theta %g and factor %g must be positive", c.theta, c.factor);
  if (c.scaling < ECAD_ROPE_NONE || c.scaling > ECAD_ROPE_YARN) return refuse(st, ECAD_E_INVALID, "rope_table: scaling %d unknown", c.scaling);
  if (c.scaling == ECAD_ROPE_YARN && (!(c.original_length > 0) || !(c.beta_fast > c.beta_slow) || !(c.factor >= 1)))
    return refuse(st, ECAD_E_INVALID, "rope_table: yarn needs an original length, beta_fast > beta_slow and a factor of at least 1");
  for (int x = 0; x < c.axes; ++x) {
    const int d = c.axes_dims[x];
    if (d < 2 || d % 2 || a.pairs + d / 2 > ROPE_MAX_PAIRS) return refuse(st, ECAD_E_INVALID, "rope_table: axis %d has %d elements (even, at least 2, at most %d over all axes)", x, d, 2 * ROPE_MAX_PAIRS);
    const double theta = c.scaling == ECAD_ROPE_NTK && d > 2 ? c.theta * pow(c.factor, (double)d / (d - 2)) : c.theta;
    for (int j = 0; j < d / 2; ++j) {
      double f = pow(theta, -2.0 * j / d);
      if (c.scaling == ECAD_ROPE_LINEAR) f /= c.factor;
      if (c.scaling == ECAD_ROPE_YARN) {
        double keep = (c.original_length * f / two_pi - c.beta_slow) / (c.beta_fast - c.beta_slow);
        keep = keep < 0 ? 0 : (keep > 1 ? 1 : keep);
        f = f * keep + f / c.factor * (1 - keep);
      }
      a.quarters[a.pairs] = 4.0 * f / two_pi;
      a.axis[a.pairs++] = (unsigned char)x;
    }
  }
  if (c.S == 0) return ECAD_OK;
  if (!c.positions || !c.table || !aligned(c.positions, 4) || !aligned(c.table, 8)) return refuse(st, ECAD_E_INVALID, "rope_table: NULL or unaligned pointer");
  if (meet(vector(c.table, (int64_t)c.S * a.pairs * 2, 4), vector(c.positions, (int64_t)c.S * c.axes, 4))) return refuse(st, ECAD_E_INVALID, "rope_table: the table overlaps the positions");
  a.positions = c.positions; a.table = c.table; a.positions_float = c.positions_float; a.axes = c.axes; a.S = c.S;
  a.size = c.scaling == ECAD_ROPE_YARN ? (float)(0.1 * log(c.factor) + 1.0) : 1.0f;
  a.rows_per_block = a.pairs >= 512 ? 1 : 512 / a.pairs;
  const int threads = (a.rows_per_block * a.pairs + 63) / 64 * 64;
  const int64_t blocks = ((int64_t)c.S + a.rows_per_block - 1) / a.rows_per_block, most = (int64_t)ctx.num_cus * 8;
  hipLaunchKernelGGL(rope_table_kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(threads), 0, ctx.stream, a);
  return launched(st, "rope_table");
}

int op_rope(const OpCtx& ctx, const EcadRope& c, OpStatus& st) noexcept {
  if (c.B < 0 || c.S < 0 || c.q.H < 1 || c.k.H < 0 || c.q.H > (1 << 20) || c.k.H > (1 << 20) || c.D < 2 || c.D > (1 << 24) || c.rot < 2 || c.rot % 2 || c.rot > c.D || c.table_rows < 0)
    return refuse(st, ECAD_E_INVALID, "rope: %d samples of %d tokens, %lld + %lld heads of %d elements, %d of them turned (even, 2 to the head's size)", c.B, c.S,
                  (long long)c.q.H, (long long)c.k.H, c.D, c.rot);
  if (c.B == 0 || c.S == 0) return ECAD_OK;
  if (!c.q.x || !c.q.out || (c.k.H && (!c.k.x || !c.k.out)) || (!c.table && c.table_rows)) return refuse(st, ECAD_E_INVALID, "rope: NULL pointer");  // (no rows: every index lies outside)
  if (!aligned(c.q.x, 2) || !aligned(c.q.out, 2) || !aligned(c.k.x, 2) || !aligned(c.k.out, 2) || !aligned(c.table, 4) || !aligned(c.index, 4)) return refuse(st, ECAD_E_INVALID, "rope: pointers are not aligned to their type");
  if (!c.index && c.table_rows < c.S) return refuse(st, ECAD_E_INVALID, "rope: the table has %d rows for %d tokens", c.table_rows, c.S);
  auto negative = [](const EcadRopeHeads& x) { return x.sample < 0 || x.token < 0 || x.head < 0 || x.out_sample < 0 || x.out_token < 0 || x.out_head < 0; };
  if (negative(c.q) || (c.k.H && negative(c.k)) || c.index_stride < 0) return refuse(st, ECAD_E_INVALID, "rope: a stride is negative");
  const bool q_in = c.q.x == c.q.out, k_in = c.k.H == 0 || c.k.x == c.k.out;
  if (c.k.H && q_in != k_in) return refuse(st, ECAD_E_INVALID, "rope: queries and keys are both turned in place or both not");
  // (a stride over one sample, token or head is never taken)
  auto same = [&](const EcadRopeHeads& x) { return (c.B == 1 || x.sample == x.out_sample) && (c.S == 1 || x.token == x.out_token) && (x.H == 1 || x.head == x.out_head); };
  if (q_in && (!same(c.q) || (c.k.H && !same(c.k)))) return refuse(st, ECAD_E_INVALID, "rope: in place needs the same strides on both sides");
  auto in_of = [&](const EcadRopeHeads& x) { return Region{x.H ? (const char*)x.x : nullptr, {1, c.B, c.S, x.H}, {0, 2 * x.sample, 2 * x.token, 2 * x.head}, (int64_t)2 * c.D}; };
  auto out_of = [&](const EcadRopeHeads& x) { return Region{x.H ? (const char*)x.out : nullptr, {1, c.B, c.S, x.H}, {0, 2 * x.out_sample, 2 * x.out_token, 2 * x.out_head}, (int64_t)2 * c.D}; };
  const Region q = in_of(c.q), k = in_of(c.k), qo = out_of(c.q), ko = out_of(c.k);
  const Region in[] = {vector(c.table, (int64_t)c.table_rows * c.rot, 4), matrix(c.index, c.index_stride ? c.B : 1, c.S, c.index_stride, 4)};
  if (!distinct(qo) || (c.k.H && !distinct(ko))) return refuse(st, ECAD_E_INVALID, "rope: an output overlaps itself");
  if (meet(qo, ko) || meets_any(qo, in) || meets_any(ko, in) || meet(qo, k) || meet(ko, q) || (!q_in && (meet(qo, q) || meet(ko, k)))) return refuse(st, ECAD_E_INVALID, "rope: an output overlaps another argument");
  RopeArgs a{};
  a.q = c.q; a.k = c.k; a.table = c.table; a.index = c.index; a.index_stride = c.index_stride; a.S = c.S; a.D = c.D; a.rot = c.rot; a.table_rows = c.table_rows; a.copy = !q_in;
  a.sign = c.inverse ? -1.f : 1.f;
  a.tokens = (int64_t)c.B * c.S;
  a.turning = c.half ? (c.rot / 2 + 7) / 8 : (c.rot + 7) / 8;
  a.units = c.half ? a.turning + (a.copy ? (c.D - c.rot + 7) / 8 : 0) : (a.copy ? (c.D + 7) / 8 : a.turning);
  a.groups = (int)((c.q.H + c.k.H + ROPE_HEADS - 1) / ROPE_HEADS);
  const int64_t per_token = (int64_t)a.units * a.groups;
  if (per_token > (1 << 24)) return refuse(st, ECAD_E_UNSUPPORTED, "rope: %lld pieces a token", (long long)per_token);
  constexpr int64_t most = 1 << 23;  // workgroups; more tokens than that: several turns of one
  const int64_t one = per_token >= 256 ? 1 : 256 / per_token, many = (a.tokens + most - 1) / most;
  if (many > one && many * per_token > 0x7fffffff) return refuse(st, ECAD_E_UNSUPPORTED, "rope: %lld tokens are more than one launch takes", (long long)a.tokens);
  a.tokens_per_block = (int)(many > one ? many : one);
  const int64_t blocks = (a.tokens + a.tokens_per_block - 1) / a.tokens_per_block;
  const dim3 grid((unsigned)blocks), block(256);
  if (ctx.dtype == ECAD_DTYPE_F16) {
    if (c.half) hipLaunchKernelGGL((rope_kernel<f16_t, true>), grid, block, 0, ctx.stream, a);
    else hipLaunchKernelGGL((rope_kernel<f16_t, false>), grid, block, 0, ctx.stream, a);
  } else {
    if (c.half) hipLaunchKernelGGL((rope_kernel<bf16_t, true>), grid, block, 0, ctx.stream, a);
    else hipLaunchKernelGGL((rope_kernel<bf16_t, false>), grid, block, 0, ctx.stream, a);
  }
  return launched(st, "rope");
}

}  // namespace ecad
