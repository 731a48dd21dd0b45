"""The launches of an 8-bit transformer block (-m gpu): ecad_op_quantize_int8, ecad_op_gemm_int8, ecad_op_gate_norm, ecad_op_rope_table, ecad_op_rope against their
definitions in 64 bits.

Tolerances, per element and fixed before the first run: one rounding to the storage type, eps / 2 of the value (plus half of the smallest fp16 step), and the fp32
arithmetic in front of it, a stated multiple of 2^-24 of the magnitudes that enter the sum (`extra`).  8-bit integers and their scales are exact."""
import math
import threading

import pytest
import torch

from gpu_util import small_engine

pytestmark = pytest.mark.gpu

DTYPES = ("float16", "bfloat16")
STEP = 2.0**-24  # half a step of fp32


def rand(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def near(out, ref, extra=0.0):
    """|out - ref| within the rounding of out's type and `extra`; infinities and NaN where ref has them."""
    out64, eps = out.double(), torch.finfo(out.dtype).eps
    ok = (out64 - ref).abs() <= eps / 2 * ref.abs() * (1 + eps) + torch.finfo(out.dtype).smallest_normal * eps / 2 + extra
    top = torch.finfo(out.dtype).max
    ok |= (ref.abs() > top * (1 - eps)) & (out64.abs() >= top) & (out64.sign() == ref.sign())
    ok |= ref.isnan() & out64.isnan()
    if not bool(ok.all()):
        at = (~ok).nonzero()[0].tolist()
        raise AssertionError(f"{int((~ok).sum())} of {ok.numel()} off, first at {at}: {float(out64[tuple(at)])} for {float(ref[tuple(at)])}")


def quantized(x):
    """(q, scale) by definition: the scale is the fp32 quotient, the integer is the exact quotient's."""
    amax = x.double().abs().amax(1)
    scale = torch.where(torch.isfinite(amax), amax / 127.0, torch.nan).float()  # in 64 bits first: torch divides fp32 by a number as a product with its reciprocal
    q = torch.where(scale[:, None] > 0, x.double() / scale.double()[:, None], 0.0).round()
    return torch.where(torch.isfinite(amax)[:, None], q, 0.0).to(torch.int8), scale


def int8_rows(rows, width, seed, full=False):
    g = torch.Generator().manual_seed(seed)
    buf = torch.randint(-128, 128, (rows, (width + 15) // 16 * 16), generator=g, dtype=torch.int8).cuda()  # what lies behind the row's values is not zero
    q = buf[:, :width]
    if not full:
        q.clamp_(-127, 127)
    return q


def gelu64(v):
    return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v**3)))


ACTS = {0: lambda v: v, 1: gelu64, 2: lambda v: v * torch.sigmoid(v), 3: lambda v: v}


# ---- 8-bit rows --------------------------------------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype_name", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (5, 8), (64, 72), (33, 511), (7, 1001), (130, 1152), (4, 1536), (9, 1537), (6, 4096), (5, 4608), (3, 8191), (2, 16384), (2, 32767), (1, 131071)])
def test_quantize_is_exact(dtype_name, M, K):
    dt = getattr(torch, dtype_name)
    x = rand(M, K, seed=M + K, dtype=dt, scale=3.0)
    x[0, 0] = 254.0 if M > 1 else 1.0  # a scale of 2: every odd value is a tie
    if M > 2:
        x[0, 1:] = torch.randint(-253, 254, (K - 1,), generator=torch.Generator().manual_seed(1)).to(dt).cuda() if dt == torch.float16 else x[0, 1:].round()
        x[1] = 0.0
    q, s = small_engine(dtype_name).op_quantize_int8(x)
    rq, rs = quantized(x)
    assert torch.equal(s, rs) and torch.equal(q, rq)
    assert q.stride(0) % 16 == 0


@pytest.mark.parametrize("dtype_name", DTYPES)
def test_quantize_every_border(dtype_name):
    """All 16-bit patterns against scales of many kinds: values next to and on the borders between two integers."""
    dt = getattr(torch, dtype_name)
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dt).cuda()
    tops = torch.tensor([1.0, 127.0, 126.5, 254.0, 0.37, 3.3e4, 6.1e-5, 5.9e-8, 1.7, 100.0], device="cuda").to(dt)
    if dt == torch.bfloat16:
        tops = torch.cat((tops, torch.tensor([1e-38, 3e-39, 9.2e-41, 3e38, 1e-30, 1.1e-30], device="cuda").to(dt)))
    rows = torch.stack([torch.where(every.abs() <= t, every, torch.zeros_like(every)) for t in tops])
    rows[:, 0] = tops
    q, s = small_engine(dtype_name).op_quantize_int8(rows)
    rq, rs = quantized(rows)
    assert torch.equal(s, rs) and torch.equal(q, rq)


@pytest.mark.parametrize("dtype_name", DTYPES)
def test_quantize_bad_rows_strides_and_neighbours(dtype_name):
    dt, eng = getattr(torch, dtype_name), small_engine(dtype_name)
    wide = rand(6, 301, seed=3, dtype=dt)
    x = wide[::2, 3:204]  # odd offset, odd stride
    x[0, 7], x[1, 200] = float("nan"), float("-inf")
    buf = torch.full((3, 224), 99, dtype=torch.int8, device="cuda")
    s = torch.full((5,), 7.0, device="cuda")
    eng.op_quantize_int8(x, out=(buf[:, :201], s[1:4]))
    assert bool(s[1:3].isnan().all()) and bool((buf[:2, :201] == 0).all()) and bool((buf[:, 201:] == 99).all()) and s[0] == 7 and s[4] == 7
    rq, rs = quantized(x)
    assert torch.equal(buf[2, :201], rq[2]) and s[3] == rs[2]
    q, s = eng.op_quantize_int8(wide[:0])
    assert q.shape == (0, 301) and s.shape == (0,)


# ---- the product ----------------------------------------------------------------------------------------------------------------------------------------------

SHAPES = [(1, 1, 1), (1, 17, 16), (2, 6912, 1152), (16, 100, 63), (17, 33, 65), (32, 48, 128), (33, 1152, 200), (64, 130, 4608), (65, 64, 129), (100, 257, 1000), (129, 1111, 401), (256, 288, 256),
          (300, 144, 1152), (512, 1152, 4096), (601, 577, 130), (1000, 4608, 1152)]


def takes(kernel, M, K):
    """What the named kernels refuse."""
    return not (kernel == "rows" and M > 32 or kernel in ("tile256", "tile288") and K < 256 or kernel == "tile144" and K < 384)


def product64(a, sa, w, sw, bias):
    acc = a.double() @ w.double().t()  # whole numbers below 2^31: exact
    scaled = acc * sa.double()[:, None] * sw.double()
    return scaled + (bias.double() if bias is not None else 0.0), scaled.abs() + (bias.double().abs() if bias is not None else 0.0)


@pytest.mark.parametrize("dtype_name", DTYPES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm_every_kernel_and_epilogue(dtype_name, M, N, K):
    """Four roundings to fp32 in front of the output's (sum, scales, bias, and the activation's own few): 2^-20 of the magnitudes covers them; every kernel gives the same bits."""
    dt, eng = getattr(torch, dtype_name), small_engine(dtype_name)
    a, w = int8_rows(M, K, 1), int8_rows(N, K, 2, full=True)
    sa, sw = torch.rand(M, device="cuda") * 0.02 + 1e-3, (torch.rand(N, device="cuda") + 0.1) / (60.0 * math.sqrt(K))
    bias = rand(N, seed=5)
    if M > 3:
        sa[2] = 0.0
        sa[3] = float("nan")
    for epi in range(3):
        pre, size = product64(a, sa, w, sw, bias if epi != 2 else None)
        first = None
        for kernel in eng.INT8_KERNELS:
            if not takes(kernel, M, K):
                continue
            out = eng.op_gemm_int8(epi, a, sa, w, sw, bias if epi != 2 else None, kernel=kernel)
            if first is None:
                near(out, ACTS[epi](pre), 2.0**-20 * size.nan_to_num())
                first = out
            assert torch.equal(out.view(torch.int16), first.view(torch.int16)) or (torch.equal(out.isnan(), first.isnan()) and torch.equal(out.nan_to_num(), first.nan_to_num())), (kernel, epi)


@pytest.mark.parametrize("dtype_name", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 5, 33), (8, 1152, 4608), (50, 77, 100), (70, 130, 300), (300, 1152, 640), (513, 289, 1152)])
@pytest.mark.parametrize("gate", ["table+mod", "table", "mod", "none"])
def test_gemm_gated_residual(dtype_name, M, N, K, gate):
    """Epilogue 3: the residual takes the rounded output (checked against the output that came out), one more fma and one rounding."""
    dt, eng = getattr(torch, dtype_name), small_engine(dtype_name)
    a, w = int8_rows(M, K, 3), int8_rows(N, K, 4)
    sa, sw, bias = torch.rand(M, device="cuda") * 0.02 + 1e-3, torch.rand(N, device="cuda") / (40.0 * math.sqrt(K)), rand(N, seed=6)
    rows = (M + 2) // 3
    table = rand(N, seed=7) if "table" in gate else None
    mod = rand(3, 2 * N + 3, seed=8, dtype=dt)[:, 3 : N + 3] if "mod" in gate else None
    g = torch.ones(M, N, device="cuda", dtype=torch.float64) if gate == "none" else torch.zeros(M, N, device="cuda", dtype=torch.float64)
    if table is not None:
        g = g + table.double()
    if mod is not None:
        g = g + mod.double()[torch.arange(M, device="cuda") // rows]
    pre, size = product64(a, sa, w, sw, bias)
    base = rand(M, N + 5, seed=9, dtype=dt)
    kept = None
    for kernel in eng.INT8_KERNELS:
        if not takes(kernel, M, K):
            continue
        wide = base.clone()
        out = torch.empty(M, N, device="cuda", dtype=dt)
        got = eng.op_gemm_int8(3, a, sa, w, sw, bias, resid=wide[:, 3 : N + 3], gate_table=table, gate_mod=mod, rows_per_batch=rows, out=out, kernel=kernel)
        assert got is out and torch.equal(wide[:, :3], base[:, :3]) and torch.equal(wide[:, N + 3 :], base[:, N + 3 :])
        near(out, pre, 2.0**-20 * size)
        near(wide[:, 3 : N + 3], base[:, 3 : N + 3].double() + g * out.double(), 4 * STEP * (g * out.double()).abs())
        apart = torch.empty(M, N, device="cuda", dtype=dt)  # out not wanted, the residual elsewhere
        assert eng.op_gemm_int8(3, a, sa, w, sw, bias, resid=base[:, 3 : N + 3], gate_table=table, gate_mod=mod, rows_per_batch=rows, resid_out=apart, kernel=kernel) is None
        assert torch.equal(apart, wide[:, 3 : N + 3])
        kept = apart if kept is None else kept
        assert torch.equal(apart, kept)


def test_one_row_takes_any_stride():
    """A single 8-bit row (a user's own, without padding behind it) as activation, as weight and as the quantiser's output."""
    eng = small_engine("float16")
    q = int8_rows(1, 40, 1).clone(memory_format=torch.contiguous_format)
    assert q.stride() == (40, 1)
    one = torch.ones(1, device="cuda")
    out = eng.op_gemm_int8(0, q, one * 1e-3, q, one)
    near(out, (q.double() ** 2).sum().view(1, 1) * one.double() * (one * 1e-3).double(), 2.0**-20)
    x, s = rand(1, 41, seed=1, dtype=torch.float16), torch.empty(1, device="cuda")
    buf = torch.full((1, 41), 99, dtype=torch.int8, device="cuda")
    eng.op_quantize_int8(x, out=(buf, s))
    assert all(torch.equal(a, b) for a, b in zip((buf, s), quantized(x)))


def test_gemm_largest_sums():
    """All operands at -128 over the longest K: the sum is K 2^14 = 2147467264, just inside 32 bits."""
    eng = small_engine("bfloat16")
    K = 131071
    buf = torch.full((20, (K + 15) // 16 * 16), -128, device="cuda", dtype=torch.int8)
    one = torch.ones(20, device="cuda") * 2.0**-31
    for kernel in ("rows", "tile64", "tile128", "tile256"):
        out = eng.op_gemm_int8(0, buf[:, :K], one, buf[:, :K], one * 2.0**31, kernel=kernel)
        near(out, torch.full((20, 20), K * 2.0**14 * 2.0**-31, device="cuda", dtype=torch.float64))


@pytest.mark.parametrize("kernel", ["rows", "tile64", "tile64k2", "tile128", "tile144", "tile256", "tile288"])
def test_gemm_scales_whose_product_leaves_fp32(kernel):
    """1e-23 * 1e-21 is seven steps above zero in fp32, the result 1e-37 is not; and a sum of zero stays zero where the scales' product would be infinite."""
    eng, M, N, K = small_engine("bfloat16"), 30, 40, 1152
    a, w = int8_rows(M, K, 1), int8_rows(N, K, 2)
    a.fill_(100)
    w.fill_(90)
    one = torch.ones(64, device="cuda")
    out = eng.op_gemm_int8(0, a, one[:M] * 1e-23, w, one[:N] * 1e-21, kernel=kernel)
    ref = torch.full((M, N), 9000.0 * K, device="cuda", dtype=torch.float64) * float((one * 1e-23)[0].double() * (one * 1e-21)[0].double())
    near(out, ref, 2.0**-22 * ref)
    w[:, ::2] = -90
    out = eng.op_gemm_int8(0, a, one[:M] * 1e30, w, one[:N] * 1e30, one[:N] * 3, kernel=kernel)
    assert bool((out == 3).all())


def test_gemm_offsets_beyond_32_bits():
    eng, dt = small_engine("float16"), torch.float16
    M, N, K = 300_003, 8192, 16
    a, w = int8_rows(M, K, 1), int8_rows(N, K, 2)
    sa, sw = torch.rand(M, device="cuda") * 0.02, torch.rand(N, device="cuda") * 0.02
    out = eng.op_gemm_int8(0, a, sa, w, sw)
    for at in (slice(0, 5), slice(262140, 262150), slice(M - 5, M)):
        pre, size = product64(a[at], sa[at], w, sw, None)
        near(out[at], pre, 2.0**-20 * size)


# ---- norms ----------------------------------------------------------------------------------------------------------------------------------------------------


def norm64(x, kind, eps):
    if kind == "none":
        return x, x.abs()
    c = x - x.mean(1, keepdim=True) if kind == "layer" else x
    r = 1 / ((c * c).mean(1, keepdim=True) + eps).sqrt()
    return c * r, (x.abs() + x.abs().mean(1, keepdim=True)) * r


def gate_norm64(h, y, pre, post, a, eps, rows, pre_weight=None, post_weight=None, gate_table=None, gate_mod=None, table_shift=None, table_scale=None, mod_shift=None, mod_scale=None):
    """(h', its magnitude, n, its magnitude): the magnitudes are what fp32 errors are relative to."""
    sample = torch.arange(h.shape[0], device=h.device) // rows

    def both(table, mod, base):
        if table is None and mod is None:
            return torch.full((1, 1), base, device=h.device, dtype=torch.float64)
        return (0 if table is None else table.double()) + (0 if mod is None else mod.double()[sample])

    size = h.double().abs()
    hh = h.double()
    if y is not None:
        u, us = norm64(y.double(), post, eps)
        g = both(gate_table, gate_mod, 1.0) * (1 if post_weight is None else post_weight.double())
        hh, size = a * hh + g * u, (a * hh).abs() + g.abs() * us
    if pre == "none":
        return hh, size, None, None
    n, _ = norm64(hh, pre, eps)
    _, ns = norm64(size, pre, eps)
    # rstd is the true row's, the magnitude that enters is the one before cancellation
    c = hh - hh.mean(1, keepdim=True) if pre == "layer" else hh
    ns = (size + size.mean(1, keepdim=True)) / ((c * c).mean(1, keepdim=True) + eps).sqrt()
    A = (1 if pre_weight is None else pre_weight.double()) * (1 + both(table_scale, mod_scale, 0.0))
    B = both(table_shift, mod_shift, 0.0)
    return hh, size, n * A + B, ns * A.abs() + B.abs() + n.abs() * A.abs() * ns.abs().amax(1, keepdim=True)


FULL = dict(pre_weight=True, post_weight=True, gate_table=True, gate_mod=True, table_shift=True, table_scale=True, mod_shift=True, mod_scale=True)
WIDTHS = [1, 2, 7, 8, 72, 511, 512, 513, 1023, 1152, 1536, 1537, 2048, 2049, 4096, 4097, 8192, 8193, 16384, 16391, 32768]


def norm_inputs(M, D, dt, samples, which, seed=0):
    mod = rand(samples, 3 * D, seed=seed + 1, dtype=dt, scale=0.3)
    every = dict(pre_weight=1 + rand(D, seed=seed + 2, scale=0.2), post_weight=1 + rand(D, seed=seed + 3, scale=0.2), gate_table=rand(D, seed=seed + 4, scale=0.3), gate_mod=mod[:, :D],
                 table_shift=rand(D, seed=seed + 5, scale=0.1), table_scale=rand(D, seed=seed + 6, scale=0.1), mod_shift=mod[:, D : 2 * D], mod_scale=mod[:, 2 * D :])
    return rand(M, D, seed=seed + 7, dtype=dt, scale=2.0), rand(M, D, seed=seed + 8, dtype=dt), {k: v for k, v in every.items() if which.get(k)}


@pytest.mark.parametrize("dtype_name", DTYPES)
@pytest.mark.parametrize("pre,post", [("layer", "none"), ("rms", "rms"), ("layer", "layer"), ("none", "rms"), ("rms", "none")])
@pytest.mark.parametrize("D", WIDTHS)
def test_gate_norm_widths_and_kinds(dtype_name, pre, post, D):
    """fp32 sums of D terms (pairwise over lanes, at most 32 in a row within one) and a dozen operations: 2^-19 of the magnitudes."""
    dt, eng = getattr(torch, dtype_name), small_engine(dtype_name)
    M = 9 if D > 600 else 37
    which = dict(FULL, post_weight=post != "none", **({k: pre != "none" for k in ("pre_weight", "table_shift", "table_scale", "mod_shift", "mod_scale")}))
    h, y, par = norm_inputs(M, D, dt, 3, which, seed=D)
    rows = (M + 2) // 3
    nh, n = eng.op_gate_norm(h, y, pre=pre, post=post, rows_per_batch=rows, resid_scale=0.81, eps=1e-6, **par)
    rh, sh, rn, sn = gate_norm64(h, y, pre, post, 0.81, 1e-6, rows, **par)
    near(nh, rh, 2.0**-19 * sh)
    if pre == "none":
        assert n is None
        return
    near(n, rn, 2.0**-19 * sn)
    qh, (q, s) = eng.op_gate_norm(h, y, pre=pre, post=post, rows_per_batch=rows, resid_scale=0.81, eps=1e-6, quantize=True, **par)
    uq, us = eng.op_quantize_int8(n)
    assert torch.equal(qh, nh) and torch.equal(q, uq) and torch.equal(s, us)


@pytest.mark.parametrize("dtype_name", DTYPES)
@pytest.mark.parametrize("leave_out", sorted(FULL) + ["tables", "mods", "all"])
def test_gate_norm_every_parameter_may_be_absent(dtype_name, leave_out):
    dt, eng = getattr(torch, dtype_name), small_engine(dtype_name)
    gone = {"tables": ("gate_table", "table_shift", "table_scale"), "mods": ("gate_mod", "mod_shift", "mod_scale"), "all": tuple(FULL)}.get(leave_out, (leave_out,))
    h, y, par = norm_inputs(21, 200, dt, 4, {k: k not in gone for k in FULL}, seed=3)
    nh, n = eng.op_gate_norm(h, y, pre="rms", post="layer", rows_per_batch=6, **par)
    rh, sh, rn, sn = gate_norm64(h, y, "rms", "layer", 1.0, 1e-6, 6, **par)
    near(nh, rh, 2.0**-19 * sh)
    near(n, rn, 2.0**-19 * sn)


@pytest.mark.parametrize("M", [1, 2, 5, 4095, 33001])
@pytest.mark.parametrize("D", [72, 1152, 2304])
def test_gate_norm_row_counts(M, D):
    """From one row to more than every group size; samples of one row, and samples that change inside a group."""
    eng, dt = small_engine("bfloat16"), torch.bfloat16
    for samples in {1, min(M, 7), min(M, 4095)}:
        h, y, par = norm_inputs(M, D, dt, samples, dict(FULL, pre_weight=False), seed=M)
        rows = (M + samples - 1) // samples
        nh, n = eng.op_gate_norm(h, y, pre="layer", post="rms", rows_per_batch=rows, **par)
        rh, sh, rn, sn = gate_norm64(h, y, "layer", "rms", 1.0, 1e-6, rows, **par)
        near(nh, rh, 2.0**-19 * sh)
        near(n, rn, 2.0**-19 * sn)


@pytest.mark.parametrize("dtype_name", DTYPES)
def test_gate_norm_strides_in_place_and_edges(dtype_name):
    dt, eng = getattr(torch, dtype_name), small_engine(dtype_name)
    wide = rand(10, 3 * 101, seed=1, dtype=dt)
    h, y = wide[::2, 1:102], wide[::2, 102:203]
    keep = wide.clone()
    rh, sh, rn, sn = gate_norm64(h, y, "rms", "layer", 0.5, 1e-5, 2)
    nh, n = eng.op_gate_norm(h, y, pre="rms", post="layer", resid_scale=0.5, eps=1e-5, rows_per_batch=2, out_h=h, out_n=y)
    assert nh.data_ptr() == h.data_ptr() and n.data_ptr() == y.data_ptr()
    near(h, rh, 2.0**-19 * sh)
    near(y, rn, 2.0**-19 * sn)
    for part in (wide[1::2], wide[::2, :1], wide[::2, 203:]):  # nothing around them is touched
        at = part.storage_offset()
        assert torch.equal(part, keep.as_strided(part.shape, part.stride(), at))
    # without y: h itself comes back, only the pre-norm runs
    x = rand(6, 40, seed=2, dtype=dt)
    back, n = eng.op_gate_norm(x, pre="layer")
    assert back is x
    _, _, rn, sn = gate_norm64(x, None, "layer", "none", 1.0, 1e-6, 1)
    near(n, rn, 2.0**-19 * sn)
    # constant rows, zero rows, infinities and NaN stay in their rows
    x = rand(6, 300, seed=4, dtype=dt)
    x[0], x[1], x[2, 5], x[3, 299] = 3.0, 0.0, float("inf"), float("nan")
    for pre in ("layer", "rms"):
        _, n = eng.op_gate_norm(x, pre=pre)
        _, _, rn, sn = gate_norm64(x, None, pre, "none", 1.0, 1e-6, 1)
        near(n[[0, 1, 4, 5]], rn[[0, 1, 4, 5]], 2.0**-19 * sn[[0, 1, 4, 5]])
        assert bool(n[3].isnan().all()) and bool(n[2].isnan().any())
        _, (q, s) = eng.op_gate_norm(x, pre=pre, quantize=True)
        assert bool(s[2:4].isnan().all()) and bool((q[2:4] == 0).all()) and bool(s[[0, 1, 4, 5]].isfinite().all())
    empty = x[:0]
    nh, n = eng.op_gate_norm(empty, empty, pre="rms")
    assert nh.shape == n.shape == (0, 300)


def test_gate_norm_large_means_do_not_cancel():
    """Rows around 200 with a spread of 1: a one-pass variance would be wrong in the third digit."""
    eng = small_engine("float16")
    x = (rand(16, 1152, seed=5) + 200).to(torch.float16)
    _, n = eng.op_gate_norm(x, pre="layer")
    ref = (x.double() - x.double().mean(1, keepdim=True)) / (x.double().var(1, unbiased=False, keepdim=True) + 1e-6).sqrt()
    near(n, ref, 2.0**-14)  # 200 * 2^-24 * rstd, and the mean's own error: 2^-14 is ten times that


def test_row_offsets_beyond_32_bits():
    """More than 2^31 elements in rows of 32768: the last rows are the test."""
    eng, dt, D, M = small_engine("bfloat16"), torch.bfloat16, 32768, 65600
    h = torch.zeros(M, D, device="cuda", dtype=dt)
    h[-3:] = rand(3, D, seed=1, dtype=dt)
    nh, n = eng.op_gate_norm(h, h, pre="rms", resid_scale=0.5)
    rh, sh, rn, sn = gate_norm64(h[-3:], h[-3:], "rms", "none", 0.5, 1e-6, 1)
    near(nh[-3:], rh, 2.0**-19 * sh)
    near(n[-3:], rn, 2.0**-19 * sn)
    q, s = eng.op_quantize_int8(n)
    rq, rs = quantized(n[-3:])
    assert torch.equal(q[-3:], rq) and torch.equal(s[-3:], rs) and bool((s[:-3] == 0).all())
    del q, nh, n
    table = eng.op_rope_table(torch.arange(M, device="cuda", dtype=torch.int32), 64)
    x = h.view(1, M, 256, 128)
    out, _ = eng.op_rope(x, None, table, layout="half")
    near(out[0, -3:], rope64(x[:, -3:], table[-3:], "half")[0])


def test_more_rows_than_one_launch_counts():
    """A launch has fewer than 2^32 threads: 2^26 rows at four to a workgroup, 2^24 at one, as many tiles of 64 rows are more."""
    eng, dt = small_engine("float16"), torch.float16
    for M, K in ((2**26 + 5, 8), (2**24 + 3, 1544)):
        x = torch.zeros(M, K, device="cuda", dtype=dt)
        at = [0, 1, M // 2, M - 6, M - 3, M - 1]
        x[at] = rand(len(at), K, seed=1, dtype=dt)
        q, s = eng.op_quantize_int8(x)
        rq, rs = quantized(x[at])
        assert torch.equal(q[at], rq) and torch.equal(s[at], rs)
        assert int((s != 0).sum()) == len(at)
        del x, q, s
    M = 2**30 + 65
    a = torch.ones(M, 16, device="cuda", dtype=torch.int8)
    w, one = int8_rows(1, 16, 2), torch.ones(1, device="cuda")
    out = eng.op_gemm_int8(0, a, one.expand(M).contiguous(), w, one)
    assert bool((out == w.sum(dtype=torch.int32).to(dt)).all())
    with pytest.raises(ValueError, match="more than one launch"):
        eng.op_gemm_int8(0, a, out.float().view(-1), w, one, kernel="tile64")


def test_rope_of_more_tokens_than_one_launch_counts():
    eng, dt = small_engine("float16"), torch.float16
    B, S = 70_000, 65_536  # 256 tokens of one pair a workgroup: more than 2^24 of those
    table = eng.op_rope_table(torch.arange(S, device="cuda", dtype=torch.int32), 2)
    x = torch.ones(1, device="cuda", dtype=dt).expand(B * S * 2).contiguous().view(B, S, 1, 2)
    expected = rope64(x[:1], table, "half")[0]
    eng.op_rope(x, None, table, layout="half", out=(x, None))
    near(x[:1], expected)
    assert all(torch.equal(part, x[:1].expand_as(part)) for part in x.split(7000))


# ---- rotary positions -----------------------------------------------------------------------------------------------------------------------------------------


def table64(positions, dims, theta=10000.0, scaling="none", factor=1.0, original=0, fast=32.0, slow=1.0):
    cols = []
    p = positions.double().cpu()
    p = p[:, None] if p.dim() == 1 else p
    size = 0.1 * math.log(factor) + 1 if scaling == "yarn" else 1.0
    for axis, d in enumerate(dims):
        base = theta * factor ** (d / (d - 2)) if scaling == "ntk" and d > 2 else theta
        for j in range(d // 2):
            f = base ** (-2 * j / d)
            if scaling == "linear":
                f /= factor
            if scaling == "yarn":
                w = min(1.0, max(0.0, (original * f / (2 * math.pi) - slow) / (fast - slow)))
                f = f * w + f / factor * (1 - w)
            cols.append(torch.stack(((p[:, axis] * f).cos(), (p[:, axis] * f).sin()), -1) * size)
    return torch.stack(cols, 1).cuda(), size


@pytest.mark.parametrize("S,dims", [(1, (2,)), (5, (64,)), (1000, (16, 56, 56)), (333, (2, 4, 6)), (4097, (128,)), (70, (512,)), (3, (2,) * 8)])
@pytest.mark.parametrize("scaling,factor", [("none", 1.0), ("linear", 4.0), ("ntk", 8.0), ("yarn", 16.0)])
@pytest.mark.parametrize("kind", ["int", "float"])
def test_rope_table(S, dims, scaling, factor, kind):
    """The remainder of the angle is rounded to fp32 once and two short sums follow: 4 * 2^-24 of the table's size at any position (the 64-bit angle itself: 2^-29 at 10^7)."""
    g = torch.Generator().manual_seed(S)
    pos = torch.randint(-1000, 10_000_000, (S, len(dims)), generator=g, dtype=torch.int32)
    pos = pos.cuda() if kind == "int" else (pos.float() / 7).cuda()
    if len(dims) == 1 and S % 2:
        pos = pos[:, 0].contiguous()
    out = small_engine().op_rope_table(pos, dims if len(dims) > 1 else dims[0], theta=500000.0, scaling=scaling, factor=factor, original_length=4096)
    ref, size = table64(pos, dims, 500000.0, scaling, factor, 4096)
    assert out.dtype == torch.float32 and float((out.double() - ref).abs().max()) <= 4.5 * STEP * size * 1.0001


def test_rope_table_quarter_turns_and_odd_values():
    eng = small_engine()
    out = eng.op_rope_table(torch.zeros(4, dtype=torch.int32, device="cuda"), 8)
    assert torch.equal(out, torch.tensor([1.0, 0.0], device="cuda").expand(4, 4, 2))
    pos = torch.tensor([0.0, math.pi / 2, math.pi, 1.5 * math.pi, 2 * math.pi, -math.pi / 4, math.pi / 4, 2.0**31, float("inf"), float("nan")], device="cuda")
    out = eng.op_rope_table(pos, 2)
    ref, _ = table64(pos[:-2], (2,))
    assert float((out[:-2].double() - ref).abs().max()) <= 2.0**-22 and bool(out[-2:].isnan().all())
    keep = torch.full((6, 4, 2), 9.0, device="cuda")
    eng.op_rope_table(torch.arange(4, device="cuda", dtype=torch.int32), 8, out=keep[1:5])
    assert bool((keep[[0, 5]] == 9).all()) and not bool((keep[1:5] == 9).any())
    assert eng.op_rope_table(torch.zeros(0, dtype=torch.int32, device="cuda"), 8).shape == (0, 4, 2)


def rope64(x, rows, layout, inverse=False):
    """x [B, S, H, D] turned by rows [S or B, S, rot / 2, 2], in 64 bits."""
    rot = 2 * rows.shape[-2]
    c, s = (rows.double()[..., i].unsqueeze(-2) for i in (0, 1))
    s = -s if inverse else s
    x = x.double().clone()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if layout == "interleaved" else (x[..., : rot // 2], x[..., rot // 2 : rot])
    u, v = a * c - b * s, a * s + b * c
    if layout == "interleaved":
        x[..., 0:rot:2], x[..., 1:rot:2] = u, v
    else:
        x[..., : rot // 2], x[..., rot // 2 : rot] = u, v
    return x


@pytest.mark.parametrize("dtype_name", DTYPES)
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("B,S,H,Hk,D,rot", [(1, 1, 1, 1, 2, 2), (2, 7, 3, 1, 8, 4), (1, 33, 5, 5, 72, 72), (3, 5, 4, 2, 72, 48), (2, 100, 8, 2, 128, 128), (1, 9, 9, 3, 100, 34), (2, 3, 2, 0, 20, 14),
                                                (1, 257, 16, 16, 64, 64), (4, 1, 32, 8, 256, 256), (1, 3, 1, 1, 15, 10)])
def test_rope_layouts_parts_and_strides(dtype_name, layout, B, S, H, Hk, D, rot):
    """Two products and a sum in fp32: 3 * 2^-24 of |a c| + |b s|, at most twice the larger element; what does not turn keeps its bits."""
    dt, eng = getattr(torch, dtype_name), small_engine(dtype_name)
    qkv = rand(B, S, (H + 2 * Hk) * D, seed=D + S, dtype=dt)
    q = qkv[:, :, : H * D].view(B, S, H, D)
    k = qkv[:, :, H * D : (H + Hk) * D].view(B, S, Hk, D) if Hk else None
    table = eng.op_rope_table(torch.arange(3, S + 3, device="cuda", dtype=torch.int32), rot)
    for inverse in (False, True):
        oq, ok = eng.op_rope(q, k, table, layout=layout, inverse=inverse)
        for x, o in ((q, oq), (k, ok)):
            if x is None:
                assert o is None
                continue
            near(o, rope64(x, table, layout, inverse), 6 * STEP * x.double().abs().amax(-1, keepdim=True))
            assert torch.equal(o[..., rot:], x[..., rot:])
    # in place inside the fused projection, and the third part of it is not touched
    oq, ok = eng.op_rope(q, k, table, layout=layout)
    keep = qkv.clone()
    rq, rk = eng.op_rope(q, k, table, layout=layout, out=(q, k))
    assert rq is q and rk is k and torch.equal(q, oq) and (k is None or torch.equal(k, ok)) and torch.equal(qkv[:, :, (H + Hk) * D :], keep[:, :, (H + Hk) * D :])
    # heads first in memory
    swapped = oq.transpose(1, 2).contiguous().transpose(1, 2)
    again, _ = eng.op_rope(swapped, None, table, layout=layout, inverse=True)
    plain, _ = eng.op_rope(oq, None, table, layout=layout, inverse=True)
    assert torch.equal(again, plain)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rope_index(layout):
    eng, dt = small_engine("float16"), torch.float16
    B, S, H, D, rot = 3, 6, 5, 24, 16
    q, k = rand(B, S, H, D, seed=1, dtype=dt), rand(B, S, 2, D, seed=2, dtype=dt)
    table = eng.op_rope_table(torch.arange(100, device="cuda", dtype=torch.int32), rot)
    wide = torch.tensor([[4, 99, 0, 4, -1, 7, 5], [100, 1, 2, 3, 4, 5, 5], [-2147483648, 2147483647, 98, 0, 0, 0, 5]], device="cuda", dtype=torch.int32)
    for index in (wide[:, :S], wide[0, :S]):  # one list per sample (at a stride), one list for all
        rows = index.expand(B, S).long()
        inside = (rows >= 0) & (rows < 100)
        oq, ok = eng.op_rope(q, k, table, layout=layout, index=index)
        for x, o in ((q, oq), (k, ok)):
            near(o[inside], rope64(x, table[rows.clamp(0, 99)], layout)[inside], 6 * STEP * x.double().abs().amax())
            assert torch.equal(o[~inside], x[~inside])  # a row outside the table leaves its token as it is
        x = q.clone()
        eng.op_rope(x, None, table, layout=layout, index=index, out=(x, None))
        assert torch.equal(x, oq)


def test_rope_turns_back_and_keeps_inner_products():
    """The inverse is the gradient: <R x, y> = <x, R^-1 y>, and directional differences of the (linear) rotation are its values."""
    eng, dt = small_engine("float16"), torch.float16
    x, y = rand(2, 40, 4, 72, seed=1, dtype=dt), rand(2, 40, 4, 72, seed=2, dtype=dt)
    table = eng.op_rope_table(torch.arange(40, device="cuda", dtype=torch.int32) * 1000, 48)
    for layout in ("interleaved", "half"):
        rx, _ = eng.op_rope(x, None, table, layout=layout)
        back, _ = eng.op_rope(rx, None, table, layout=layout, inverse=True)
        ry, _ = eng.op_rope(y, None, table, layout=layout, inverse=True)
        big = float(x.abs().max() * 2)
        assert float((back.double() - x.double()).abs().max()) <= 2.5 * 2.0**-11 * big  # two roundings, the first one turned
        left, right = (rx.double() * y.double()).sum(-1), (x.double() * ry.double()).sum(-1)
        assert float((left - right).abs().max()) <= 2 * 2.0**-11 * float(((x.double() ** 2).sum(-1) * (y.double() ** 2).sum(-1)).sqrt().max())
        step = (x.float() + 0.5 * y.float()).to(dt)
        moved, _ = eng.op_rope(step, None, table, layout=layout)
        delta, _ = eng.op_rope((step.float() - x.float()).to(dt), None, table, layout=layout)
        assert float((moved.double() - rx.double() - delta.double()).abs().max()) <= 4 * 2.0**-11 * big


# ---- together -------------------------------------------------------------------------------------------------------------------------------------------------


def block(eng, h, y, st):
    """norm -> 8-bit QKV -> rotary positions -> attention -> 8-bit out projection onto the gated residual -> norm -> 8-bit feed-forward onto the gated residual."""
    B, S, H, Dh = st["B"], st["S"], st["H"], st["Dh"]
    D, M = H * Dh, B * S
    rows = dict(rows_per_batch=S)
    h1, (q8, s8) = eng.op_gate_norm(h, y, pre="layer", post="rms", quantize=True, gate_mod=st["mod"][:, :D], mod_shift=st["mod"][:, D : 2 * D], mod_scale=st["mod"][:, 2 * D : 3 * D], **rows)
    qkv0 = eng.op_gemm_int8(0, q8, s8, *st["qkv"], st["b_qkv"])
    qkv = qkv0.clone()
    heads = qkv.view(B, S, 3 * H, Dh)
    eng.op_rope(heads[:, :, :H], heads[:, :, H : 2 * H], st["table"], layout="half", out=(heads[:, :, :H], heads[:, :, H : 2 * H]))
    att = eng.op_attention(qkv[:, :D], qkv[:, D : 2 * D], qkv[:, 2 * D :], B, H, S, S, Dh)
    h2 = torch.empty_like(h)
    eng.op_gemm_int8(3, *eng.op_quantize_int8(att), *st["o"], None, resid=h1, resid_out=h2, gate_mod=st["mod"][:, :D], **rows)
    _, (q8b, s8b) = eng.op_gate_norm(h2, pre="rms", quantize=True)
    mid = eng.op_gemm_int8(1, q8b, s8b, *st["up"], st["b_up"])
    h3 = h2.clone()
    cache = torch.empty_like(h)
    eng.op_gemm_int8(3, *eng.op_quantize_int8(mid), *st["down"], None, resid=h3, gate_table=st["gate"], out=cache, **rows)
    return h1, q8, s8, qkv0, qkv, att, h2, q8b, s8b, mid, cache, h3


def block_state(eng, dt, B=2, S=100, H=4, Dh=72, seed=0):
    D = H * Dh
    weight = lambda n, k, s: eng.op_quantize_int8(rand(n, k, seed=seed + s, dtype=dt, scale=k**-0.5))  # noqa: E731
    return dict(B=B, S=S, H=H, Dh=Dh, mod=rand(B, 3 * D, seed=seed + 1, dtype=dt, scale=0.3), table=eng.op_rope_table(torch.arange(S, device="cuda", dtype=torch.int32), 48),
                qkv=weight(3 * D, D, 2), o=weight(D, D, 3), up=weight(4 * D, D, 4), down=weight(D, 4 * D, 5), b_qkv=rand(3 * D, seed=seed + 6, scale=0.1), b_up=rand(4 * D, seed=seed + 7, scale=0.1),
                gate=rand(D, seed=seed + 8)), rand(B * S, D, seed=seed + 9, dtype=dt, scale=2.0), rand(B * S, D, seed=seed + 10, dtype=dt)


@pytest.mark.parametrize("dtype_name", DTYPES)
def test_a_block_of_them(dtype_name):
    """All of them in turn, as a block uses them, next to the framework's attention: every tensor on the way against the definition in 64 bits of the tensors it was made from (a
    comparison of the last tensor alone would say little: an error of d of a rounded step in front of an 8-bit rounding leaves a whole step with probability d)."""
    dt, eng = getattr(torch, dtype_name), small_engine(dtype_name)
    st, h, y = block_state(eng, dt)
    B, S, H, Dh = st["B"], st["S"], st["H"], st["Dh"]
    D, eps = H * Dh, torch.finfo(dt).eps
    h1, q8, s8, qkv0, qkv, att, h2, q8b, s8b, mid, cache, h3 = block(eng, h, y, st)
    gate, shift, scale = st["mod"].split(D, 1)
    par = dict(gate_mod=gate, mod_shift=shift, mod_scale=scale)
    rh, sh, rn, sn = gate_norm64(h, y, "layer", "rms", 1.0, 1e-6, S, **par)
    near(h1, rh, 2.0**-19 * sh)
    again, n = eng.op_gate_norm(h, y, pre="layer", post="rms", rows_per_batch=S, **par)
    near(n, rn, 2.0**-19 * sn)
    assert torch.equal(again, h1) and all(torch.equal(a, b) for a, b in zip((q8, s8), quantized(n)))
    pre, size = product64(q8, s8, *st["qkv"], st["b_qkv"])
    near(qkv0, pre, 2.0**-20 * size)
    heads0, heads = qkv0.view(B, S, 3, H, Dh), qkv.view(B, S, 3, H, Dh)
    for i in (0, 1):
        near(heads[:, :, i], rope64(heads0[:, :, i], st["table"], "half"), 6 * STEP * heads0[:, :, i].double().abs().amax(-1, keepdim=True))
    assert torch.equal(heads[:, :, 2], heads0[:, :, 2])
    q, k, v = (heads[:, :, i].double().transpose(1, 2).contiguous() for i in range(3))
    p = torch.softmax(torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(Dh), -1)
    ref = torch.matmul(p, v).transpose(1, 2).reshape(B * S, D)
    assert float((att.double() - ref).norm() / ref.norm()) <= {"float16": 6e-4, "bfloat16": 4.5e-3}[dtype_name]  # the attention's own bound (test_gpu_ops.py)
    g = gate.double().repeat_interleave(S, 0)
    o, size = product64(*quantized(att), *st["o"], None)
    near(h2, h1.double() + g * o.to(dt).double(), 4 * STEP * g.abs() * size + g.abs() * eps * o.abs())  # o itself is not kept: its rounding may be the other one
    _, n = eng.op_gate_norm(h2, pre="rms")
    _, _, rn, sn = gate_norm64(h2, None, "rms", "none", 1.0, 1e-6, 1)
    near(n, rn, 2.0**-19 * sn)
    assert all(torch.equal(a, b) for a, b in zip((q8b, s8b), quantized(n)))
    pre, size = product64(q8b, s8b, *st["up"], st["b_up"])
    near(mid, gelu64(pre), 2.0**-20 * size)
    pre, size = product64(*quantized(mid), *st["down"], None)
    near(cache, pre, 2.0**-20 * size)
    near(h3, h2.double() + st["gate"].double() * cache.double(), 4 * STEP * (st["gate"].double() * cache.double()).abs())


def test_a_block_captured_replayed_and_on_another_stream():
    """Captured into one graph and replayed with eager work in between; eager on a side stream; two graphs that share nothing run in turn: the same bits every time."""
    dt, eng = torch.float16, small_engine("float16")
    st, h, y = block_state(eng, dt, seed=20)
    other, h2, y2 = block_state(eng, dt, B=1, S=257, seed=40)
    eager, eager2 = block(eng, h, y, st), block(eng, h2, y2, other)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        apart = block(eng, h, y, st)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(apart, eager))
    graphs = []
    for state, hh, yy in ((st, h, y), (other, h2, y2)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = block(eng, hh, yy, state)
        graphs.append((g, outs))
    for turn in range(4):
        for (g, outs), ref in zip(graphs, (eager, eager2)):
            for o in outs:
                o.fill_(float("nan") if o.is_floating_point() else 99)
            g.replay()
            assert all(torch.equal(a, b) for a, b in zip(block(eng, h, y, st), eager))  # eager work behind the replay
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, ref)), turn


def test_calls_on_two_streams_at_once():
    eng = small_engine("bfloat16")
    dt = torch.bfloat16
    streams = [torch.cuda.Stream() for _ in range(2)]
    states = [block_state(eng, dt, B=1, S=150, seed=60 + 20 * i) for i in range(2)]
    alone = [block(eng, h, y, st) for st, h, y in states]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(3):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                outs[i].append(block(eng, states[i][1], states[i][2], states[i][0]))
    torch.cuda.synchronize()
    for i in range(2):
        for got in outs[i]:
            assert all(torch.equal(a, b) for a, b in zip(got, alone[i]))


def test_two_threads_share_an_engine():
    """Calls and refusals of two threads on one engine: results are right, and each thread is told what it did wrong itself."""
    eng, dt = small_engine("float16"), torch.float16
    x = rand(64, 64, seed=1, dtype=dt)
    q, s = eng.op_quantize_int8(x)
    rq, rs = quantized(x)
    wrong = []

    def quantiser():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(300):
                try:
                    eng.op_quantize_int8(x, out=(x.view(torch.int8)[:, :64], s))
                except ValueError as e:
                    wrong.extend([str(e)] if "quantize_int8" not in str(e) else [])
                out = eng.op_quantize_int8(x)
            torch.cuda.current_stream().synchronize()
            wrong.extend(["quantised"] if not (torch.equal(out[0], rq) and torch.equal(out[1], rs)) else [])

    def norm():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(300):
                try:
                    eng.op_gate_norm(x, pre="rms", out_n=x)
                except ValueError as e:
                    wrong.extend([str(e)] if "gate_norm" not in str(e) else [])
                n = eng.op_gate_norm(x, pre="layer")[1]
            torch.cuda.current_stream().synchronize()
            wrong.extend(["norm"] if not torch.equal(n, first) else [])

    first = eng.op_gate_norm(x, pre="layer")[1]
    torch.cuda.synchronize()
    threads = [threading.Thread(target=f) for f in (quantiser, norm)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong



def test_refusals_reach_the_caller():
    eng = small_engine("float16")
    h = rand(2, 40000, seed=1, dtype=torch.float16)
    with pytest.raises(ValueError, match="32768"):
        eng.op_gate_norm(h, pre="rms")
    with pytest.raises(ValueError, match="few-rows"):
        eng.op_gemm_int8(0, int8_rows(33, 16, 1), torch.ones(33, device="cuda"), int8_rows(4, 16, 2), torch.ones(4, device="cuda"), kernel="rows")
    with pytest.raises(ValueError, match="multiple of 16"):
        eng.op_gemm_int8(0, torch.zeros(4, 40, dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda"), int8_rows(4, 40, 2), torch.ones(4, device="cuda"))
    with pytest.raises(ValueError, match="table has 3 rows"):
        eng.op_rope(rand(1, 4, 1, 8, dtype=torch.float16), None, torch.zeros(3, 4, 2, device="cuda"))
    with pytest.raises(ValueError, match="is on cpu"):
        eng.op_quantize_int8(torch.zeros(2, 8, dtype=torch.float16))


@pytest.mark.parametrize("dtype_name", DTYPES)
def test_gate_norm_modulations_shared_by_all_samples(dtype_name):
    """A modulation expanded over the samples; a shared one beside one per sample is refused, as modulations it would be read with the other's stride, and goes into its table."""
    dt, eng = getattr(torch, dtype_name), small_engine(dtype_name)
    M, D, rows = 37, 200, 10
    h, y, par = norm_inputs(M, D, dt, 4, dict(mod_shift=True, mod_scale=True, gate_mod=True), seed=11)
    own_shift, own_scale = par["mod_shift"], par["mod_scale"]
    one = dict(mod_shift=own_shift[1:2], mod_scale=own_scale[2:3])
    shared = {k: v.expand(4, D) for k, v in one.items()}
    for par in (dict(shared, gate_mod=par["gate_mod"][:1].expand(4, D)), dict(mod_shift=shared["mod_shift"]), dict(mod_scale=shared["mod_scale"])):
        nh, n = eng.op_gate_norm(h, y, pre="layer", rows_per_batch=rows, **par)
        rh, sh, rn, sn = gate_norm64(h, y, "layer", "none", 1.0, 1e-6, rows, **par)
        near(nh, rh, 2.0**-19 * sh)
        near(n, rn, 2.0**-19 * sn)
    for mixed in (dict(mod_shift=shared["mod_shift"], mod_scale=own_scale), dict(mod_shift=own_shift, mod_scale=shared["mod_scale"])):
        for quantize in (False, True):
            with pytest.raises(ValueError, match="same stride"):
                eng.op_gate_norm(h, y, pre="layer", rows_per_batch=rows, quantize=quantize, **mixed)
        nh, n = eng.op_gate_norm(h, y, pre="layer", rows_per_batch=M, **mixed)  # all rows are one sample's: the strides do not matter
        rh, sh, rn, sn = gate_norm64(h, y, "layer", "none", 1.0, 1e-6, M, **mixed)
        near(n, rn, 2.0**-19 * sn)
    for mixed in (dict(table_shift=one["mod_shift"][0].float(), mod_scale=own_scale), dict(mod_shift=own_shift, table_scale=one["mod_scale"][0].float())):
        nh, n = eng.op_gate_norm(h, y, pre="layer", rows_per_batch=rows, **mixed)
        rh, sh, rn, sn = gate_norm64(h, y, "layer", "none", 1.0, 1e-6, rows, **mixed)
        near(n, rn, 2.0**-19 * sn)
        _, (q, s) = eng.op_gate_norm(h, y, pre="layer", rows_per_batch=rows, quantize=True, **mixed)
        assert all(torch.equal(a, b) for a, b in zip((q, s), quantized(n)))
