"""The entry points of an 8-bit transformer block without a GPU: what they refuse (in the binding and in the library, before anything is launched) and what the timed
cases of perf/operators.py are made of."""
import ctypes as C
import random
import subprocess

import pytest
import torch

from ecad_amd import _lib as L
from ecad_amd.engine import EcadEngine, _overlap


class _NoLibrary:
    """Stands in for the shared library: a refused call must not reach it."""

    def __getattr__(self, name):
        def call(*args):
            raise AssertionError(f"{name} was called")

        return call


@pytest.fixture
def eng():
    e = object.__new__(EcadEngine)
    e.lib, e._h, e.dtype, e.device, e.cfg = _NoLibrary(), C.c_void_p(), torch.float16, torch.device("cpu"), L.EcadModelCfg()
    return e


def f16(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def i8(rows, width):
    return torch.zeros((rows, (width + 15) // 16 * 16), dtype=torch.int8)[:, :width]


f32 = torch.zeros


def test_quantize_refusals(eng):
    with pytest.raises(ValueError, match="torch.float16"):
        eng.op_quantize_int8(torch.zeros(4, 8))
    with pytest.raises(ValueError, match="shape"):
        eng.op_quantize_int8(f16(4, 8, 2))
    with pytest.raises(ValueError, match="dense last"):
        eng.op_quantize_int8(f16(8, 4).t())
    with pytest.raises(ValueError, match="gradient"):
        eng.op_quantize_int8(f16(4, 8).requires_grad_())
    with pytest.raises(ValueError, match="q must"):
        eng.op_quantize_int8(f16(4, 8), out=(i8(4, 9), f32(4)))
    with pytest.raises(ValueError, match="overlaps"):
        buf = f16(4, 16)
        eng.op_quantize_int8(buf, out=(buf.view(torch.int8)[:, :16], f32(4)))


def test_gemm_refusals(eng):
    a, w, sa, sw = i8(3, 40), i8(7, 40), f32(3), f32(7)
    call = lambda epi=0, **k: eng.op_gemm_int8(epi, *(k.pop(x, d) for x, d in (("a", a), ("sa", sa), ("w", w), ("sw", sw))), **k)  # noqa: E731
    for bad, match in [
        (dict(w=i8(7, 41)), "shape"),
        (dict(sa=f32(4)), "a_scale"),
        (dict(sw=None), "needed"),
        (dict(bias=f16(7)), "bias"),
        (dict(kernel="fast"), "unknown"),
        (dict(resid=f16(3, 7)), "epilogue 3"),
        (dict(epi=3), "needs resid"),
        (dict(epi=3, resid=f16(3, 8)), "resid"),
        (dict(epi=3, resid=f16(3, 7), gate_mod=f16(1, 7), rows_per_batch=2), "samples"),
        (dict(epi=3, resid=f16(3, 7), gate_mod=f16(1, 7), rows_per_batch=0), "rows_per_batch"),
        (dict(out=f16(1, 7).expand(3, 7)), "overlaps itself"),
        (dict(a=a.float()), "int8"),
    ]:
        with pytest.raises(ValueError, match=match):
            call(**bad)
    r = f16(3, 7)
    with pytest.raises(ValueError, match="overlaps"):
        call(epi=3, resid=r, out=r)
    with pytest.raises(ValueError, match="overlaps"):
        wide = f16(3, 14)
        call(epi=3, resid=r, resid_out=wide[:, :7], out=wide[:, 6:13])


def test_gate_norm_refusals(eng):
    h, y = f16(4, 24), f16(4, 24)
    for args, match in [
        ((h, f16(4, 23), {}), "shape"),
        ((h, y, dict(pre="batch")), "one of"),
        ((h, y, dict(pre_weight=f16(24))), "pre_weight"),
        ((h, y, dict(gate_mod=f16(24))), "samples"),
        ((h, y, dict(mod_shift=f16(3, 24))), "samples"),
        ((h, y, dict(mod_shift=f16(2, 24), mod_scale=f16(2, 48)[:, :24], rows_per_batch=2)), "same stride"),
        ((h, y, dict(pre="none", quantize=True)), "quantise"),
        ((h, None, dict(out_h=f16(4, 24))), "out_h"),
        ((h, y, dict(pre="none", out_n=f16(4, 24))), "out_n"),
        ((h, y, dict(out_h=y)), "overlaps"),
        ((h, y, dict(out_n=h)), "overlaps"),
        ((h, y, dict(out_h=h, out_n=h)), "overlaps"),
        ((h.double(), y, {}), "torch.float16"),
    ]:
        with pytest.raises(ValueError, match=match):
            eng.op_gate_norm(args[0], args[1], **args[2])


def test_rope_refusals(eng):
    q, k, t = f16(2, 3, 4, 16), f16(2, 3, 2, 16), f32(3, 8, 2)
    for args, kw, match in [
        ((q, f16(2, 3, 2, 8), t), {}, "k of shape"),
        ((q, k, f32(3, 8)), {}, "table"),
        ((q, k, t), dict(layout="full"), "layout"),
        ((q, k, t), dict(index=torch.zeros(4, dtype=torch.int32)), "index"),
        ((q, k, t), dict(index=torch.zeros(3, dtype=torch.int64)), "int32"),
        ((q, k, t), dict(out=(k, q)), "shape"),
        ((q, k, t), dict(out=(f16(2, 1, 4, 16).expand(2, 3, 4, 16), k)), "overlaps itself"),
        ((q[:, :2], k[:, :2], t), dict(out=(q[:, 1:], f16(2, 2, 2, 16))), "overlaps"),
        ((f16(3, 4, 16), k, t), {}, "shape"),
    ]:
        with pytest.raises(ValueError, match=match):
            eng.op_rope(*args, **kw)
    for args, kw, match in [
        ((torch.zeros(4, dtype=torch.int64), 16), {}, "int32"),
        ((torch.zeros(4, 2, dtype=torch.int32), 16), {}, "axes"),
        ((torch.zeros(4, dtype=torch.int32), 16), dict(scaling="cubic"), "unknown"),
    ]:
        with pytest.raises(ValueError, match=match):
            eng.op_rope_table(*args, **kw)


def test_overlap_sees_columns_side_by_side():
    qkv = torch.zeros(2, 5, 3 * 8)
    q, k, v = (qkv[:, :, 8 * i : 8 * i + 8].view(2, 5, 2, 4) for i in range(3))
    assert not _overlap(q, k) and not _overlap(k, v) and not _overlap(v, q) and _overlap(q, q)
    assert _overlap(qkv[:, :, :9], qkv[:, :, 8:]) and not _overlap(qkv[0], qkv[1]) and _overlap(qkv, qkv[1, 2])
    assert not _overlap(qkv[:, ::2], qkv[:, 1::2][:, :, :0]) and _overlap(qkv[:, 1:], qkv[:, :4])


# ---- the library's own checks: the functions behind the C entry points, called with a context that has no device (a refusal comes before any launch) -------------


class _Ctx(C.Structure):
    _fields_ = [("dtype", C.c_int), ("num_cus", C.c_int), ("stream", C.c_void_p)]


class _Quantize(C.Structure):
    _fields_ = [("x", C.c_void_p), ("ldx", C.c_int64), ("q", C.c_void_p), ("ldq", C.c_int64), ("scale", C.c_void_p), ("M", C.c_int), ("K", C.c_int)]


class _Gemm(C.Structure):
    _fields_ = [("A", C.c_void_p), ("lda", C.c_int64), ("sa", C.c_void_p), ("W", C.c_void_p), ("ldw", C.c_int64), ("sw", C.c_void_p), ("bias", C.c_void_p), ("out", C.c_void_p), ("ldo", C.c_int64),
                ("resid", C.c_void_p), ("ldr", C.c_int64), ("resid_out", C.c_void_p), ("ldro", C.c_int64), ("gate_table", C.c_void_p), ("gate_mod", C.c_void_p), ("gate_stride", C.c_int64),
                ("M", C.c_int), ("N", C.c_int), ("K", C.c_int), ("epi", C.c_int), ("rows_per_batch", C.c_int), ("kernel", C.c_int)]


class _Norm(C.Structure):
    _fields_ = L.EcadGateNorm._fields_


class _Table(C.Structure):
    _fields_ = [("positions", C.c_void_p), ("positions_float", C.c_int), ("axes_dims", C.POINTER(C.c_int32)), ("axes", C.c_int), ("S", C.c_int), ("scaling", C.c_int), ("table", C.c_void_p),
                ("theta", C.c_double), ("factor", C.c_double), ("original_length", C.c_double), ("beta_fast", C.c_double), ("beta_slow", C.c_double)]


class _Heads(C.Structure):
    _fields_ = [("x", C.c_void_p), ("out", C.c_void_p)] + [(n, C.c_int64) for n in ("sb", "ss", "sh", "ob", "os", "oh")] + [("H", C.c_int)]


class _Rope(C.Structure):
    _fields_ = [("q", _Heads), ("k", _Heads), ("table", C.c_void_p), ("index", C.c_void_p), ("index_stride", C.c_int64)] + [(n, C.c_int) for n in ("B", "S", "D", "rot", "table_rows", "half", "inverse")]


@pytest.fixture(scope="module")
def library():
    lib = L.load()
    names = {}
    for line in subprocess.run(["nm", "-D", "--defined-only", str(L.lib_path())], capture_output=True, text=True, check=True).stdout.splitlines():
        sym = line.split()[-1]
        for op in ("op_quantize_int8", "op_gemm_int8", "op_gate_norm", "op_rope_table", "op_rope"):
            if sym.startswith(f"_ZN4ecad{len(op)}{op}E"):
                names[op] = getattr(lib, sym)

    def call(op, record):
        msg = C.create_string_buffer(320)
        rc = names[op](C.byref(_Ctx(0, 256, None)), C.byref(record), msg)
        return rc, msg.value.decode()

    return call


AT = 1 << 20  # stands for a pointer: never followed


def test_library_refusals_quantize(library):
    good = dict(x=AT, ldx=40, q=AT, ldq=48, scale=AT, M=3, K=40)
    for bad in (dict(K=0), dict(K=131072), dict(M=-1), dict(x=None), dict(scale=None), dict(ldx=39), dict(ldq=40), dict(ldq=32), dict(q=AT + 8), dict(x=AT + 1)):
        rc, msg = library("op_quantize_int8", _Quantize(**{**good, **bad}))
        assert rc == L.ECAD_E_INVALID and "quantize_int8" in msg, (bad, rc, msg)
    assert library("op_quantize_int8", _Quantize(**{**good, "M": 0, "x": None}))[0] == 0


def test_library_refusals_gemm(library):
    good = dict(A=AT, lda=48, sa=AT, W=AT, ldw=48, sw=AT, out=AT, ldo=7, M=3, N=7, K=40, rows_per_batch=1)
    resid = dict(epi=3, resid=AT, ldr=7, resid_out=AT, ldro=7)
    for bad in (dict(K=0), dict(K=131072), dict(M=-1), dict(epi=4), dict(epi=-1), dict(A=None), dict(sw=None), dict(out=None), dict(lda=40), dict(lda=32), dict(ldw=56), dict(A=AT + 8), dict(W=AT + 1),
                dict(ldo=6), dict(out=AT + 1), dict(bias=AT + 2), {**resid, "resid": None}, {**resid, "resid_out": None}, {**resid, "ldr": 6}, {**resid, "rows_per_batch": 0}, dict(kernel=99), dict(lda=1 << 24)):
        rc, msg = library("op_gemm_int8", _Gemm(**{**good, **bad}))
        assert rc == L.ECAD_E_INVALID and "gemm_int8" in msg, (bad, rc, msg)
    rc, msg = library("op_gemm_int8", _Gemm(**{**good, "M": 65, "kernel": 1}))
    assert rc == L.ECAD_E_UNSUPPORTED and "64 rows" in msg
    for none in (dict(M=0), dict(N=0)):
        assert library("op_gemm_int8", _Gemm(**{**good, **none, "A": None}))[0] == 0


def test_library_refusals_gate_norm(library):
    good = dict(h=AT, ldh=24, y=AT, ldy=24, h_out=AT, ldho=24, n_out=AT, ldn=24, M=4, D=24, rows_per_batch=1, post=1, pre=2, resid_scale=1.0, eps=1e-6)
    for bad in (dict(D=0), dict(M=-1), dict(post=3), dict(pre=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(resid_scale=float("inf")), dict(rows_per_batch=0), dict(y=None), dict(h_out=None),
                dict(n_out=None), dict(q=AT, ldq=32, q_scale=AT), dict(n_out=None, q=AT, ldq=32), dict(n_out=None, q=AT, ldq=24, q_scale=AT), dict(n_out=None, q=AT + 4, ldq=32, q_scale=AT), dict(pre=0),
                dict(post=0, post_weight=AT), dict(ldh=23), dict(ldy=1), dict(ldho=23), dict(ldn=8), dict(h=AT + 1), dict(gate_table=AT + 2), dict(mod_shift=AT + 1),
                dict(y=None, post=0, resid_scale=0.5), dict(y=None, post=0, gate_mod=AT), dict(y=None, post=0, pre=0, n_out=None)):
        rc, msg = library("op_gate_norm", _Norm(**{**good, **bad}))
        assert rc == L.ECAD_E_INVALID and "gate_norm" in msg, (bad, rc, msg)
    rc, msg = library("op_gate_norm", _Norm(**{**good, **{k: 40000 for k in ("D", "ldh", "ldy", "ldho", "ldn")}}))
    assert rc == L.ECAD_E_UNSUPPORTED and "32768" in msg
    assert library("op_gate_norm", _Norm(**{**good, "M": 0, "h": None}))[0] == 0


def test_library_refusals_rope(library):
    dims = (C.c_int32 * 2)(16, 56)
    good = dict(positions=AT, axes_dims=dims, axes=2, S=5, table=AT, theta=1e4, factor=1.0)
    for bad in (dict(axes=0), dict(axes=9), dict(S=-1), dict(theta=0.0), dict(factor=0.0), dict(factor=float("nan")), dict(scaling=4), dict(scaling=3, factor=2.0), dict(axes_dims=(C.c_int32 * 2)(16, 3)),
                dict(axes_dims=(C.c_int32 * 2)(0, 2)), dict(axes_dims=(C.c_int32 * 2)(512, 2)), dict(positions=None), dict(table=AT + 4),
                dict(scaling=3, factor=2.0, original_length=64.0, beta_fast=1.0, beta_slow=1.0), dict(scaling=3, factor=0.5, original_length=64.0, beta_fast=32.0, beta_slow=1.0)):
        rc, msg = library("op_rope_table", _Table(**{**good, **bad}))
        assert rc == L.ECAD_E_INVALID and "rope_table" in msg, (bad, rc, msg)
    assert library("op_rope_table", _Table(**{**good, "S": 0}))[0] == 0

    heads = dict(x=AT, out=2 * AT, sb=192, ss=64, sh=16, ob=192, os=64, oh=16)
    good = dict(q=_Heads(**heads, H=4), k=_Heads(**heads, H=2), table=AT, B=2, S=3, D=16, rot=16, table_rows=3)
    for bad in (dict(D=1), dict(rot=3), dict(rot=0), dict(rot=18), dict(q=_Heads(**heads, H=0)), dict(k=_Heads(**heads, H=-1)), dict(q=_Heads(**{**heads, "x": None}, H=4)), dict(table=None),
                dict(table_rows=2), dict(q=_Heads(**{**heads, "out": AT}, H=4)), dict(B=-1), dict(q=_Heads(**{**heads, "out": AT + 1}, H=4)),
                dict(q=_Heads(**{**heads, "out": AT, "oh": 32}, H=4), k=_Heads(H=0))):
        rc, msg = library("op_rope", _Rope(**{**good, **bad}))
        assert rc == L.ECAD_E_INVALID and "rope" in msg, (bad, rc, msg)
    for none in (dict(B=0), dict(S=0)):
        assert library("op_rope", _Rope(**{**good, **none}))[0] == 0


def test_struct_layouts_match_the_header():
    """EcadGateNorm as ctypes lays it out: what the C compiler makes of include/ecad_hip.h."""
    import tempfile
    from pathlib import Path

    root = Path(__file__).resolve().parents[1]
    with tempfile.TemporaryDirectory() as d:
        src = Path(d) / "t.c"
        fields = [n for n, _ in L.EcadGateNorm._fields_]
        src.write_text('#include "ecad_hip.h"\n#include <stdio.h>\nint main(void) { printf("%zu", sizeof(EcadGateNorm)); ' + "".join(f'printf(" %zu", offsetof(EcadGateNorm, {n}));' for n in fields) + " return 0; }\n")
        subprocess.run(["gcc", "-I", str(root / "include"), str(src), "-o", str(Path(d) / "t")], check=True)
        sizes = list(map(int, subprocess.run([str(Path(d) / "t")], capture_output=True, text=True, check=True).stdout.split()))
    assert sizes == [C.sizeof(L.EcadGateNorm)] + [getattr(L.EcadGateNorm, n).offset for n in fields]


def test_timed_cases_stay_in_their_ranges():
    from perf import operators

    listed = operators.listed()
    names = [c["name"] for c in listed]
    assert len(set(names)) == len(names) and not operators.own
    most = {k: max(operators.work(c)[k] for c in listed) for k in ("bytes", "flops")}
    for seed in range(300):
        case = operators.draw(random.Random(seed))
        work = operators.work(case)
        assert work["bytes"] <= 1.05 * most["bytes"] and work["flops"] <= 1.05 * most["flops"], case
