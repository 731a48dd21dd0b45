"""The entry points of an 8-bit transformer block without a GPU: what they refuse (in the binding and in the library, before anything is launched) and what the timed
cases of perf/operators.py are made of."""
import ctypes as C
import random
import struct
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from ecad_amd import _lib as L
from ecad_amd.engine import EcadEngine


class _Calls:
    """Stands in for the shared library: five entry points that say that they were called (a refused call does not get that far)."""

    def __init__(self):
        P, I, I64, D = C.c_void_p, C.c_int, C.c_int64, C.c_double
        prototypes = {"quantize_int8": [P, P, I64, P, I64, P, I, I, P], "gemm_int8": [P, P, P], "gate_norm": [P, P, P], "rope_table": [P, P, I, P, I, I, I, D, D, D, D, D, P, P], "rope": [P, P, P]}
        self.last = C.create_string_buffer(64)
        self.kept = []
        for name, types in prototypes.items():
            def call(*args, name=name):
                self.last.value = f"{name} was called".encode()
                return L.ECAD_E_HIP

            self.kept.append(C.CFUNCTYPE(I, *types)(call))
        self.kept.append(C.CFUNCTYPE(P, P)(lambda handle: C.addressof(self.last)))
        self.addresses = tuple(C.cast(f, P).value for f in self.kept)


@pytest.fixture
def eng():
    """An engine without a device: CPU tensors are 'its' tensors, and a call that passes the checks ends in a RuntimeError that names it."""
    calls, ops = _Calls(), L.load_ops()
    e = object.__new__(EcadEngine)
    e._h, e.cfg, e.calls = C.c_void_p(), L.EcadModelCfg(), calls
    e._ops = ops, ops.engine(calls.addresses, 1 << 20, L.ECAD_DTYPE_F16, -1, lambda index: 0)
    return e


def f16(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def i8(rows, width):
    return torch.zeros((rows, (width + 15) // 16 * 16), dtype=torch.int8)[:, :width]


f32 = torch.zeros


def test_quantize_refusals(eng):
    with pytest.raises(ValueError, match="torch.float16"):
        eng.op_quantize_int8(torch.zeros(4, 8))
    with pytest.raises(ValueError, match="two dimensions"):
        eng.op_quantize_int8(f16(4, 8, 2))
    with pytest.raises(ValueError, match="dense last"):
        eng.op_quantize_int8(f16(8, 4).t())
    with pytest.raises(ValueError, match="gradient"):
        eng.op_quantize_int8(f16(4, 8).requires_grad_())
    with pytest.raises(ValueError, match="q must"):
        eng.op_quantize_int8(f16(4, 8), out=(i8(4, 9), f32(4)))


def test_gemm_refusals(eng):
    a, w, sa, sw = i8(3, 40), i8(7, 40), f32(3), f32(7)
    call = lambda epi=0, **k: eng.op_gemm_int8(epi, *(k.pop(x, d) for x, d in (("a", a), ("sa", sa), ("w", w), ("sw", sw))), **k)  # noqa: E731
    for bad, match in [
        (dict(w=i8(7, 41)), "w must have shape"),
        (dict(sa=f32(4)), "a_scale"),
        (dict(sw=None), "needed"),
        (dict(a=None), "a is needed"),
        (dict(w=[1]), "must be a tensor, got list"),
        (dict(bias=f16(7)), "bias"),
        (dict(kernel="fast"), "unknown"),
        (dict(resid=f16(3, 7)), "epilogue 3"),
        (dict(epi=3), "needs resid"),
        (dict(epi=3, resid=f16(3, 8)), "resid"),
        (dict(epi=3, resid=f16(3, 7), gate_mod=f16(1, 7), rows_per_batch=2), "samples"),
        (dict(epi=3, resid=f16(3, 7), gate_mod=f16(1, 7), rows_per_batch=0), "rows_per_batch"),
        (dict(out=f16(3, 8)), "out must"),
        (dict(a=a.float()), "int8"),
    ]:
        with pytest.raises(ValueError, match=match):
            call(**bad)


def test_gate_norm_refusals(eng):
    h, y = f16(4, 24), f16(4, 24)
    for args, match in [
        ((h, f16(4, 23), {}), "shape"),
        ((h, y, dict(pre="batch")), "one of"),
        ((h, y, dict(pre_weight=f16(24))), "pre_weight"),
        ((h, y, dict(gate_mod=f16(24))), "two dimensions"),
        ((h, y, dict(mod_shift=f16(3, 24))), "samples"),
        ((h, y, dict(mod_shift=f16(2, 24), mod_scale=f16(2, 48)[:, :24], rows_per_batch=2)), "same stride"),
        ((h, y, dict(pre="none", quantize=True)), "quantize"),
        ((h, None, dict(out_h=f16(4, 24))), "out_h"),
        ((h, y, dict(pre="none", out_n=f16(4, 24))), "out_n"),
        ((h, y, dict(out_n=f16(3, 24))), "out_n"),
        ((h, y, dict(quantize=True, out_n=(i8(4, 24), None))), "out_n"),
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
        ((q, k, t), dict(out=(q, None)), "k_out"),
        ((q.requires_grad_(False), k, f32(3, 8, 2).requires_grad_()), {}, "gradient"),
        ((q, k, torch.zeros(2, 3, 8).permute(1, 2, 0)), {}, "contiguous"),
        ((q, None, t), dict(out=(q.transpose(1, 2), None)), "shape"),
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


# ---- the library's own checks: the functions behind the C entry points, called with a context that has no device (a refusal comes before any launch) -------------


class _Ctx(C.Structure):
    _fields_ = [("dtype", C.c_int), ("num_cus", C.c_int), ("stream", C.c_void_p)]


class _Quantize(C.Structure):
    _fields_ = [("x", C.c_void_p), ("ldx", C.c_int64), ("q", C.c_void_p), ("ldq", C.c_int64), ("scale", C.c_void_p), ("M", C.c_int), ("K", C.c_int)]


class _Packed:
    """One of the records that the binding packs by struct, by member name."""

    def __init__(self, layout, names, **values):
        assert set(values) <= set(names), set(values) - set(names)
        self.data = layout.pack(*(values.get(n) or 0 for n in names))


# the argument records of include/ecad_hip.h: members in the header's order, and their struct codes (P pointer, q int64, i int32, f float; no padding)
GEMM = "A lda a_scale W ldw w_scale bias out ldo resid ldr resid_out ldro gate_table gate_mod gate_mod_stride M N K epi rows_per_batch kernel".split()
NORM = ("h ldh y ldy h_out ldho n_out ldn q ldq q_scale post_weight pre_weight gate_table gate_mod gate_mod_stride table_shift table_scale mod_shift mod_scale mod_stride "
        "M D rows_per_batch post pre reserved resid_scale eps").split()
HEADS = "x out sample token head out_sample out_token out_head H".split()
_HEADS = "PPqqqqqqq"
INT8_GEMM_CODES = struct.Struct("PqPPqPPPqPqPqPPqiiiiii")
GATE_NORM_CODES = struct.Struct("PqPqPqPqPqPPPPPqPPPPqiiiiiiff")
ROPE_CODES = struct.Struct(_HEADS + _HEADS + "PPqiiiiiiii")
ROPE = [f"{t}.{n}" for t in "qk" for n in HEADS] + "table index index_stride B S D rot table_rows half inverse reserved".split()


def _Gemm(**v):
    return _Packed(INT8_GEMM_CODES, GEMM, **v)


def _Norm(**v):
    return _Packed(GATE_NORM_CODES, NORM, **v)


def _Rope(q, k, **v):
    return _Packed(ROPE_CODES, ROPE, **{f"q.{n}": x for n, x in q.items()}, **{f"k.{n}": x for n, x in k.items()}, **v)


class _Table(C.Structure):
    _fields_ = [("positions", C.c_void_p), ("positions_float", C.c_int), ("axes_dims", C.POINTER(C.c_int32)), ("axes", C.c_int), ("S", C.c_int), ("scaling", C.c_int), ("table", C.c_void_p),
                ("theta", C.c_double), ("factor", C.c_double), ("original_length", C.c_double), ("beta_fast", C.c_double), ("beta_slow", C.c_double)]


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
        rc = names[op](C.byref(_Ctx(0, 256, None)), record.data if isinstance(record, _Packed) else C.byref(record), msg)
        return rc, msg.value.decode()

    return call


AT = 1 << 20  # stands for a pointer: never followed


def test_library_refusals_quantize(library):
    good = dict(x=AT, ldx=40, q=2 * AT, ldq=48, scale=3 * AT, M=3, K=40)
    for bad in (dict(K=0), dict(K=131072), dict(M=-1), dict(x=None), dict(scale=None), dict(ldx=39), dict(ldq=40), dict(ldq=32), dict(q=2 * AT + 8), dict(x=AT + 1),
                dict(q=AT), dict(q=AT + 32), dict(scale=AT + 8), dict(scale=2 * AT + 132)):
        rc, msg = library("op_quantize_int8", _Quantize(**{**good, **bad}))
        assert rc == L.ECAD_E_INVALID and "quantize_int8" in msg, (bad, rc, msg)
    assert library("op_quantize_int8", _Quantize(**{**good, "M": 0, "x": None}))[0] == 0


def test_library_refusals_gemm(library):
    good = dict(A=AT, lda=48, a_scale=AT, W=AT, ldw=48, w_scale=AT, out=2 * AT, ldo=7, M=3, N=7, K=40, rows_per_batch=1)
    resid = dict(epi=3, resid=3 * AT, ldr=7, resid_out=3 * AT, ldro=7)
    for bad in (dict(K=0), dict(K=131072), dict(M=-1), dict(epi=4), dict(epi=-1), dict(A=None), dict(w_scale=None), dict(out=None), dict(lda=40), dict(lda=32), dict(ldw=56), dict(A=AT + 8), dict(W=AT + 1),
                dict(ldo=6), dict(out=AT + 1), dict(bias=AT + 2), {**resid, "resid": None}, {**resid, "resid_out": None}, {**resid, "ldr": 6}, {**resid, "rows_per_batch": 0}, dict(kernel=99), dict(lda=1 << 24),
                dict(out=AT), dict(out=AT + 100), dict(bias=2 * AT + 40), dict(w_scale=2 * AT), {**resid, "out": 3 * AT}, {**resid, "resid_out": 3 * AT + 2}, {**resid, "resid_out": 2 * AT},
                {**resid, "ldro": 8}, {**resid, "gate_table": 3 * AT + 40}, {**resid, "gate_mod": 3 * AT, "gate_mod_stride": 7}):
        rc, msg = library("op_gemm_int8", _Gemm(**{**good, **bad}))
        assert rc == L.ECAD_E_INVALID and "gemm_int8" in msg, (bad, rc, msg)
    rc, msg = library("op_gemm_int8", _Gemm(**{**good, "M": 33, "kernel": 1}))
    assert rc == L.ECAD_E_UNSUPPORTED and "32 rows" in msg
    for none in (dict(M=0), dict(N=0)):
        assert library("op_gemm_int8", _Gemm(**{**good, **none, "A": None}))[0] == 0


def test_library_refusals_gate_norm(library):
    good = dict(h=AT, ldh=24, y=2 * AT, ldy=24, h_out=AT, ldho=24, n_out=2 * AT, ldn=24, M=4, D=24, rows_per_batch=1, post=1, pre=2, resid_scale=1.0, eps=1e-6)
    for bad in (dict(D=0), dict(M=-1), dict(post=3), dict(pre=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(resid_scale=float("inf")), dict(rows_per_batch=0), dict(y=None), dict(h_out=None),
                dict(n_out=None), dict(q=AT, ldq=32, q_scale=AT), dict(n_out=None, q=AT, ldq=32), dict(n_out=None, q=AT, ldq=24, q_scale=AT), dict(n_out=None, q=AT + 4, ldq=32, q_scale=AT), dict(pre=0),
                dict(post=0, post_weight=AT), dict(ldh=23), dict(ldy=1), dict(ldho=23), dict(ldn=8), dict(h=AT + 1), dict(gate_table=AT + 2), dict(mod_shift=AT + 1),
                dict(y=None, post=0, resid_scale=0.5), dict(y=None, post=0, gate_mod=AT), dict(y=None, post=0, pre=0, n_out=None),
                dict(h_out=2 * AT), dict(n_out=AT), dict(h_out=AT + 2), dict(ldho=25), dict(n_out=2 * AT + 20), dict(pre_weight=AT + 96), dict(gate_mod=2 * AT, gate_mod_stride=24),
                dict(n_out=None, q=AT, ldq=32, q_scale=4 * AT), dict(n_out=None, q=3 * AT, ldq=32, q_scale=3 * AT), dict(n_out=None, q=3 * AT, ldq=32, q_scale=2 * AT)):
        rc, msg = library("op_gate_norm", _Norm(**{**good, **bad}))
        assert rc == L.ECAD_E_INVALID and "gate_norm" in msg, (bad, rc, msg)
    rc, msg = library("op_gate_norm", _Norm(**{**good, **{k: 40000 for k in ("D", "ldh", "ldy", "ldho", "ldn")}}))
    assert rc == L.ECAD_E_UNSUPPORTED and "32768" in msg
    assert library("op_gate_norm", _Norm(**{**good, "M": 0, "h": None}))[0] == 0


def test_library_refusals_rope(library):
    dims = (C.c_int32 * 2)(16, 56)
    good = dict(positions=AT, axes_dims=dims, axes=2, S=5, table=2 * AT, theta=1e4, factor=1.0)
    for bad in (dict(axes=0), dict(axes=9), dict(S=-1), dict(theta=0.0), dict(factor=0.0), dict(factor=float("nan")), dict(scaling=4), dict(scaling=3, factor=2.0), dict(axes_dims=(C.c_int32 * 2)(16, 3)),
                dict(axes_dims=(C.c_int32 * 2)(0, 2)), dict(axes_dims=(C.c_int32 * 2)(512, 2)), dict(positions=None), dict(table=2 * AT + 4), dict(table=AT + 8),
                dict(scaling=3, factor=2.0, original_length=64.0, beta_fast=1.0, beta_slow=1.0), dict(scaling=3, factor=0.5, original_length=64.0, beta_fast=32.0, beta_slow=1.0)):
        rc, msg = library("op_rope_table", _Table(**{**good, **bad}))
        assert rc == L.ECAD_E_INVALID and "rope_table" in msg, (bad, rc, msg)
    assert library("op_rope_table", _Table(**{**good, "S": 0}))[0] == 0

    heads = dict(x=AT, out=2 * AT, sample=192, token=64, head=16, out_sample=192, out_token=64, out_head=16, H=4)
    good = dict(q=heads, k=dict(heads, x=3 * AT, out=4 * AT, H=2), table=5 * AT, B=2, S=3, D=16, rot=16, table_rows=3)
    wide = dict(heads, sample=288, token=96, out_sample=288, out_token=96)  # q and k as columns of one buffer, in place
    side = dict(good, q=dict(wide, out=AT), k=dict(wide, x=AT + 128, out=AT + 128, H=2))
    for bad in (dict(D=1), dict(rot=3), dict(rot=0), dict(rot=18), dict(q=dict(heads, H=0)), dict(k=dict(heads, H=-1)), dict(q=dict(heads, x=None)), dict(table=None), dict(table_rows=2),
                dict(q=dict(heads, out=AT)), dict(B=-1), dict(q=dict(heads, out=2 * AT + 1)), dict(q=dict(heads, out=AT, out_head=32), k={}), dict(q=dict(heads, out_head=8), k={}),
                dict(q=dict(heads, out_sample=0), k={}), dict(q=dict(heads, out=AT + 32), k={}), dict(q=dict(heads, out=3 * AT)), dict(k=dict(heads, x=3 * AT, out=2 * AT + 64, H=2)),
                dict(table=2 * AT), dict(index=2 * AT + 4), dict(side, k=dict(wide, x=AT + 96, out=AT + 96, H=2))):
        rc, msg = library("op_rope", _Rope(**{**good, **bad}))
        assert rc == L.ECAD_E_INVALID and "rope" in msg, (bad, rc, msg)
    for none in (dict(B=0), dict(S=0)):
        assert library("op_rope", _Rope(**{**good, **none}))[0] == 0


def test_struct_layouts_match_the_header():
    """The records of these tests and of anyone who binds the library without a C compiler: sizes and offsets as the C compiler lays out include/ecad_hip.h."""
    import tempfile
    from pathlib import Path

    root = Path(__file__).resolve().parents[1]
    records = {"EcadInt8Gemm": (INT8_GEMM_CODES, GEMM), "EcadGateNorm": (GATE_NORM_CODES, NORM), "EcadRope": (ROPE_CODES, ROPE)}
    with tempfile.TemporaryDirectory() as d:
        src = Path(d) / "t.c"
        body = "".join(f'printf("%zu", sizeof({r})); ' + "".join(f'printf(" %zu", offsetof({r}, {n}));' for n in names) + ' printf("\\n");' for r, (_, names) in records.items())
        src.write_text('#include "ecad_hip.h"\n#include <stdio.h>\nint main(void) { ' + body + " return 0; }\n")
        subprocess.run(["gcc", "-I", str(root / "include"), str(src), "-o", str(Path(d) / "t")], check=True)
        lines = subprocess.run([str(Path(d) / "t")], capture_output=True, text=True, check=True).stdout.splitlines()
    for line, (layout, names) in zip(lines, records.values()):
        size, *offsets = map(int, line.split())
        codes = layout.format
        assert len(codes) == len(names) and layout.size == size
        assert offsets == [struct.calcsize(codes[:i] + "0" + c) if i else 0 for i, c in enumerate(codes)]


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


def test_gradients_are_refused_while_they_are_recorded(eng):
    """Under no_grad a parameter may be passed; the call then reaches the library."""
    x = f16(4, 16).requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        eng.op_gate_norm(f16(4, 16), x)
    with pytest.raises(ValueError, match="gradient"):
        eng.op_gate_norm(f16(4, 16), pre_weight=torch.ones(16, requires_grad=True))
    with torch.no_grad(), pytest.raises(RuntimeError, match="gate_norm was called"):
        eng.op_gate_norm(f16(4, 16), x, pre_weight=torch.ones(16, requires_grad=True))


def test_calls_that_fit_reach_the_library(eng):
    a, w, sa, sw, r = i8(3, 40), i8(7, 40), f32(3), f32(7), f16(3, 7)
    t, q, k, at = f32(3, 8, 2), f16(2, 3, 4, 16), f16(2, 3, 2, 20)[..., :16], torch.zeros(3, dtype=torch.int32)
    for name, call in [
        ("quantize_int8", lambda: eng.op_quantize_int8(f16(4, 9)[:, 1:])),
        ("quantize_int8", lambda: eng.op_quantize_int8(f16(4, 8), out=(i8(4, 8), f32(4)))),
        ("gemm_int8", lambda: eng.op_gemm_int8(1, a, sa, w, sw, f32(7), out=f16(3, 9)[:, :7], kernel="tile64")),
        ("gemm_int8", lambda: eng.op_gemm_int8(3, a, sa, w, sw, resid=r, gate_table=f32(7), gate_mod=f16(2, 20)[:, 3:10], rows_per_batch=2)),
        ("gate_norm", lambda: eng.op_gate_norm(f16(4, 8), f16(4, 8), pre="none", post="rms", post_weight=f32(8))),
        ("gate_norm", lambda: eng.op_gate_norm(f16(4, 8), quantize=True, out_n=(i8(4, 8), f32(4)))),
        ("rope_table", lambda: eng.op_rope_table(at, 16)),
        ("rope_table", lambda: eng.op_rope_table(f32(5, 3), [16, 56, 56], scaling="yarn", factor=2, original_length=64, out=f32(5, 64, 2))),
        ("rope", lambda: eng.op_rope(q, k, t, index=at)),
        ("rope", lambda: eng.op_rope(q, None, t, layout="half", index=at.expand(2, 3), inverse=True, out=(q, None))),
    ]:
        with pytest.raises(RuntimeError, match=f"^{name} was called"):
            call()


def test_wrong_kinds_of_arguments(eng):
    for call in [lambda: eng.op_gate_norm(f16(4, 8), rows_per_batch="2"), lambda: eng.op_gate_norm(f16(4, 8), eps="small"), lambda: eng.op_gemm_int8(None, i8(3, 40), f32(3), i8(7, 40), f32(7)),
                 lambda: eng.op_rope_table(f32(5), ("16",))]:
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError, match="out of range"):
        eng.op_gate_norm(f16(4, 8), rows_per_batch=1 << 40)
    eng._ops = eng._ops[0], None
    with pytest.raises(RuntimeError, match="closed"):
        eng.op_quantize_int8(f16(4, 8))
    with pytest.raises(RuntimeError, match="closed"):
        eng._ops = None
        eng.op_quantize_int8(f16(4, 8))


def test_native_calls_keep_reference_counts(eng):
    import sys

    x, out = f16(4, 16), (i8(4, 16), f32(4))
    before = [sys.getrefcount(o) for o in (x, out, *out, eng._ops[1], None)][:-1]
    for _ in range(50):
        with pytest.raises(RuntimeError):
            eng.op_quantize_int8(x, out=out)
        with pytest.raises(ValueError):
            eng.op_gate_norm(x, x[:2])
    assert [sys.getrefcount(o) for o in (x, out, *out, eng._ops[1], None)][:-1] == before


def test_library_refuses_negative_strides(library):
    gemm = dict(A=AT, lda=48, a_scale=AT, W=AT, ldw=48, w_scale=AT, out=2 * AT, ldo=7, M=3, N=7, K=40, rows_per_batch=1, epi=3, resid=3 * AT, ldr=7, resid_out=3 * AT, ldro=7, gate_mod=5 * AT)
    norm = dict(h=AT, ldh=24, y=2 * AT, ldy=24, h_out=AT, ldho=24, n_out=2 * AT, ldn=24, M=4, D=24, rows_per_batch=1, post=1, pre=2, resid_scale=1.0, eps=1e-6, gate_mod=5 * AT, mod_scale=6 * AT)
    heads = dict(x=AT, out=2 * AT, sample=192, token=64, head=16, out_sample=192, out_token=64, out_head=16, H=4)
    rope = dict(q=heads, k=dict(heads, x=3 * AT, out=4 * AT, H=2), table=5 * AT, B=2, S=3, D=16, rot=16, table_rows=3)
    calls = [("op_gemm_int8", _Gemm, dict(gemm, gate_mod_stride=-7)), ("op_gate_norm", _Norm, dict(norm, gate_mod_stride=-24)), ("op_gate_norm", _Norm, dict(norm, mod_stride=-24)),
             ("op_rope", _Rope, dict(rope, index=6 * AT, index_stride=-3))]
    calls += [("op_rope", _Rope, dict(rope, **{part: dict(rope[part], **{name: -16})})) for part in "qk" for name in ("sample", "token", "head", "out_head")]
    for name, struct_of, args in calls:
        rc, msg = library(name, struct_of(**args))
        assert rc == L.ECAD_E_INVALID and "negative" in msg, (name, args, rc, msg)


def test_generated_loops_are_what_their_generator_writes():
    """ecad_amd/csrc/gemm_int8_asm.h is generated and committed: `--check` writes it anew in memory and compares."""
    root = Path(__file__).resolve().parents[1]
    r = subprocess.run([sys.executable, str(root / "scripts" / "gen_gemm_i8.py"), "--check"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-400:]


# ---- calls that go through: an engine whose library answers that all is well ----------------------------------------------------------------------------------------


class _Accepts:
    """Five entry points that return 0; `records` holds what the three that take one were given, by member name."""

    def __init__(self):
        P, I, I64, D = C.c_void_p, C.c_int, C.c_int64, C.c_double
        self.records, self.kept = [], []

        def record_of(codes, names):
            def call(handle, record, stream):
                self.records.append(dict(zip(names, codes.unpack(C.string_at(record, codes.size)))))
                return 0

            return C.CFUNCTYPE(I, P, P, P)(call)

        self.kept.append(C.CFUNCTYPE(I, P, P, I64, P, I64, P, I, I, P)(lambda *args: 0))
        self.kept += [record_of(INT8_GEMM_CODES, GEMM), record_of(GATE_NORM_CODES, NORM)]
        self.kept.append(C.CFUNCTYPE(I, P, P, I, P, I, I, I, D, D, D, D, D, P, P)(lambda *args: 0))
        self.kept += [record_of(ROPE_CODES, ROPE), C.CFUNCTYPE(P, P)(lambda handle: None)]
        self.addresses = tuple(C.cast(f, P).value for f in self.kept)


@pytest.fixture
def accepting():
    calls, ops = _Accepts(), L.load_ops()
    e = object.__new__(EcadEngine)
    e._h, e.cfg, e.calls = C.c_void_p(), L.EcadModelCfg(), calls
    e._ops = ops, ops.engine(calls.addresses, 1 << 20, L.ECAD_DTYPE_F16, -1, lambda index: 0)
    return e


def test_modulations_reach_the_library_with_strides_that_hold_for_both(accepting):
    """Shift and scale have one stride between samples in the library: one that all samples share (stride 0) beside one per sample would be read past its end."""
    h, shared, own = f16(4, 24), f16(1, 24).expand(4, 24), f16(4, 72)[:, :24]
    for pair in ((shared, own), (own, shared)):
        for kw in ({}, dict(quantize=True)):
            with pytest.raises(ValueError, match="same stride"):
                accepting.op_gate_norm(h, mod_shift=pair[0], mod_scale=pair[1], **kw)
    assert not accepting.calls.records
    for kw, stride in [
        (dict(mod_shift=shared, mod_scale=shared), 0),
        (dict(mod_shift=own, mod_scale=own), 72),
        (dict(mod_shift=shared), 0),
        (dict(mod_scale=own), 72),
        (dict(mod_shift=shared, mod_scale=own, rows_per_batch=4), 0),  # one sample: nothing lies between samples
        (dict(mod_shift=f16(2, 24), mod_scale=own, rows_per_batch=5), 0),
        (dict(mod_shift=f16(1, 24), mod_scale=own, rows_per_batch=4), 0),
    ]:
        accepting.op_gate_norm(h, **kw)
        assert accepting.calls.records.pop()["mod_stride"] == stride, kw
