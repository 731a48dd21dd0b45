"""Calls of the operators of an 8-bit transformer block that the documentation allows, without a GPU: an engine whose library answers that all is well."""
import ctypes as C
import subprocess
import sys
import threading
import time
from pathlib import Path

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from ecad_amd import _lib as L
from ecad_amd.engine import EcadEngine
from test_cpu_operators import AT, _Norm, accepting, eng, f16, f32, i8, library  # noqa: F401  (accepting, eng, library: fixtures)


def test_no_rows_into_given_8bit_outputs(accepting):  # noqa: F811
    """An empty tensor has no address: that is not the absence of a scale."""
    x, q, s = f16(4, 24), i8(4, 24), f32(4)
    out = (q[:0], s[:0])
    got = accepting.op_quantize_int8(x[:0], out=out)
    assert got[0] is out[0] and got[1] is out[1]
    _, got = accepting.op_gate_norm(x[:0], pre="rms", quantize=True, out_n=out)
    assert got[0] is out[0] and got[1] is out[1]


@pytest.mark.parametrize("asks", [dict(post=1), dict(post=2, post_weight=AT), dict(pre=0, n_out=None), dict(gate_table=AT), dict(gate_mod=AT), dict(resid_scale=0.5)])
def test_no_rows_of_a_sublayer(library, asks):  # noqa: F811
    """h and y of zero rows have no addresses, and a NULL y is not a call without y there."""
    norm = dict(h=AT, ldh=24, y=2 * AT, ldy=24, h_out=AT, ldho=24, n_out=2 * AT, ldn=24, M=4, D=24, rows_per_batch=1, post=0, pre=2, resid_scale=1.0, eps=1e-6)
    empty = dict(M=0, h=None, y=None, h_out=None, n_out=None)
    assert library("op_gate_norm", _Norm(**{**norm, **asks, **empty})) == (0, "")
    rc, msg = library("op_gate_norm", _Norm(**{**norm, **asks, "y": None}))
    assert rc == L.ECAD_E_INVALID and "without y" in msg


def test_forward_mode_tangents_are_refused(accepting):  # noqa: F811
    """Of a tensor, of what it is a view of, of an output that would be written behind its tangent; not where forward gradients are switched off."""
    h, w = f16(4, 24), f32(24)
    with forward_ad.dual_level():
        dual, wide = forward_ad.make_dual(h, f16(4, 24)), forward_ad.make_dual(f16(4, 48), f16(4, 48))
        for call in [lambda: accepting.op_gate_norm(dual), lambda: accepting.op_gate_norm(wide[:, :24]), lambda: accepting.op_gate_norm(h, pre_weight=forward_ad.make_dual(w, w)),
                     lambda: accepting.op_gate_norm(h, h.clone(), out_h=dual), lambda: accepting.op_quantize_int8(dual)]:
            with pytest.raises(ValueError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):  # no_grad is the other mode's
                call()
            with torch.inference_mode():
                call()
        accepting.op_gate_norm(forward_ad.unpack_dual(dual).primal)


def test_tracing_is_refused(accepting):  # noqa: F811
    """A tracer would record the allocation of the result and nothing that fills it."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    h, out = f16(4, 24), f16(4, 24)
    norm = lambda x: accepting.op_gate_norm(x)[1]  # noqa: E731
    for trace in (lambda: make_fx(norm)(h), lambda: make_fx(norm, tracing_mode="fake")(h), lambda: torch.jit.trace(norm, (h,), check_trace=False)):
        with pytest.raises(RuntimeError, match="traced"):
            trace()
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        with pytest.raises(RuntimeError, match="traced"):
            norm(h)
        with pytest.raises(RuntimeError, match="traced"):
            accepting.op_gate_norm(h, out_n=out)  # nothing fake in it: it would run
    fake = mode.from_tensor(h)
    for call in (lambda: norm(fake), lambda: accepting.op_gate_norm(h, pre_weight=mode.from_tensor(f32(24))), lambda: torch.func.functionalize(norm)(h)):
        with pytest.raises(RuntimeError, match="holds no values"):
            call()
    for transform in (lambda: torch.func.jvp(norm, (h,), (h,)), lambda: torch.func.grad(lambda x: norm(x).sum())(h), lambda: torch.vmap(norm)(f16(2, 4, 24))):
        with pytest.raises(RuntimeError):
            transform()
    assert not accepting.calls.records


def test_modes_that_only_watch_are_not_tracing(accepting):  # noqa: F811
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with Watch():
        accepting.op_gate_norm(f16(4, 24))
    assert len(accepting.calls.records) == 1


def test_lazily_negated_tensors_are_refused(accepting):  # noqa: F811
    """Their memory holds the values with the other sign, a zero tensor's holds nothing."""
    h, w = f16(4, 24), torch.complex(torch.ones(1), torch.ones(1)).conj().imag
    assert w.is_neg() and w.is_contiguous()
    for call in [lambda: accepting.op_gate_norm(f16(4, 1), pre_weight=w), lambda: accepting.op_gate_norm(h, h.clone(), out_h=torch._neg_view(h)), lambda: accepting.op_quantize_int8(torch._neg_view(h)),
                 lambda: accepting.op_quantize_int8(torch._efficientzerotensor(4, 24, dtype=torch.float16))]:
        with pytest.raises(ValueError, match="lazily negated"):
            call()
    accepting.op_gate_norm(f16(4, 1), pre_weight=w.resolve_neg())


def test_what_is_written_in_place_has_a_new_version(accepting, eng):  # noqa: F811
    """Autograd's saved tensors are checked by it."""
    h, y, n, q8, s = f16(4, 24), f16(4, 24), f16(4, 24), i8(4, 24), f32(4)
    w, sw, r, r2, o, t, pos = i8(24, 24), f32(24), f16(4, 24), f16(4, 24), f16(4, 24), f32(3, 8, 2), torch.zeros(3, dtype=torch.int32)
    q, k, q2, k2 = f16(2, 3, 4, 16), f16(2, 3, 2, 16), f16(2, 3, 4, 16), f16(2, 3, 2, 16)
    for outs, ins, call in [
        ([q8, s], [h], lambda e: e.op_quantize_int8(h, out=(q8, s))),
        ([o], [q8, s, w, sw], lambda e: e.op_gemm_int8(0, q8, s, w, sw, out=o)),
        ([r], [q8, s, w, sw], lambda e: e.op_gemm_int8(3, q8, s, w, sw, resid=r)),
        ([r2, o], [r], lambda e: e.op_gemm_int8(3, q8, s, w, sw, resid=r, resid_out=r2, out=o)),
        ([h, y], [], lambda e: e.op_gate_norm(h, y, out_h=h, out_n=y)),
        ([n], [h], lambda e: e.op_gate_norm(h, out_n=n)),
        ([q8, s], [h], lambda e: e.op_gate_norm(h, quantize=True, out_n=(q8, s))),
        ([t], [pos], lambda e: e.op_rope_table(pos, 16, out=t)),
        ([q, k], [t], lambda e: e.op_rope(q, k, t, out=(q, k))),
        ([q2, k2], [q, k, t], lambda e: e.op_rope(q, k, t, out=(q2, k2))),
    ]:
        before = [x._version for x in outs + ins]
        call(accepting)
        assert [x._version - b for x, b in zip(outs + ins, before)] == [1] * len(outs) + [0] * len(ins)
        before = [x._version for x in outs]
        with pytest.raises(RuntimeError, match="was called"):  # a launch that failed has written nothing
            call(eng)
        assert [x._version for x in outs] == before
    wide = f16(4, 48)
    accepting.op_gate_norm(h, out_n=wide[:, :24])  # a view's version is its base's
    assert wide._version == 1
    x = torch.ones(4, 24, dtype=torch.float16, requires_grad=True)
    product = x * h
    accepting.op_gate_norm(h, y, out_h=h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
    with torch.inference_mode():
        inside = f16(4, 24)
        accepting.op_gate_norm(h, out_n=inside)
    accepting.op_gate_norm(h, out_n=inside)  # no version to count


def test_every_thread_finds_its_own_message():
    """Calls that fail in two threads at once; both without a device (no configuration, and a device that is not there)."""
    lib, wrong = L.load(), []

    def fail(call, says):
        for _ in range(4000):
            if call() == 0 or lib.ecad_last_error(None) not in says:
                wrong.append(lib.ecad_last_error(None))
                return

    cfg, handle = L.EcadModelCfg(), C.c_void_p()
    calls = [(lambda: lib.ecad_create(None, 0, None), (b"NULL argument",)), (lambda: lib.ecad_create(C.byref(cfg), 1 << 20, C.byref(handle)), (b"no HIP device visible", b"device index out of range"))]
    threads = [threading.Thread(target=fail, args=c) for c in calls * 2]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    assert calls[0][0]() != 0 and lib.ecad_last_error(None) == b"NULL argument"
    seen = []
    t = threading.Thread(target=lambda: seen.append(lib.ecad_last_error(None)))  # a thread that had none: the last one of all
    t.start()
    t.join()
    assert seen == [b"NULL argument"]


@pytest.fixture
def waiting(tmp_path):
    """An engine whose launches wait (20 s at most) until `go` is set, as one does while the device's queue is full; `entered` and `left` count them, `destroyed` is what `left`
    was when the engine went."""
    (tmp_path / "waiting.c").write_text("""#include <stdatomic.h>
#include <unistd.h>
atomic_int entered, left, go, destroyed = -1;
int launch(void) {
  ++entered;
  for (int i = 0; i < 20000 && !go; ++i) usleep(1000);
  ++left;
  return 0;
}
const char* last_error(void* e) { return ""; }
void destroy(void* e) { destroyed = left; }
""")
    subprocess.run(["gcc", "-shared", "-fPIC", str(tmp_path / "waiting.c"), "-o", str(tmp_path / "waiting.so")], check=True)
    lib, ops = C.CDLL(str(tmp_path / "waiting.so")), L.load_ops()
    at = lambda name: C.cast(getattr(lib, name), C.c_void_p).value  # noqa: E731
    e = object.__new__(EcadEngine)
    e._h, e.cfg, e._donor = C.c_void_p(1 << 20), L.EcadModelCfg(), None
    e.lib = type("Library", (), {"ecad_destroy": staticmethod(lib.destroy)})
    e._ops = ops, ops.engine((at("launch"),) * 5 + (at("last_error"),), 1 << 20, L.ECAD_DTYPE_F16, -1, lambda index: 0)
    e.count = lambda name: C.c_int.in_dll(lib, name)
    yield e
    e.count("go").value = 1


def until(condition):
    while not condition():
        time.sleep(0.001)


def test_a_launch_that_waits_stops_no_other_thread(waiting):
    x = f16(4, 24)
    caller = threading.Thread(target=lambda: waiting.op_quantize_int8(x))
    caller.start()
    until(lambda: waiting.count("entered").value)
    assert waiting.count("left").value == 0  # this thread runs beside the launch
    waiting.count("go").value = 1
    caller.join()
    assert waiting.count("left").value == 1


def test_closing_waits_for_the_calls_of_other_threads(waiting):
    x, seen = f16(4, 24), []

    def call():
        waiting.op_quantize_int8(x)
        try:
            waiting.op_quantize_int8(x)
        except RuntimeError as e:
            seen.append(str(e))

    callers = [threading.Thread(target=call) for _ in range(2)]
    for t in callers:
        t.start()
    until(lambda: waiting.count("entered").value == 2)
    closer = threading.Thread(target=waiting.close)
    closer.start()
    until(lambda: not waiting._h.value)
    time.sleep(0.1)  # (it is in close() by now)
    assert closer.is_alive() and waiting.count("destroyed").value == -1
    waiting.count("go").value = 1
    for t in (closer, *callers):
        t.join()
    assert seen == ["the engine is closed"] * 2 and waiting.count("entered").value == 2 and waiting.count("destroyed").value == 2
    with pytest.raises(RuntimeError, match="closed"):
        waiting.op_quantize_int8(x)
    waiting.close()


def test_first_calls_of_several_threads_share_one_handle(waiting, monkeypatch):
    """close() waits for the calls on the handle it knows: the first calls of two threads must not make one each."""
    made = []

    class Ops:
        @staticmethod
        def engine(*args):
            time.sleep(0.05)
            made.append(args)
            return object()

        @staticmethod
        def close(engine):
            pass

    monkeypatch.setattr(L, "load_ops", lambda: Ops)
    waiting.lib = type("Library", (), {"ecad_destroy": waiting.lib.ecad_destroy, **{n: C.CFUNCTYPE(C.c_int)(lambda: 0) for n in (
        "ecad_op_quantize_int8", "ecad_op_gemm_int8", "ecad_op_gate_norm", "ecad_op_rope_table", "ecad_op_rope", "ecad_last_error")}})
    waiting._ops, waiting.dtype, waiting.device_index, handles = None, torch.float16, 0, []
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    threads = [threading.Thread(target=lambda: handles.append(waiting._native())) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 1 and all(h is handles[0] for h in handles) and len(handles) == 4


def test_the_library_is_built_without_torch():
    """The default target where Python has no torch (here: no site packages) is the library alone; where it has, the binding too, without a path to that torch in it."""
    root = Path(__file__).resolve().parents[1]
    make = lambda python: subprocess.run(["make", "-n", "-B", "-C", str(root / "ecad_amd" / "csrc"), f"PYTHON={python}"], capture_output=True, text=True)  # noqa: E731
    without, beside = make(f"{sys.executable} -I -S"), make(sys.executable)
    for run in (without, beside):
        assert run.returncode == 0 and not run.stderr and "operators.hip" in run.stdout and "-o ../libecad_hip.so" in run.stdout, run.stderr
    assert "binding.cpp" not in without.stdout and "no torch" in without.stdout
    assert "binding.cpp" in beside.stdout
    dynamic = subprocess.run(["readelf", "-d", str(root / "ecad_amd" / "_ops.so")], capture_output=True, text=True, check=True).stdout
    assert "RPATH" not in dynamic and "RUNPATH" not in dynamic


def test_the_accumulator_audit_covers_every_unit():
    """scripts/audit_agpr.py by itself compiles what the Makefile does, with its flags."""
    root = Path(__file__).resolve().parents[1]
    sys.path.insert(0, str(root / "scripts"))
    try:
        import audit_agpr
    finally:
        sys.path.pop(0)
    run = subprocess.run(["make", "-n", "-B", "-C", str(root / "ecad_amd" / "csrc")], capture_output=True, text=True, check=True).stdout
    built = {}
    for line in run.splitlines():
        if "-save-temps -c ../" in line:
            built[line.split("-save-temps -c ../")[1].split()[0]] = set(line.split("hipcc ")[1].split(" -save-temps")[0].split())
    assert set(built) == set(audit_agpr.UNITS)
    for unit, flags in built.items():
        assert flags - {"-Wall", "-Wno-unused-function"} == set(audit_agpr.UNITS[unit]) - {"-S", "--cuda-device-only"}, unit
