"""Calls of the operators of an 8-bit transformer block that the documentation allows (-m gpu); tolerances as in test_gpu_operators.py."""
import pytest
import torch

from gpu_util import small_engine
from test_gpu_operators import DTYPES, STEP, gate_norm64, near, quantized, rand, rope64, table64  # noqa: F401

pytestmark = pytest.mark.gpu


def test_no_rows():
    """Nothing is done, whatever else the call asks for."""
    eng, dt = small_engine("float16"), torch.float16
    x = rand(4, 24, seed=1, dtype=dt)
    q, s = torch.full((4, 32), 9, device="cuda", dtype=torch.int8), torch.full((4,), 9.0, device="cuda")
    out = (q[:0, :24], s[:0])
    assert eng.op_quantize_int8(x[:0], out=out)[0] is out[0]
    assert eng.op_gate_norm(x[:0], pre="rms", quantize=True, out_n=out)[1][1] is out[1]
    for kw in (dict(pre="rms", post="rms"), dict(pre="layer", gate_table=torch.ones(24, device="cuda")), dict(pre="rms", resid_scale=0.5)):
        nh, n = eng.op_gate_norm(x[:0], x[:0], **kw)
        assert nh.shape == n.shape == (0, 24)
    nh, n = eng.op_gate_norm(x[:0], x[:0], pre="none")
    assert nh.shape == (0, 24) and n is None
    torch.cuda.synchronize()
    assert bool((q == 9).all()) and bool((s == 9).all())
