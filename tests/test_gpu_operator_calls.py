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


def test_rope_table_of_positions_without_a_place_in_the_turn():
    """Beyond 2^53 quarters the angle's 64 bits do not say where in the turn it is; cosine and sine are still those of one angle: each within 4.5 * 2^-24, so their squares' sum
    within 2 * 4.5 * 2^-24 * (|c| + |s|) <= 13 * 2^-24 of 1."""
    pos = torch.tensor([2.0**49, 2.0**50, 2.0**51, 2.0**52, 1e16, 1e17, -1e17, 1.3e18, -1.3e18, 1e20, 7e25, 1e30, -2e35, 3.4e38], device="cuda")
    for dims in (2, 64):
        table = small_engine().op_rope_table(pos, dims, theta=500000.0).double()
        assert float(((table**2).sum(-1) - 1).abs().max()) <= 13 * STEP
    near_ones = torch.tensor([2.0**30, -(2.0**33), 2.0**36], device="cuda")  # the angle is off by 2^-53 of it at most: 2^-17 at 2^36
    ref, _ = table64(near_ones, (2,))
    assert float((small_engine().op_rope_table(near_ones, 2).double() - ref).abs().max()) <= 4.5 * STEP + 2.0**-17


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rope_in_place_through_another_view(layout):
    """One token a sample, one sample, one head: the stride of such a dimension differs from view to view and means nothing."""
    eng, dt = small_engine("float16"), torch.float16
    table = eng.op_rope_table(torch.arange(9, device="cuda", dtype=torch.int32) + 5, 24)
    for B, S, H in ((4, 1, 3), (1, 9, 3), (5, 9, 1), (1, 1, 1)):
        wide = rand(B, S, 2 * H, 24, seed=B + S, dtype=dt)
        q, k = wide[:, :, :H], wide[:, :, H:]
        expected = eng.op_rope(q, k, table, layout=layout)
        strides = [x if n > 1 else 7 + i for i, (n, x) in enumerate(zip(q.shape, q.stride()))]
        outs = tuple(x.as_strided(x.shape, strides, x.storage_offset()) for x in (q, k))
        assert outs[0].stride() != q.stride()
        eng.op_rope(q, k, table, layout=layout, out=outs)
        assert torch.equal(q, expected[0]) and torch.equal(k, expected[1])


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rope_with_an_empty_table(layout):
    """Every index lies outside it: no token turns."""
    eng, q = small_engine("float16"), rand(2, 5, 3, 24, seed=1, dtype=torch.float16)
    table, index = torch.empty(0, 8, 2, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda")
    out, _ = eng.op_rope(q, None, table, layout=layout, index=index)
    assert torch.equal(out, q)
    x = q.clone()
    eng.op_rope(x, None, table, layout=layout, index=index, out=(x, None))
    assert torch.equal(x, q)
    with pytest.raises(ValueError, match="0 rows for 5 tokens"):
        eng.op_rope(q, None, table, layout=layout)
