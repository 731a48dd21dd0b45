"""Calls of the operators of an 8-bit transformer block that the documentation allows, without a GPU: an engine whose library answers that all is well."""
import torch

from test_cpu_operators import accepting, f16, f32, i8  # noqa: F401  (accepting: a fixture)


def test_no_rows_into_given_8bit_outputs(accepting):  # noqa: F811
    """An empty tensor has no address: that is not the absence of a scale."""
    x, q, s = f16(4, 24), i8(4, 24), f32(4)
    out = (q[:0], s[:0])
    got = accepting.op_quantize_int8(x[:0], out=out)
    assert got[0] is out[0] and got[1] is out[1]
    _, got = accepting.op_gate_norm(x[:0], pre="rms", quantize=True, out_n=out)
    assert got[0] is out[0] and got[1] is out[1]
