"""The CPU's evaluation at the ends of the range: norms beyond fp32."""
import math

import pytest
import torch

from kharon_b200 import ops


@pytest.mark.parametrize("n", [1, 4, 1000])
def test_norm_beyond_the_range_of_fp32(n):
    """The norm shows as inf, its factor is what it is: 1 / norm, a subnormal fp32 number at most half a step of 2^-149 off."""
    t = torch.full((n,), 3e38)
    want = float(t[0].double()) * math.sqrt(n)
    out, sumsq = torch.zeros(2), torch.zeros(1, dtype=torch.float64)
    ops.grad_norm(ops.TensorList([t]), out, max_norm=1.0, sumsq=sumsq)
    assert float(out[0]) == pytest.approx(want, rel=1e-6) if want < 3.4e38 else math.isinf(float(out[0]))
    assert abs(float(out[1]) - 1.0 / want) <= 2 ** -150 and float(sumsq) == pytest.approx(want ** 2, rel=1e-12)
    first = out.clone()
    ops.clip_factor(sumsq, out.zero_(), 1.0)
    assert torch.equal(out, first)
    ops.clip_grads(ops.TensorList([t]), 1e38, out)
    assert float(t.double().norm()) == pytest.approx(1e38, rel=1e-6)


def test_norm_and_factor_of_another_shape():
    """``out`` is two values, whatever its shape."""
    t, out = torch.full((4,), 2.0), torch.zeros(1, 2)
    ops.clip_grads(ops.TensorList([t]), 1.0, out)
    assert out.tolist() == [[4.0, 0.25]] and t.tolist() == [0.5] * 4
