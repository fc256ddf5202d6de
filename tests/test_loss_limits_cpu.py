"""The CPU's evaluation at the ends of the range: norms beyond fp32, rows with an infinite logit."""
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


INF = math.inf
ROWS = [[INF, 0.0, 1.0, 2.0], [0.0, INF, -INF, INF], [-INF] * 4, [math.nan, 0.0, 1.0, 2.0], [0.0, math.nan, INF, 1.0]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t", [0, 1, 3])
def test_rows_with_an_infinite_logit_are_nan(t, dtype):
    """What log softmax gives, whatever the target, on a GPU too; the other rows are as without them."""
    x = torch.cat([torch.tensor(ROWS), torch.tensor([[0.0, 1.0, 2.0, -INF]])]).to(dtype)
    R, tgt = x.shape[0], torch.full((x.shape[0],), t, dtype=torch.int32)
    for kw in (dict(), dict(old_logp=torch.full((R,), -1.0)), dict(old_logp=torch.full((R,), -1.0), ref_logp=torch.full((R,), -1.0), beta=0.5)):
        out = {k: torch.zeros(R) for k in ("rowloss", "logp")}
        grad = torch.zeros(R, 8, dtype=dtype)
        ops.policy_loss(x, 4, tgt, torch.ones(R), dlogits=grad, **out, **kw)
        assert bool(torch.isnan(out["logp"][:5]).all()) and bool(torch.isnan(out["rowloss"][:5]).all()) and bool(torch.isnan(grad[:5, :4]).all()) and not bool(grad[:, 4:].any())
        assert float(out["logp"][5]) == pytest.approx(float(torch.log_softmax(x[5].float(), -1)[t]), rel=1e-6)
    logp, loss, grad = torch.zeros(R), torch.zeros(R // 2), torch.zeros(R, 8, dtype=dtype)
    ops.preference_loss(x, 4, tgt, torch.arange(R + 1, dtype=torch.int32), loss=loss, logp=logp, dlogits=grad)
    assert bool(torch.isnan(logp[:5]).all()) and bool(torch.isnan(loss).all()) and bool(torch.isnan(grad[:5, :4]).all())
