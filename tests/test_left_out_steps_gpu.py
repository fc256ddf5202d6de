"""Steps that are left out because the gradient's norm is not finite, on a GPU: those behind them are the steps of a run that never had them."""
import math

import pytest
import torch

from kharon_b200 import ops
from kharon_b200.engine import TrainEngine
from kharon_b200.utils.rng import Rng

pytestmark = pytest.mark.gpu
DEV = "cuda"
KW = dict(layers=2, d_model=256, heads=4, vocab=1000, seq=64, mbatch=2, n_micro=2, device="cuda:0", lr=1e-3, max_norm=0.5)


def test_counts():
    t, out, n, sq = torch.ones(4, device=DEV), torch.zeros(2, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.float64, device=DEV)
    lst = ops.TensorList([t])
    for v, want in ((1.0, 0), (math.inf, 1), (2.0, 1), (math.nan, 2), (3e38, 2)):
        t[1] = v
        ops.grad_norm(lst, out, max_norm=1.0, sumsq=sq, left_out=n)
        assert int(n) == want
        ops.grad_norm(lst, out, max_norm=1.0)                      # (without it nothing is counted)
        assert int(n) == want
    sq.fill_(math.inf)
    ops.clip_factor(sq, out, 1.0, left_out=n)
    assert int(n) == 3 and math.isnan(float(out[1]))
    with pytest.raises(ValueError):
        ops.grad_norm(lst, out, left_out=n.cpu())
    with pytest.raises(ValueError):
        ops.clip_factor(sq, out, 1.0, left_out=n.cpu())
    with pytest.raises(ValueError):
        ops.adamw(t, t.clone(), t.clone(), t.clone(), None, lr=1, beta1=0, beta2=0, eps=1, wd=0, step=1, factor=out[1:], left_out=n.cpu())
    ops.check_device_status()


@pytest.mark.parametrize("n", [5, 4096, 100003])
@pytest.mark.parametrize("step,left", [(2, 1), (7, 0), (1000, 37), (5, 4), (100000, 3)])
def test_adamw_counts_the_steps_that_were_taken(n, step, left):
    """The same moments, to the bit.  The bias corrections are powers in 64 bits by squaring, here, and by the host's function, each rounded once to fp32: one fp32 step of
    2^-23 apart at most each, which the update lr m / bc1 / (sqrt(v / bc2) + eps) + lr wd p passes on once and by a half, with a few roundings of its own."""
    mk = lambda: [torch.randn(n, generator=torch.Generator(device=DEV).manual_seed(i), device=DEV).abs() for i in range(4)]  # noqa: E731
    for b1, b2 in ((0.9, 0.95), (0.9, 0.999)):
        kw = dict(lr=1e-2, beta1=b1, beta2=b2, eps=1e-8, wd=0.1)
        x, y = mk(), mk()
        f = torch.tensor([0.25], device=DEV)
        pb, pb2 = (torch.zeros(n, device=DEV, dtype=torch.bfloat16) for _ in range(2))
        ops.adamw(*x, pb, step=step, factor=f, left_out=torch.tensor([left], dtype=torch.int32, device=DEV), **kw)
        ops.adamw(*y, pb2, step=step - left, factor=f, **kw)
        assert all(torch.equal(a, b) for a, b in zip(x[1:], y[1:]))
        p = mk()[0]
        moved = (y[0] - p).abs() + 0.1 * 1e-2 * p.abs()
        assert bool(((x[0] - y[0]).abs() <= moved * 2 ** -21 + p.abs() * 2 ** -23).all())
        if left == 0 or step - left == 1:                          # (nothing to round differently: 1 - beta)
            assert torch.equal(x[0], y[0]) and torch.equal(pb, pb2)


def test_engine():
    def make(data, bad):
        e = TrainEngine(**KW)
        sync = e._sync_sp_grads
        for s, (idx, tgt) in enumerate(data):
            def poisoned():
                sync()
                e.model.params.g[5] = math.inf
            e._sync_sp_grads = poisoned if s in bad else sync
            e.train_step(idx, tgt)
        return e
    r = Rng(3)
    tokens = KW["mbatch"] * KW["n_micro"] * KW["seq"]
    data = [tuple(t.pin_memory() for t in r.batch(tokens, KW["vocab"])) for _ in range(2)]
    a, b = make(data, (0,)), make(data[1:], ())
    assert int(a.model.left_out) == 1 and a.model.step == 2 and torch.equal(a.model.params.w, b.model.params.w) and torch.equal(a.model.params.wb, b.model.params.wb)
    assert a.grad_norm() == b.grad_norm()
    ops.check_device_status()
