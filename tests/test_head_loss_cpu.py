"""GPT.backward with another loss than the cross-entropy: what belongs to the cross-entropy is refused, not passed over."""
import pytest
import torch

from kharon_b200 import ops
from kharon_b200.models import GPT, Config


@pytest.mark.parametrize("kw", [dict(coef=torch.ones(16)), dict(loss_scale=1.0), dict(inv_mb=0.5), dict(accumulate_loss=True)], ids=lambda kw: next(iter(kw)))
def test_arguments_of_the_cross_entropy_are_refused(kw):
    m = GPT(Config(1, 32, 2, 64, 8, 2), "cpu", torch.float32)
    m.init_weights(1)
    idx = torch.arange(16, dtype=torch.int32)
    m.set_input(idx, idx)
    m.forward(compute_loss=False)
    with pytest.raises(ValueError):
        m.backward(head_loss=lambda x, V, t: ops.policy_loss(x, V, t, torch.ones(2), dlogits=x), **kw)
    assert not bool(m.params.g.any())
    m.backward(head_loss=lambda x, V, t: ops.policy_loss(x, V, t, torch.ones(2), dlogits=x))
    assert bool(m.params.g.any())
