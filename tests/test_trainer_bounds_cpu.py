"""The bound on the gradient holds for every update of the trainer."""
import pytest
import torch

from kharon_b200.rl import AddTask, GRPOTrainer

TOP = 1e-3


def test_supervised_steps_are_bounded():
    """Adam's first moment of the first step is (1 - beta1) times the gradient that it was given: its norm is the bound, each element rounded twice on the way."""
    mk = lambda **kw: GRPOTrainer(AddTask(), layers=1, d_model=32, heads=2, G=4, prompts=4, device="cpu", dtype=torch.float32, **kw)  # noqa: E731
    free, loose, bound = mk(), mk(max_norm=1e6), mk(max_norm=TOP)
    for t in (free, loose, bound):
        t.sft_step()
    norm = float(free.policy.params.m.double().norm()) / (1 - 0.9)
    assert norm > TOP and torch.equal(free.policy.params.w, loose.policy.params.w)
    assert float(bound.policy.params.m.double().norm()) / (1 - 0.9) == pytest.approx(TOP, rel=1e-5)
    assert float(bound.norm_out[0]) == pytest.approx(norm, rel=1e-5)
