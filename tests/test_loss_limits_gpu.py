"""Losses of a policy at the ends of the range: slopes among and below the smallest normal fp32 numbers, rows with an infinite logit."""
import math

import pytest
import torch

from kharon_b200 import ops
from policy_exact import check_policy, check_preference, policy, preference
from test_policy_gpu import DEV, HALF, run_policy, run_preference, starts_of

pytestmark = pytest.mark.gpu

# Slopes from the smallest normal fp32 number down to 0: a margin, or a log ratio, of 84 to 112 in steps of a half (bf16 holds these between 64 and 128).
FAR = [84.0 + 0.5 * k for k in range(57)]


def far_rows(V, ld, seed):
    """A row for each of FAR in turn, flat, of some spread and nearly certain of another column than the target, which is column 0."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.zeros(len(FAR), 3, ld, device=DEV, dtype=torch.bfloat16)
    x[:, 1, :V] = (torch.randn(len(FAR), V, generator=g, device=DEV) * 4).bfloat16()
    x[:, 2, V - 1] = 30.0
    return x


@pytest.mark.parametrize("V,ld,times", [(8, 8, 1), (250, 256, 1), (250, 256, 120), (1003, 1008, 1), (2040, 2040, 1), (5000, 5000, 1), (9001, 9008, 1), (50257, 50304, 1),
                                        (128256, 128256, 1)])
def test_policy_loss_with_slopes_at_the_end_of_the_range(V, ld, times):
    """Ratios exp(-84) to exp(-112), which the clamp doesn't hold where A > 0: gradients of next to nothing, whatever is left of the slope in fp32.  The gradient's bound is
    policy_exact's (2^-126 and what the formula gives); the ratio's own relative error, 2^-17 of an argument of about 100, is far below that."""
    x = far_rows(V, ld, V).repeat(1, times, 1).view(-1, ld)
    R = x.shape[0]
    t = torch.zeros(R, dtype=torch.int32, device=DEV)
    far = torch.tensor(FAR, dtype=torch.float64, device=DEV).repeat_interleave(3 * times)
    lp = policy(x, V, t)["logp"]
    for scale in (1.0, 4.0, -0.25):
        for add in (0.0, 2.0):
            adv, old = torch.full((R,), scale, device=DEV), (lp + far + add).float()
            out, want = run_policy(x, V, t, adv, old, weight=torch.full((R,), 0.5, device=DEV)), policy(x, V, t, adv, old, uniform=0.5)
            check_policy({k: out[k] for k in ("logp", "clipped", "grad")}, want, V, HALF)


@pytest.mark.parametrize("V,ld", [(8, 8), (250, 256), (500, 504), (1003, 1008), (2040, 2040), (5000, 5000), (9001, 9008), (50257, 50304)])
def test_preference_loss_with_slopes_at_the_end_of_the_range(V, ld):
    """Margins of 84 to 112 and a little more: slopes exp(-margin) from 2^-121 down to 0."""
    x = torch.stack([far_rows(V, ld, V), far_rows(V, ld, V + 1)], 2)                     # [margin, form, chosen | rejected, ld]
    x[:, :, 1, 0] = x[:, :, 1, 0] - torch.tensor(FAR, device=DEV)[:, None].bfloat16()
    x = x.view(-1, ld)
    P = x.shape[0] // 2
    t, starts = torch.zeros(2 * P, dtype=torch.int32, device=DEV), starts_of([1] * (2 * P))
    for kw in (dict(beta=1.0), dict(beta=1.0, uniform=0.125), dict(beta=1.0, uniform=3.0)):
        out, want = run_preference(x, V, t, starts, **kw), preference(x, V, t, starts, **kw)
        check_preference(out, want, V, starts, kw["beta"], 0.0, None, kw.get("uniform", 1.0), HALF)
    ops.check_device_status()


@pytest.mark.parametrize("V,ld", [(8, 8), (250, 256), (1003, 1008), (2040, 2040), (5000, 5000), (9001, 9008), (50257, 50304), (128256, 128256)])
def test_rows_with_an_infinite_logit_are_nan(V, ld):
    """As on the CPU: NaN in all that is written of the row, whatever its target, and in its pair's other row by the pair's slope; zeros beyond the vocabulary."""
    x = torch.zeros(10, ld, device=DEV, dtype=torch.bfloat16)
    x[0, 3], x[1, V - 1], x[2, 0], x[3, :V], x[4, V // 2] = math.inf, math.inf, math.inf, -math.inf, math.nan
    x[1, 4] = -math.inf
    t = torch.tensor([3, 0, 1, 2, V - 1, 0, 0, 0, 0, 0], device=DEV, dtype=torch.int32)
    old = torch.full((10,), -8.0, device=DEV)
    for kw in (dict(), dict(old=old), dict(old=old, ref=old, beta=0.5)):
        out = run_policy(x, V, t, torch.ones(10, device=DEV), **kw)
        assert all(bool(torch.isnan(out[k][:5]).all()) and bool(torch.isfinite(out[k][5:]).all()) for k in ("loss", "logp"))
        assert bool(torch.isnan(out["grad"][:5, :V]).all()) and bool(torch.isfinite(out["grad"][5:]).all()) and not bool(out["grad"][:, V:].any())
    out = run_preference(x, V, t, starts_of([1] * 10))
    assert bool(torch.isnan(out["logp"][:5]).all()) and bool(torch.isnan(out["loss"][:3]).all()) and bool(torch.isnan(out["grad"][:6, :V]).all())
    assert bool(torch.isfinite(out["loss"][3:]).all()) and bool(torch.isfinite(out["grad"][6:]).all()) and not bool(out["grad"][:, V:].any())
    ops.check_device_status()
