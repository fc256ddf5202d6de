"""Clipped updates of the trainer on two ranks against one rank with all prompts: gradients, weights and the statistics that are shared."""
import datetime
import os
import sys
import tempfile

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from test_parallel_cpu import ROOT, _free_port
from test_preference_ranks_cpu import PROMPTS, REWARDS, _trainer

KW = dict(clip_eps=0.05, inner=3, max_norm=0.5)


def _worker(rank, port, out_dir):
    sys.path.insert(0, ROOT)
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE="2", LOCAL_RANK=str(rank))
    dist.init_process_group("gloo", rank=rank, world_size=2, timeout=datetime.timedelta(seconds=60))
    t, grads = _trainer(REWARDS["uneven"][rank], rank * PROMPTS, dp_group=dist.group.WORLD, dp_rank=rank, dp=2, **KW)
    st = t.grpo_step(1)
    torch.save(dict(grads=grads, stats=st, w=t.policy.params.w.clone(), norm=float(t.norm_out[0])), os.path.join(out_dir, "r%d.pt" % rank))
    dist.barrier()
    dist.destroy_process_group()


def test_clipped_updates_are_the_same_on_two_ranks():
    one, grads = _trainer([p for r in REWARDS["uneven"] for p in r], 0, **KW)
    st = one.grpo_step(1)
    assert len(grads) == 3 and st["clipped"] > 0 and float(grads[0].abs().max()) > 0
    with tempfile.TemporaryDirectory() as d:
        mp.spawn(_worker, args=(_free_port(), d), nprocs=2, join=True)
        res = [torch.load(os.path.join(d, "r%d.pt" % r), weights_only=False) for r in range(2)]
    assert torch.equal(res[0]["w"], res[1]["w"]) and res[0]["norm"] == res[1]["norm"]
    for r in res:
        # fp32 sums in another order; the later updates pass the earlier ones' differences on
        for a, b, tol in zip(r["grads"], grads, (1e-5, 1e-4, 1e-4)):
            assert float((a - b).abs().max()) <= tol * float(b.abs().max())
        for k in ("loss", "kl", "mean_reward"):
            assert r["stats"][k] == pytest.approx(st[k], rel=1e-4, abs=1e-6)
        assert abs(r["stats"]["clipped"] - st["clipped"]) <= 1e-6
