"""Preference updates of the trainer: every pair weighs the same wherever it was sampled, and a batch without a pair is no update."""
import datetime
import os
import sys
import tempfile

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from kharon_b200.rl import AddTask, GRPOTrainer
from test_parallel_cpu import ROOT, _free_port

G, PROMPTS = 4, 2                                  # of a rank
# rewards of the samples of two ranks' prompts: 4 pairs that count and 1; 4 and none; none at all
REWARDS = {"uneven": [[[1.0, 0.0, 0.5, 0.2], [0.0, 1.0, 0.5, 0.75]], [[0.0, 0.0, 1.0, 0.0], [1.0, 1.0, 1.0, 1.0]]],
           "one_rank": [[[1.0, 0.0, 0.5, 0.2], [0.0, 1.0, 0.5, 0.75]], [[0.0] * 4, [1.0] * 4]],
           "none": [[[0.0] * 4, [1.0] * 4], [[1.0] * 4, [0.0] * 4]]}
PAIRS = {"uneven": 5, "one_rank": 4, "none": 0}


def _trainer(rewards, first, **kw):
    """A trainer whose rollouts are fixed rows (those of prompts ``first`` on) with the given rewards, whose policy has moved off its reference and whose moments are not zero; and a
    list that receives the gradient of each update."""
    t = GRPOTrainer(AddTask(), layers=1, d_model=32, heads=2, G=G, prompts=len(rewards), device="cpu", dtype=torch.float32, dpo_beta=1.0, rllr=1e-3, **kw)
    t.ref.init_weights(77)
    t.policy.params.m.fill_(1e-3)
    t.policy.params.v.fill_(1e-4)
    g = torch.Generator().manual_seed(5)
    rows = torch.randint(0, t.task.vocab, (2 * PROMPTS * G, t.T), generator=g).tolist()[first * G:(first + len(rewards)) * G]

    def rollout(step):
        t.h_rew.copy_(torch.tensor(rewards).view(-1))
        return rows, dict(mean_reward=float(t.h_rew.mean()), rollout_tok_s=1.0, prefix_saved_per_prompt=0.0, rollout_ms=1.0)
    t._rollout = rollout
    grads, step = [], t.policy.adamw_step

    def keep(*a, **k):
        grads.append(t.policy.params.g.clone())
        return step(*a, **k)
    t.policy.adamw_step = keep
    return t, grads


def _worker(rank, port, case, out_dir):
    sys.path.insert(0, ROOT)
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE="2", LOCAL_RANK=str(rank))
    dist.init_process_group("gloo", rank=rank, world_size=2, timeout=datetime.timedelta(seconds=60))
    t, grads = _trainer(REWARDS[case][rank], rank * PROMPTS, dp_group=dist.group.WORLD, dp_rank=rank, dp=2)
    w = t.policy.params.w.clone()
    st = t.dpo_step(1)
    torch.save(dict(grads=grads, stats=st, w=t.policy.params.w.clone(), moved=not torch.equal(w, t.policy.params.w), step=t.policy.step), os.path.join(out_dir, "r%d.pt" % rank))
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("case", list(REWARDS))
def test_pairs_weigh_the_same_on_every_rank(case):
    one, grads = _trainer([p for r in REWARDS[case] for p in r], 0)
    st = one.dpo_step(1)
    assert st["pairs"] == PAIRS[case] and len(grads) == (1 if PAIRS[case] else 0)
    with tempfile.TemporaryDirectory() as d:
        mp.spawn(_worker, args=(_free_port(), case, d), nprocs=2, join=True)
        res = [torch.load(os.path.join(d, "r%d.pt" % r), weights_only=False) for r in range(2)]
    assert torch.equal(res[0]["w"], res[1]["w"])
    for r in res:
        assert r["stats"]["pairs"] == st["pairs"] and r["stats"]["pair_accuracy"] == pytest.approx(st["pair_accuracy"], abs=1e-6)
        # sums of some hundred fp32 terms in another order: some 2^-24 times 10 of the largest term
        assert r["stats"]["loss"] == pytest.approx(st["loss"], rel=1e-5) and r["stats"]["mean_reward"] == pytest.approx(st["mean_reward"], rel=1e-6)
        assert len(r["grads"]) == len(grads)
        for a, b in zip(r["grads"], grads):
            assert float((a - b).abs().max()) <= 1e-5 * float(b.abs().max())
        assert r["moved"] == bool(PAIRS[case]) and r["step"] == (1 if PAIRS[case] else 0)


def test_no_pair_no_update():
    """Moments of earlier updates move no weight where no pair counts."""
    t, grads = _trainer(REWARDS["none"][0], 0)
    w = t.policy.params.w.clone()
    st = t.dpo_step(1)
    assert torch.equal(w, t.policy.params.w) and t.policy.step == 0 and not grads
    assert st["pairs"] == 0 and st["loss"] == 0 and st["pair_accuracy"] == 0
