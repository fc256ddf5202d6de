"""A step that is left out because its gradient's norm is not finite leaves no trace: the steps behind it are those of a run that never had it, on every mesh and behind a checkpoint."""
import datetime
import math
import os
import sys
import tempfile

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from kharon_b200 import ops
from kharon_b200.engine import TrainEngine
from kharon_b200.rl import AddTask, GRPOTrainer
from test_parallel_cpu import KW, ROOT, _batches, _free_port

TOP = 0.05


def poison(e, where=5):
    """The next step of the engine finds an infinite gradient."""
    sync = e._sync_sp_grads

    def once():
        sync()
        e.model.params.g[where] = math.inf
        e._sync_sp_grads = sync
    e._sync_sp_grads = once


def run(e, data, bad, where=5):
    for s, d in enumerate(data):
        if s in bad:
            poison(e, where)
        e.train_step(*d)


@pytest.mark.parametrize("bad", [(0,), (1, 2), (0, 1, 3)])
def test_engine(bad):
    a, b = TrainEngine(max_norm=TOP, **KW), TrainEngine(max_norm=TOP, **KW)
    data = _batches(0, 5, a.tokens_per_step, KW["vocab"])
    run(a, data, bad)
    run(b, [d for s, d in enumerate(data) if s not in bad], ())
    for x, y in ((a.model.params.w, b.model.params.w), (a.model.params.m, b.model.params.m), (a.model.params.v, b.model.params.v)):
        assert torch.equal(x, y)
    assert a.model.step == 5 and int(a.model.left_out) == len(bad) and int(b.model.left_out) == 0


def test_checkpoint():
    """The step of a checkpoint is the number of updates: the run goes on from it as without the steps that were left out."""
    a, b = TrainEngine(max_norm=TOP, **KW), TrainEngine(max_norm=TOP, **KW)
    data = _batches(0, 4, a.tokens_per_step, KW["vocab"])
    run(a, data[:3], (0,))
    with tempfile.TemporaryDirectory() as d:
        a.save(os.path.join(d, "x"))
        run(b, data[2:3], (0,))                                # (a count of its own, which the load forgets)
        b.load(os.path.join(d, "x"))
    assert b.model.step == 2 and int(b.model.left_out) == 0
    run(a, data[3:], ())
    run(b, data[3:], ())
    assert torch.equal(a.model.params.w, b.model.params.w) and torch.equal(a.model.params.m, b.model.params.m)


def _worker(rank, world, port, tp, pp, dp, out_dir):
    sys.path.insert(0, ROOT)
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world), LOCAL_RANK=str(rank))
    dist.init_process_group("gloo", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=60))
    from kharon_b200.parallel.mesh import Mesh
    out = []
    mesh = Mesh(tp, pp, dp, timeout_s=60)
    for bad in ((0,), ()):
        e = TrainEngine(mesh=mesh, max_norm=TOP, untied_head=True, **KW)
        data = _batches(mesh.c.dp_rank, 3, e.tokens_per_step, KW["vocab"])
        run(e, data if bad else data[1:], bad if rank == 0 else ())          # one rank's gradient is infinite, all leave the step out
        e.gather_master()
        out.append((e.model.params.w.clone(), int(e.model.left_out), e.model.step))
    torch.save(out, os.path.join(out_dir, "r%d.pt" % rank))
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("tp,pp,dp", [(2, 1, 1), (1, 2, 1), (1, 1, 2)])
def test_meshes(tp, pp, dp):
    with tempfile.TemporaryDirectory() as d:
        mp.spawn(_worker, args=(2, _free_port(), tp, pp, dp, d), nprocs=2, join=True)
        for r in range(2):
            (w, left, step), (w2, left2, step2) = torch.load(os.path.join(d, "r%d.pt" % r), weights_only=False)
            assert torch.equal(w, w2) and (left, step, left2, step2) == (1, 3, 0, 2)


def test_trainer():
    mk = lambda: GRPOTrainer(AddTask(), layers=1, d_model=32, heads=2, G=4, prompts=4, device="cpu", dtype=torch.float32, max_norm=0.1)  # noqa: E731
    a, b = mk(), mk()
    sync = a._sync_grads

    def bad():
        sync()
        a.policy.params.g[3] = math.nan
        a._sync_grads = sync
    a._sync_grads = bad
    state = a.rng.state
    a.sft_step()
    a.rng.state = state
    for t in (a, b):
        t.sft_step()
        t.sft_step()
    assert torch.equal(a.policy.params.w, b.policy.params.w) and int(a.policy.left_out) == 1 and a.policy.step == 3


@pytest.mark.parametrize("step,left", [(2, 1), (7, 0), (1000, 37), (5, 4)])
def test_adamw_counts_the_steps_that_were_taken(step, left):
    mk = lambda: [torch.randn(50, generator=torch.Generator().manual_seed(i)).abs() for i in range(4)]  # noqa: E731
    kw = dict(lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8, wd=0.1)
    x, y = mk(), mk()
    f = torch.tensor([0.25])
    ops.adamw(*x, None, step=step, factor=f, left_out=torch.tensor([left], dtype=torch.int32), **kw)
    ops.adamw(*y, None, step=step - left, factor=f, **kw)
    assert all(torch.equal(a, b) for a, b in zip(x, y))


def test_counts_and_refusals():
    t, out, n, sq = torch.ones(4), torch.zeros(2), torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.float64)
    for v, want in ((1.0, 0), (math.inf, 1), (2.0, 1), (math.nan, 2), (3e38, 2)):
        t[1] = v
        ops.grad_norm(ops.TensorList([t]), out, max_norm=1.0, sumsq=sq, left_out=n)
        assert int(n) == want
    sq.fill_(math.inf)
    ops.clip_factor(sq, out, 1.0, left_out=n)
    assert int(n) == 3
    for bad in (torch.zeros(1), torch.zeros(2, dtype=torch.int32)):
        with pytest.raises(ValueError):
            ops.grad_norm(ops.TensorList([t]), out, left_out=bad)
        with pytest.raises(ValueError):
            ops.clip_factor(sq, out, 1.0, left_out=bad)
        with pytest.raises(ValueError):
            ops.adamw(t, t.clone(), t.clone(), t.clone(), None, lr=1, beta1=0, beta2=0, eps=1, wd=0, step=1, factor=torch.ones(1), left_out=bad)
    with pytest.raises(ValueError):
        ops.grad_norm(ops.TensorList([t]), sumsq=sq, left_out=n)
    with pytest.raises(ValueError):
        ops.adamw(t, t.clone(), t.clone(), t.clone(), None, lr=1, beta1=0, beta2=0, eps=1, wd=0, step=1, left_out=n)
