"""Critic-free GRPO: supervised warm start, group rollouts through the paged-KV engine with
prefix sharing, group-relative advantages, KL penalty (k3 estimator gradient) to a frozen
snapshot of the SFT policy, one AdamW step per rollout batch (on-policy, ratio = 1).

Behaviour follows the reference's src/grpo_train.c:67-191 and src/core/grpo.c:7-20:

    adv      = (r - mean_group) / (std_group_population + 1e-4)
    coef[t]  = mask[t] * (adv[row] - beta * (1 - p_ref / max(p_cur, 1e-8))) / N_completion_tokens
    dlogits  = coef * (softmax - onehot)          (fused into the cross-entropy kernel)

with mask = the positions whose logits predict completion tokens.  Additions: a second task
(reverse an 8-digit string, reward 1 / 0), rollouts of all prompts of a step in one engine batch,
and data parallelism over prompts (gradients averaged over the DP group, every rank steps the
same replicated policy) -- the reference is single-GPU only.

Also beyond the reference: several updates on one rollout batch (``inner``) with the clipped policy loss, a bound on the gradient's norm (``max_norm``), and
preference training on the same rollouts (``dpo_step``): the best sample of a prompt against the worst, the second best against the second worst and so on.
"""
from __future__ import annotations

import ctypes as C

import torch
import torch.distributed as dist

from .. import _native, ops
from ..infer import InferEngine
from ..models import GPT, Config
from ..utils.rng import Rng


def advantages(rewards: torch.Tensor, n_groups: int, group: int, eps: float = 1e-4) -> torch.Tensor:
    r = rewards.detach().to("cpu", torch.float32).contiguous()
    out = torch.empty_like(r)
    _native.rt().kh_grpo_advantages(r.data_ptr(), n_groups, group, eps, out.data_ptr())
    return out


def coefficients(adv, p_cur, p_ref, rows, T, t0, t1, beta) -> torch.Tensor:
    a = adv.detach().to("cpu", torch.float32).contiguous()
    pc = p_cur.detach().to("cpu", torch.float32).contiguous()
    pr = p_ref.detach().to("cpu", torch.float32).contiguous()
    out = torch.empty(rows * T, dtype=torch.float32)
    _native.rt().kh_grpo_coef(a.data_ptr(), pc.data_ptr(), pr.data_ptr(), rows, T, t0, t1, beta, out.data_ptr())
    return out


class AddTask:
    """Single-digit addition ``a+b=`` -> one digit (the reference's task, grpo_train.c:23-44):
    reward 0.1 for any digit plus 1.0 for the exact answer."""
    plen, nnew, vocab = 4, 1, 256

    def sample(self, rng: Rng):
        while True:
            a, b = rng.u32() % 10, rng.u32() % 10
            if a + b <= 9:
                return [48 + a, ord("+"), 48 + b, ord("=")], [48 + a + b]

    def reward(self, completion, answer):
        r = 0.1 if 48 <= completion[0] <= 57 else 0.0
        return r + (1.0 if completion[0] == answer[0] else 0.0)

    def eval_set(self):
        return [([48 + a, ord("+"), 48 + b, ord("=")], [48 + a + b]) for a in range(10) for b in range(10) if a + b <= 9]


class ReverseTask:
    """Reverse a random 8-digit string: prompt = 8 digits + separator, completion = the digits
    reversed + EOS; reward 1 on an exact match, else 0."""
    n, sep, eos, vocab = 8, ord("|"), ord("\n"), 256
    plen, nnew = 9, 9

    def sample(self, rng: Rng):
        digs = [48 + rng.u32() % 10 for _ in range(self.n)]
        return digs + [self.sep], digs[::-1] + [self.eos]

    def reward(self, completion, answer):
        return 1.0 if list(completion) == list(answer) else 0.0

    def eval_set(self):
        r = Rng(999)
        return [self.sample(r) for _ in range(64)]


class GRPOTrainer:
    def __init__(self, task, layers=4, d_model=256, heads=8, seq=None, G=8, prompts=16, lr=1e-3, rllr=1e-4, temp=1.0,
                 beta=0.02, device="cuda", dtype=torch.bfloat16, dp_group=None, dp_rank=0, dp=1, seed=1337,
                 task_seed=20260530, inner=1, clip_eps=0.0, max_norm=0.0, dpo_beta=0.1):
        """``inner`` updates on each rollout batch, with the ratio to the policy that sampled it held within 1 -+ ``clip_eps`` (0 with one update: the
        reference's step); ``max_norm`` > 0 bounds the gradient's norm in every update, the supervised ones too; ``dpo_beta``: the preference loss's."""
        if inner < 1 or not 0 <= clip_eps <= 1 or not max_norm >= 0 or (inner > 1 and clip_eps == 0):
            raise ValueError("inner=%s, clip_eps=%s (0 to 1, above 0 for several updates), max_norm=%s" % (inner, clip_eps, max_norm))
        self.inner, self.clip_eps, self.max_norm, self.dpo_beta = inner, clip_eps, max_norm, dpo_beta
        self.task, self.G, self.NP = task, G, prompts
        self.T = task.plen + task.nnew
        self.B = prompts * G
        self.lr, self.rllr, self.temp, self.beta = lr, rllr, temp, beta
        self.dp_group, self.dp, self.dp_rank = dp_group, dp, dp_rank
        self.device = torch.device(device)
        # the model sequence length is the trained window; ``seq`` only sizes the position table
        self.cfg = Config(layers, d_model, heads, task.vocab, self.T if seq is None else max(seq, self.T), self.B)
        train_cfg = Config(layers, d_model, heads, task.vocab, self.T, self.B)
        self.train_cfg = train_cfg
        self.policy = self._make(seed, dtype)
        self.ref = self._make(seed, dtype)
        self.engine = InferEngine(self.policy, block_size=2, n_blocks=self.B * self.T + 64 + prompts * 8,
                                  max_tokens=self.B * self.T + 64, max_seqs=self.B + prompts + 1)
        self.rng = Rng(task_seed + dp_rank)
        pin = self.device.type == "cuda"
        self.h_idx = torch.zeros(self.B * self.T, dtype=torch.int32, pin_memory=pin)
        self.h_tgt = torch.zeros(self.B * self.T, dtype=torch.int32, pin_memory=pin)
        self.d_coef = torch.zeros(self.B * self.T, dtype=torch.float32, device=self.device)
        self.h_rew = torch.zeros(self.B, dtype=torch.float32, pin_memory=pin)
        self.d_rew = torch.zeros(self.B, dtype=torch.float32, device=self.device)
        self.d_adv = torch.zeros(self.B, dtype=torch.float32, device=self.device)
        self.d_pcur = torch.zeros(self.B * self.T, dtype=torch.float32, device=self.device)
        R = self.B * self.T
        vec = lambda n=R: torch.zeros(n, dtype=torch.float32, device=self.device)  # noqa: E731
        self.d_old, self.d_ref, self.d_kl, self.d_clip, self.d_loss, self.d_sum = vec(), vec(), vec(), vec(), vec(), vec(4)
        self.grad_list = ops.TensorList([self.policy.params.g]) if max_norm > 0 else None
        self.norm_out = vec(2)
        if max_norm > 0:
            self.policy.left_out = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.pairs = None
        self.stats = {}

    def _make(self, seed, dtype):
        # positions: the engine needs wpe rows up to cfg.seq, training uses rows [0, T)
        m = GPT(Config(self.train_cfg.n_layer, self.train_cfg.d_model, self.train_cfg.n_head, self.train_cfg.vocab,
                       self.T, self.B), self.device, dtype)
        m.init_weights(seed)
        return m

    # ------------------------------------------------------------------ helpers
    def _fill_rows(self, rows):
        """Token rows -> the pinned input / target staging buffers (target = next token, 0 after the last)."""
        t = torch.tensor(rows, dtype=torch.int32)                     # [B, T]
        self.h_idx.view(self.B, self.T).copy_(t)
        tg = self.h_tgt.view(self.B, self.T)
        tg[:, :-1].copy_(t[:, 1:])
        tg[:, -1].zero_()

    def _mask_targets(self):
        """Leaves the targets of the completions alone (the losses on log probabilities pass over negative ones)."""
        tg = self.h_tgt.view(self.B, self.T)
        tg[:, :self.task.plen - 1] = -1
        tg[:, -1] = -1

    def _update(self, lr):
        """Gradient exchange, bound and AdamW step."""
        self._sync_grads()
        factor = None
        if self.grad_list is not None:
            ops.grad_norm(self.grad_list, self.norm_out, max_norm=self.max_norm, left_out=self.policy.left_out)
            factor = self.norm_out[1:]
        self.policy.adamw_step(lr, 0.9, 0.95, 1e-8, 0.0, factor=factor)

    def _rollout(self, step):
        """Samples G completions of each of this step's prompts: (rows of tokens in prompt order, rewards in ``h_rew``, statistics)."""
        task, G, T = self.task, self.G, self.T
        self.engine.set_sampling(self.temp, 0x1234 * step + 1 + 7919 * self.dp_rank)
        probs = [task.sample(self.rng) for _ in range(self.NP)]
        outs, st, ms = self.engine.generate_groups([p for p, _ in probs], G, task.nnew)
        rows, rew = [], self.h_rew
        for pi, (p, ans) in enumerate(probs):
            for g in range(G):
                seq = (outs[pi][g] + [0] * T)[:T]
                rows.append(seq)
                rew[pi * G + g] = task.reward(seq[task.plen:task.plen + task.nnew], ans)
        return rows, dict(mean_reward=float(rew.mean()), rollout_tok_s=st["tokens_decoded"] * 1000.0 / max(ms, 1e-9),
                          prefix_saved_per_prompt=st["prefix_blocks_saved"] / self.NP, rollout_ms=ms)

    def _share_stats(self, names):
        """Means over the data-parallel ranks of the named statistics."""
        if self.dp > 1:
            t = torch.tensor([self.stats[n] for n in names], device=self.device)
            dist.all_reduce(t, group=self.dp_group)
            for n, v in zip(names, (t / self.dp).tolist()):
                self.stats[n] = v
        return self.stats

    heartbeat = None        # utils.watchdog.Heartbeat of the job, when the entry point set one up

    def _sum_ranks(self, t, what):
        """Sum of ``t`` over the data-parallel ranks, in place; a dead rank is an exception where there is a heartbeat."""
        if self.dp > 1:
            if self.heartbeat is not None:
                from ..utils.watchdog import guarded
                self.heartbeat.check()
                guarded(dist.all_reduce(t, group=self.dp_group, async_op=True), self.heartbeat,
                        timeout_s=120.0, group=self.dp_group, what="%s all-reduce" % what)
            else:
                dist.all_reduce(t, group=self.dp_group)
        return t

    def _sync_grads(self):
        if self.dp > 1:
            self._sum_ranks(self.policy.params.g, "gradient").div_(self.dp)

    def sft_step(self):
        rows = []
        for _ in range(self.B):
            p, a = self.task.sample(self.rng)
            rows.append(p + a)
        self._fill_rows(rows)
        m = self.policy
        m.set_input(self.h_idx, self.h_tgt)
        m.forward(compute_loss=False)
        m.backward(loss_scale=1.0)
        self._update(self.lr)
        return m.loss()

    def snapshot_reference(self):
        """Freeze the current policy as the KL reference (grpo_train.c:126-127)."""
        self.ref.params.w.copy_(self.policy.params.w)
        self.ref.sync_bf16()

    def eval_accuracy(self):
        self.engine.set_sampling(0.0, 1)
        es = self.task.eval_set()
        outs, _, _ = self.engine.generate([p for p, _ in es], self.task.nnew, max_active=min(len(es), self.B))
        ok = sum(1 for (p, a), o in zip(es, outs) if o[len(p):len(p) + len(a)] == list(a))
        return ok / len(es)

    def grpo_step(self, step: int):
        if self.clip_eps > 0:
            return self._clipped_step(step)
        task, G, NP, T, B = self.task, self.G, self.NP, self.T, self.B
        rows, stats = self._rollout(step)
        # rewards go up (B floats); advantages, p(action) of both models and the coefficients stay on the device
        self.d_rew.copy_(self.h_rew, non_blocking=True)
        ops.grpo_advantages(self.d_rew, NP, G, 1e-4, self.d_adv)
        self._fill_rows(rows)
        m, ref = self.policy, self.ref
        m.set_input(self.h_idx, self.h_tgt)
        m.forward(compute_loss=False)
        self.d_pcur.copy_(m.gather_prob())
        ref.set_input(self.h_idx, self.h_tgt)
        ref.forward(compute_loss=False)
        p_ref = ref.gather_prob()
        ops.grpo_coef(self.d_adv, self.d_pcur, p_ref, B, T, task.plen - 1, T - 2, self.beta, self.d_coef)
        m.backward(coef=self.d_coef)
        self._update(self.rllr)
        self.stats = stats
        return self._share_stats(["mean_reward"])

    def _clipped_step(self, step: int):
        """``inner`` updates of the clipped policy loss on one rollout batch.  The first is on-policy (its log probabilities are the old ones of the others)."""
        m, n = self.policy, self.B * self.task.nnew
        rows, stats = self._rollout(step)
        self.d_rew.copy_(self.h_rew, non_blocking=True)
        ops.grpo_advantages(self.d_rew, self.NP, self.G, 1e-4, self.d_adv)
        self._fill_rows(rows)
        self._mask_targets()
        self.ref.set_input(self.h_idx, self.h_tgt)
        self.ref.forward(compute_loss=False)
        self.ref.gather_logp(self.d_ref)
        m.set_input(self.h_idx, self.h_tgt)
        for i in range(self.inner):
            m.forward(compute_loss=False)
            m.backward(head_loss=lambda logits, V, tgt: ops.policy_loss(
                logits, V, tgt, self.d_adv, old_logp=self.d_old if i else None, ref_logp=self.d_ref, clip_lo=self.clip_eps, clip_hi=self.clip_eps,
                beta=self.beta, uniform=1.0 / n, rowloss=self.d_loss, logp=None if i else self.d_old, kl=self.d_kl, clipped=self.d_clip, dlogits=logits))
            self._update(self.rllr)
        for k, v in enumerate((self.d_loss, self.d_kl, self.d_clip)):
            ops.sum_f32(v, self.d_sum[k:k + 1], scale=1.0 if k == 0 else 1.0 / n)
        loss, kl, clipped = self.d_sum[:3].tolist()
        self.stats = dict(stats, loss=loss, kl=kl, clipped=clipped)
        return self._share_stats(["mean_reward", "loss", "kl", "clipped"])

    def dpo_step(self, step: int):
        """One update of the preference loss on a rollout batch: of each prompt's G samples (an even number), ordered by reward, the first against the last and so on; pairs of
        equal reward do not count.  The loss is the mean over the pairs of all data-parallel ranks; where none counts there is no update."""
        if self.G % 2:
            raise ValueError("dpo_step: an even number of samples of each prompt is needed, not %d" % self.G)
        m, B, T, G, P = self.policy, self.B, self.T, self.G, self.B // 2
        rows, stats = self._rollout(step)
        order = torch.sort(self.h_rew.view(self.NP, G), dim=1, descending=True, stable=True).indices
        order = torch.stack([order[:, :G // 2], order.flip(1)[:, :G // 2]], 2) + G * torch.arange(self.NP)[:, None, None]
        order = order.reshape(-1).tolist()                                       # chosen, rejected, chosen, rejected, ...
        rew = self.h_rew[order]
        counts = (rew[0::2] > rew[1::2]).float()
        n = float(counts.sum())
        if self.dp > 1:
            n = float(self._sum_ranks(torch.tensor([n], device=self.device), "number of pairs"))
        self.stats = dict(stats, loss=0.0, pairs=n, pair_accuracy=0.0)
        if n == 0:
            return self._share_stats(["mean_reward"])
        self._fill_rows([rows[i] for i in order])
        self._mask_targets()
        if self.pairs is None:
            self.pairs = dict(starts=torch.arange(0, B * T + 1, T, dtype=torch.int32, device=self.device), work=ops.preference_work(B * T, P, self.device),
                              weight=torch.zeros(P, device=self.device), loss=torch.zeros(P, device=self.device), margin=torch.zeros(P, device=self.device))
        q = self.pairs
        q["weight"].copy_(counts * self.dp / n)                                  # (the ranks' gradients are averaged)
        self.ref.set_input(self.h_idx, self.h_tgt)
        self.ref.forward(compute_loss=False)
        self.ref.gather_logp(self.d_ref)
        m.set_input(self.h_idx, self.h_tgt)
        m.forward(compute_loss=False)
        m.backward(head_loss=lambda logits, V, tgt: ops.preference_loss(
            logits, V, tgt, q["starts"], ref_logp=self.d_ref, beta=self.dpo_beta, weight=q["weight"], loss=q["loss"], margin=q["margin"], dlogits=logits,
            work=q["work"]))
        self._update(self.rllr)
        ordered = float((q["margin"].cpu()[counts > 0] > 0).sum())
        self.stats.update(loss=float(q["loss"].sum()), pair_accuracy=ordered * self.dp / n)
        return self._share_stats(["mean_reward", "loss", "pair_accuracy"])
