"""The 8-bit paged cache on the CPU: the plain evaluation against the definition in 64 bits, and what the operators refuse."""
import math

import pytest
import torch

from kharon_b200 import ops
from kharon_b200 import bench_infer
from kharon_b200.infer import InferEngine
from kharon_b200.models import GPT, Config
from kv8_exact import attend, quantise, quantising_oracle, rows_of


def make(seed, lens, H, hd, bs, extra=2):
    g = torch.Generator().manual_seed(seed)
    pages = [(n + bs - 1) // bs for n in lens]
    nb, max_lb = sum(pages) + extra, max(pages) + 1
    perm, btab, at = torch.randperm(nb, generator=g).int(), torch.full((len(lens), max_lb), -1, dtype=torch.int32), 0
    for i, n in enumerate(pages):
        btab[i, :n] = perm[at:at + n]
        at += n
    kv = torch.zeros(nb, H, ops.kv8_record_bytes(bs, hd), dtype=torch.uint8)
    pos = torch.cat([torch.arange(n) for n in lens]).int()
    slot = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)]).int()
    qkv = torch.randn(len(pos), 3 * H * hd, generator=g)
    return kv, btab, pos, slot, qkv


def awkward(hd):
    """Rows at the format's edges, bf16."""
    x = torch.randn(12, hd, generator=torch.Generator().manual_seed(4))
    x[0] = 0.0
    x[1] = -0.0
    x[2] *= 1e-30                       # below the smallest scale
    x[3] *= 1e30                        # above the largest
    x[4, 0], x[4, 1:] = 448.0 * 2.0 ** 5, 1.0        # exactly the largest number of a scale
    x[5, 0] = 450.0 * 2.0 ** 5          # one bf16 step above it
    x[6, 3] = math.inf
    x[7, 2] = -math.inf
    x[8, 1] = math.nan
    x[9] = math.nan
    x[10, 0], x[10, 1:] = 448.0, torch.linspace(-0.02, 0.02, hd - 1)     # codes below 2^-6
    x[11, 0], x[11, 1:] = 416.0, 17.0 * 2.0 ** torch.arange(hd - 1).remainder(5)      # halfway between two codes
    return x.bfloat16()


@pytest.mark.parametrize("hd,bs", [(16, 5), (32, 2), (64, 16), (128, 1)])
def test_quantised_rows_are_the_nearest_numbers_of_the_smallest_scale(hd, bs):
    x = awkward(hd)
    n = len(x)
    kv, btab, pos, slot, _ = make(1, [n], 2, hd, bs)
    kv.fill_(0xEE)
    qkv = torch.cat([torch.zeros(n, 2 * hd), x.float(), x.flip(0).float(), x.flip(0).float(), x.float()], 1)        # q | k of two heads | v of two heads
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, 2, hd, n)
    k, v = rows_of(kv, btab[0], bs, hd, n)
    want, e = quantise(x)
    for got in (k[:, 0], k[:, 1].flip(0), v[:, 0].flip(0), v[:, 1]):
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    fine = x.double().isfinite() & (x.double().abs() < 448 * 2.0 ** 63)
    err = (want - x.double()).abs()
    assert bool((err <= 2.0 ** -4 * x.double().abs() + 2.0 ** (e.double() - 10)[:, None])[fine].all())
    for dt in (torch.bfloat16, torch.float32):
        a, b = torch.zeros(n, 2 * hd, dtype=dt), torch.zeros(n, 2 * hd, dtype=dt)
        ops.read_kv8(kv, a, b, pos, slot, btab, bs, 2, hd, n)
        for got, w in ((a, k), (b, v)):
            got = got.double().view(n, 2, hd)
            assert torch.equal(got.isnan(), w.isnan()) and torch.equal(got.nan_to_num(0.0), w.nan_to_num(0.0))


@pytest.mark.parametrize("hd,H,bs", [(32, 3, 2), (64, 2, 16)])
def test_attention_of_cached_prompts_and_new_tokens(hd, H, bs):
    lens = [1, 7, 33]
    kv, btab, pos, slot, qkv = make(2, [n + 1 for n in lens], H, hd, bs)
    d, old = H * hd, torch.cat([torch.arange(n + 1) < n for n in lens])
    n = int(old.sum())
    sel = lambda t, m: t[m].contiguous()
    ops.append_kv8(sel(qkv, old), kv, sel(pos, old), sel(slot, old), btab, bs, H, hd, n)
    runs, at = [], 0
    for k in lens:
        runs.append((at, k))
        at += k
    out = torch.zeros(n, d)
    ops.paged_prefill8(sel(qkv, old), kv, out, sel(pos, old), sel(slot, old), btab, bs, H, hd, runs, 64)
    new = torch.full((3, d), 7.0)
    ops.paged_attn8(sel(qkv, ~old), kv, new[:, :d], sel(pos, ~old), sel(slot, ~old), btab, bs, H, hd, 3, 64, append=True)
    for got, m in ((out, old), (new, ~old)):
        for i, t in enumerate(torch.nonzero(m).flatten().tolist()):
            k, v = rows_of(kv, btab[int(slot[t])], bs, hd, int(pos[t]) + 1)
            want, tol = attend(qkv[t, :d].double().view(H, hd), k, v)
            assert bool(((got[i].double().view(H, hd) - want).abs() <= tol).all())
    pool = torch.stack([kv, kv.flip(0)]).contiguous()
    before = pool.clone()
    ops.copy_blocks8(pool, torch.tensor([0, 2, 1, 3], dtype=torch.int32), 2)
    assert torch.equal(pool[:, 2], before[:, 0]) and torch.equal(pool[:, 3], before[:, 1]) and torch.equal(pool[:, 4:], before[:, 4:])


def test_refused_arguments():
    H, hd, bs, n = 2, 32, 4, 6
    kv, btab, pos, slot, qkv = make(3, [n], H, hd, bs)
    out = torch.zeros(n, H * hd)
    app = lambda **k: ops.append_kv8(*[{**dict(qkv=qkv, kv=kv, pos=pos, slot=slot, btab=btab, bs=bs, H=H, hd=hd, ntok=n), **k}[x]
                                       for x in ("qkv", "kv", "pos", "slot", "btab", "bs", "H", "hd", "ntok")])
    for bad in (dict(hd=48), dict(hd=64), dict(bs=0), dict(bs=8), dict(H=3), dict(kv=kv.short()), dict(kv=kv[:, :, :-32]), dict(kv=kv.transpose(0, 1)),
                dict(pos=pos.long()), dict(slot=slot[:3]), dict(pos=torch.stack([pos, pos], 1)[:, 0]), dict(btab=btab.long()), dict(btab=btab[0]),
                dict(btab=torch.zeros(3, 2, dtype=torch.int32).t()), dict(ntok=n + 1), dict(ntok=-1)):
        with pytest.raises(ValueError):
            app(**bad)
    with pytest.raises(ValueError):
        ops.read_kv8(kv, out.half(), out.half(), pos, slot, btab, bs, H, hd, n)
    with pytest.raises(ValueError):
        ops.read_kv8(kv, out, out[:2], pos, slot, btab, bs, H, hd, n)
    with pytest.raises(ValueError):
        ops.read_kv8(kv, out[:, :32], out[:, :32], pos, slot, btab, bs, H, hd, n)
    for runs in ([(0, n + 1)], [(-1, 2)], [(3, 0)]):
        with pytest.raises(ValueError):
            ops.paged_prefill8(qkv, kv, out, pos, slot, btab, bs, H, hd, runs, 64)
    kv16, btab16, pos16, slot16, qkv16 = make(3, [n], H, 16, bs)
    with pytest.raises(ValueError):
        ops.paged_prefill8(qkv16, kv16, out, pos16, slot16, btab16, bs, H, 16, [(0, n)], 64)
    with pytest.raises(ValueError):
        ops.copy_blocks8(kv, pos, 1)
    with pytest.raises(ValueError):
        ops.copy_blocks8(kv[None], pos[:3], 2)
    # positions, sequences and blocks out of range
    for p, s, t in ((torch.tensor([8 * bs]), 0, None), (torch.tensor([-1]), 0, None), (torch.tensor([0]), 5, None), (torch.tensor([0]), 0, 99)):
        tab = btab.clone()
        if t is not None:
            tab[0, 0] = t
        with pytest.raises(IndexError):
            ops.append_kv8(qkv, kv, p.int(), torch.tensor([s], dtype=torch.int32), tab, bs, H, hd, 1)
        with pytest.raises(IndexError):
            ops.paged_attn8(qkv, kv, out, p.int(), torch.tensor([s], dtype=torch.int32), tab, bs, H, hd, 1, 64)
    before = kv.clone()
    app(ntok=0)
    ops.paged_attn8(qkv, kv, out, pos, slot, btab, bs, H, hd, 0, 64, append=True)
    ops.paged_prefill8(qkv, kv, out, pos, slot, btab, bs, H, hd, [], 64)
    assert torch.equal(kv, before) and float(out.abs().max()) == 0.0


CFG = Config(2, 64, 4, 97, 48, 1)
PROMPTS = [[5, 17, 3], [9, 1, 44, 23, 8, 61, 2], [70], [11, 12, 13, 14, 15, 16, 17, 18, 19, 20, 21]]
NEW = [12, 7, 20, 9]


@pytest.fixture(scope="module")
def pair():
    m = GPT(CFG, "cpu", torch.float32)
    m.init_weights(1234)
    m.params.w.mul_(8.0)
    m.params.p["lnf_w"].fill_(1.0)
    for l in range(CFG.n_layer):
        m.params.p["l%d.ln1_w" % l].fill_(1.0)
        m.params.p["l%d.ln2_w" % l].fill_(1.0)
    return m, quantising_oracle(CFG, m)


def greedy(o, prompt, n_new):
    toks = list(prompt)
    with torch.no_grad():
        for _ in range(n_new):
            toks.append(int(o(torch.tensor([toks]))[0][0, -1].argmax()))
    return toks


@pytest.mark.parametrize("bs,active", [(4, 2), (64, 4), (8, 4), (3, 1)])
def test_engine_over_the_8bit_cache_is_token_exact(pair, bs, active):
    """Greedy decoding with the quantised keys and values, whatever the block size and however prompts and decoding sequences share steps."""
    m, o = pair
    eng = InferEngine(m, block_size=bs, max_seqs=4, kv8=True)
    assert eng.kc is None and eng.kv8.dtype == torch.uint8
    outs, st, _ = eng.generate(PROMPTS, NEW, max_active=active)
    for p, n, got in zip(PROMPTS, NEW, outs):
        assert got == greedy(o, p, n)
    assert st["tokens_decoded"] == sum(NEW)


def test_shared_prefix_over_the_8bit_cache(pair):
    m, o = pair
    eng = InferEngine(m, block_size=4, max_seqs=9, kv8=True)
    outs, st, _ = eng.generate_group(PROMPTS[3][:10], 8, 9)
    assert all(x == greedy(o, PROMPTS[3][:10], 9) for x in outs) and st["prefix_blocks_saved"] == 7 * (10 // 4)
    # per layer, head and block of 4 positions: 2 * 4 * 16 codes and 8 exponents, padded to 160 bytes; fp32 keeps 2 * 16 * 4 bytes a position
    assert eng.kv_bytes_per_position() == 2 * 4 * 160 / 4 and InferEngine(m, block_size=4, max_seqs=9).kv_bytes_per_position() == 2 * 4 * 128


def test_engine_refuses_head_widths_without_an_8bit_cache():
    with pytest.raises(ValueError):
        InferEngine(GPT(Config(1, 48, 2, 50, 16, 1), "cpu", torch.float32), block_size=4, max_seqs=2, kv8=True)


def test_bench_command_with_the_8bit_cache():
    r = bench_infer.run(["--layers", "1", "--d", "64", "--heads", "4", "--vocab", "50", "--seq", "32", "--prompt", "6", "--new", "4", "--block", "4", "--bf16", "0",
                         "--G", "1,2", "--device", "cpu", "--reps", "1", "--kv8"])
    assert len(r["decode"]) == 2 and r["decode"][0]["kv_paged_mb"] > 0
