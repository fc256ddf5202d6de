"""The 8-bit paged cache's kernels against the definition in 64 bits, at the sizes, masks and tables where they can go wrong."""
import math

import pytest
import torch

from kharon_b200 import ops
from kharon_b200.infer import InferEngine
from kharon_b200.models import GPT, Config
from kv8_exact import attend, grid, quantise, rows_of
from test_kv8_cpu import awkward

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(seed, lens, H, hd, bs, pad=0, extra=3, blocks=None):
    """An empty cache with tables for sequences of these lengths (-1 behind their pages), and bf16 rows q | k | v of all their tokens."""
    g = torch.Generator().manual_seed(seed)
    pages = [(n + bs - 1) // bs for n in lens]
    nb, max_lb = blocks or sum(pages) + extra, max(pages) + 1
    perm, btab, at = torch.randperm(nb, generator=g).int(), torch.full((len(lens), max_lb), -1, dtype=torch.int32), 0
    for i, n in enumerate(pages):
        btab[i, :n] = perm[at:at + n]
        at += n
    kv = torch.zeros(nb, H, ops.kv8_record_bytes(bs, hd), dtype=torch.uint8, device=DEV)
    pos = torch.cat([torch.arange(n) for n in lens]).int()
    slot = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)]).int()
    qkv = torch.randn(len(pos), 3 * H * hd + pad, generator=g)
    qkv[:, H * hd:2 * H * hd] *= torch.exp(torch.randn(len(pos), 1, generator=g) * 0.3)
    qkv[:, 2 * H * hd:] *= torch.exp(torch.randn(len(pos), 1, generator=g))
    return kv, btab.to(DEV), pos.to(DEV), slot.to(DEV), qkv.bfloat16().to(DEV)


def check_rows(out, q, kv, btab, bs, H, hd, pos, slot, rows, p_half_step=0.0):
    """Rows of `out` against 64 bits, from the bytes of the cache."""
    kv, btab, pos, slot, q, out = kv.cpu(), btab.cpu(), pos.cpu(), slot.cpu(), q.double().cpu(), out.double().cpu()
    cache = {}
    for t in rows:
        s, n = int(slot[t]), int(pos[t]) + 1
        if s not in cache or cache[s][0].shape[0] < n:
            cache[s] = rows_of(kv, btab[s], bs, hd, max(n, max(int(pos[u]) + 1 for u in rows if int(slot[u]) == s)))
        want, tol = attend(q[t, :H * hd].view(H, hd), cache[s][0][:n], cache[s][1][:n], p_half_step)
        err = (out[t, :H * hd].view(H, hd) - want).abs()
        assert torch.equal(err.isnan(), want.isnan() & err.isnan()) and torch.equal(want.isnan(), out[t, :H * hd].view(H, hd).isnan()), (t, n)
        assert bool((err.nan_to_num(0.0) <= tol.nan_to_num(0.0)).all()), (t, n, float((err / tol).max()))


@pytest.mark.parametrize("hd,H,bs", [(16, 3, 5), (32, 4, 2), (64, 2, 16), (128, 1, 24), (64, 5, 1), (128, 16, 64)])
def test_append_and_read_back_have_the_bits_of_the_definition(hd, H, bs):
    lens = [1, 12, 37]
    kv, btab, pos, slot, qkv = make(hd + bs, lens, H, hd, bs, pad=8)
    n, d = len(pos), H * hd
    qkv[1:13, d:d + hd] = awkward(hd).to(DEV)
    qkv[1:13, 3 * d - hd:3 * d] = awkward(hd).flip(0).to(DEV)
    kv.fill_(0xA5)
    ref_kv = kv.cpu()
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    ops.append_kv8(qkv.cpu().float(), ref_kv, pos.cpu(), slot.cpu(), btab.cpu(), bs, H, hd, n)
    same = kv.cpu() == ref_kv
    nan = (kv.cpu() & 0x7F == 0x7F) & (ref_kv & 0x7F == 0x7F)                    # either sign of NaN
    assert bool((same | nan).all())                                              # places of no listed token included
    for s in range(3):
        k, v = rows_of(kv.cpu(), btab[s].cpu(), bs, hd, lens[s])
        m = slot.cpu() == s
        for got, col in ((k, d), (v, 2 * d)):
            for h in (0, H - 1):
                want, _ = quantise(qkv.cpu()[m, col + h * hd:col + (h + 1) * hd])
                assert torch.equal(got[:, h].nan_to_num(7e77), want.nan_to_num(7e77))
    for dt in (torch.bfloat16, torch.float32):
        a, b = torch.full((n + 1, d + 8), 3.0, dtype=dt, device=DEV), torch.full((n + 1, d + 8), 3.0, dtype=dt, device=DEV)
        ops.read_kv8(kv, a, b, pos, slot, btab, bs, H, hd, n)
        for s in range(3):
            for got, want in zip((a, b), rows_of(kv.cpu(), btab[s].cpu(), bs, hd, lens[s])):
                x = got[:n][slot == s][:, :d].double().cpu().view(-1, H, hd)
                assert torch.equal(x.nan_to_num(7e77), want.nan_to_num(7e77))
        assert float((a[n] - 3).abs().max()) == 0 and float((b[:, d:] - 3).abs().max()) == 0
    assert ops.error_word() == 0


@pytest.mark.parametrize("hd,H,bs,lens", [(16, 4, 2, [1, 2, 40]), (32, 8, 2, [18]), (32, 4, 16, [1, 17, 129, 700]), (64, 2, 16, [3, 64, 1000]), (64, 16, 5, [31, 33, 1, 90]),
                                          (128, 2, 24, [700, 5]), (128, 4, 64, [1, 63, 64, 65]), (64, 4, 16, [5000]), (128, 16, 16, [40] * 160), (32, 3, 1, [300, 2])])
@pytest.mark.parametrize("append", [True, False])
def test_single_token_attention(hd, H, bs, lens, append):
    kv, btab, pos, slot, qkv = make(hd + len(lens), lens, H, hd, bs, pad=16)
    d, n = H * hd, len(pos)
    last = torch.tensor([sum(lens[:i + 1]) - 1 for i in range(len(lens))], device=DEV)
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    whole = kv.clone()
    ln = len(lens)
    if append:                                     # the last position of every sequence is missing from the cache
        blk, at = btab[slot[last].long(), pos[last].long() // bs].long(), pos[last].long() % bs
        nb = kv.shape[0]
        kv[:, :, :bs * hd].view(nb, H, bs, hd)[blk, :, at] = 0x7F
        kv[:, :, bs * hd:2 * bs * hd].view(nb, H, bs, hd)[blk, :, at] = 0x7F
    out = torch.full((ln + 2, d + 8), 9.0, device=DEV, dtype=torch.bfloat16)
    p, s, q = pos[last].contiguous(), slot[last].contiguous(), qkv[last]
    ops.paged_attn8(q, kv, out, p, s, btab, bs, H, hd, ln, max(lens) + 3, append=append)
    torch.cuda.synchronize()
    assert ops.error_word() == 0
    assert torch.equal(kv, whole)
    assert float((out[ln:] - 9).abs().max()) == 0 and float((out[:, d:] - 9).abs().max()) == 0
    check_rows(out, q, kv, btab, bs, H, hd, p, s, range(min(ln, 6)))
    again = torch.zeros_like(out)
    ops.paged_attn8(q, kv, again, p, s, btab, bs, H, hd, ln, max(lens) + 3, append=append)
    assert torch.equal(again[:ln, :d], out[:ln, :d])              # the same bits in every call


@pytest.mark.parametrize("hd,H,bs,runs", [(32, 2, 2, [(0, 1), (0, 70), (13, 24)]), (32, 8, 16, [(200, 31), (499, 1)]), (64, 2, 16, [(0, 64), (0, 65), (63, 129), (5, 3)]),
                                          (64, 3, 5, [(300, 63), (1, 260)]), (128, 2, 16, [(0, 200), (127, 128), (1000, 17)]), (128, 1, 64, [(64, 64), (10, 500)]),
                                          (128, 4, 24, [(0, 300)]), (64, 1, 1, [(100, 140)])])
def test_attention_of_runs(hd, H, bs, runs):
    lens = [p + n for p, n in runs]
    kv, btab, pos, slot, qkv = make(hd + len(runs), lens, H, hd, bs, pad=8)
    d = H * hd
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, len(pos))
    new = torch.cat([torch.arange(n) >= p for (p, _), n in zip(runs, lens)]).to(DEV)
    q, p, s = qkv[new], pos[new].contiguous(), slot[new].contiguous()
    n = len(p)
    out = torch.full((n + 3, d + 8), 9.0, device=DEV, dtype=torch.bfloat16)
    starts, at = [], 0
    for _, k in runs:
        starts.append((at, k))
        at += k
    ops.paged_prefill8(q, kv, out, p, s, btab, bs, H, hd, starts, max(lens))
    torch.cuda.synchronize()
    assert ops.error_word() == 0
    assert float((out[n:] - 9).abs().max()) == 0 and float((out[:, d:] - 9).abs().max()) == 0
    rows = sorted({t for a, k in starts for t in (a, a + 1, a + k // 2, a + k - 1) if t < a + k})
    check_rows(out, q, kv, btab, bs, H, hd, p, s, rows, p_half_step=2.0 ** -8)
    one = torch.zeros(n, d, device=DEV, dtype=torch.bfloat16)      # all rows: as the single-token kernel has them
    ops.paged_attn8(q, kv, one, p, s, btab, bs, H, hd, n, max(lens))
    err = ((one.float() - out[:n, :d].float()).norm() / one.float().norm()).item()
    assert err < 2 * 2.0 ** -8, err


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_nan_reaches_the_rows_that_see_it_and_no_others(hd):
    H, bs, lens = 2, 16, [150, 40]
    kv, btab, pos, slot, qkv = make(hd, lens, H, hd, bs)
    d = H * hd
    qkv[70, 2 * d + 3] = math.nan                                 # v of position 70, head 0
    qkv[150 + 20, d + hd + 1] = math.nan                          # k of position 20 of the second, head 1
    n = len(pos)
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    kv_free = kv.clone()
    used = torch.zeros(kv.shape[0], dtype=torch.bool, device=DEV)
    used[btab[btab >= 0].long()] = True
    kv_free[~used] = 0xFF                                         # free blocks and the places behind the last token hold NaN codes
    for i, k in enumerate(lens):
        b, at = int(btab[i, k // bs]), k % bs
        kv_free[b, :, at * hd:bs * hd] = 0x7F
        kv_free[b, :, (bs + at) * hd:2 * bs * hd] = 0x7F
        kv_free[b, :, 2 * bs * hd + 2 * at:2 * bs * hd + 2 * bs] = 0xFF
    for pool in (kv, kv_free):
        out = torch.zeros(n, d, device=DEV, dtype=torch.bfloat16)
        one = torch.zeros(n, d, device=DEV, dtype=torch.bfloat16)
        ops.paged_prefill8(qkv, pool, out, pos, slot, btab, bs, H, hd, [(0, 150), (150, 40)], 160)
        ops.paged_attn8(qkv, pool, one, pos, slot, btab, bs, H, hd, n, 160)
        torch.cuda.synchronize()
        for o in (out, one):
            assert bool(o[70:150, 3].isnan().all()) and not bool(o[:70].isnan().any()) and not bool(o[:150, hd:].isnan().any())
            assert int(o[70:150, :hd].isnan().sum()) == 80
            assert bool(o[170:, hd:].isnan().all()) and not bool(o[150:170].isnan().any()) and not bool(o[150:, :hd].isnan().any())
        rows = [0, 69, 100, 149, 150, 169, 189]
        check_rows(out, qkv, kv, btab, bs, H, hd, pos, slot, rows, p_half_step=2.0 ** -8)
        check_rows(one, qkv, kv, btab, bs, H, hd, pos, slot, rows)
    assert ops.error_word() == 0


@pytest.mark.parametrize("hd", [64, 128])
def test_scales_far_apart_and_scores_far_apart(hd):
    """Values whose scales span 2^80 between positions, keys that give scores of some hundreds: the softmax is of one position, or of those that tie."""
    H, bs, n = 2, 16, 200
    kv, btab, pos, slot, qkv = make(hd, [n], H, hd, bs)
    d = H * hd
    g = torch.Generator().manual_seed(9)
    qkv[:, 2 * d:] = (qkv[:, 2 * d:].float() * (2.0 ** torch.randint(-40, 40, (n, 1), generator=g)).to(DEV)).bfloat16()
    qkv[:, :d] = qkv[:, :d] * 20
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    out, one = (torch.zeros(n, d, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    ops.paged_prefill8(qkv, kv, out, pos, slot, btab, bs, H, hd, [(0, n)], n)
    ops.paged_attn8(qkv, kv, one, pos, slot, btab, bs, H, hd, n, n)
    rows = [0, 1, 63, 64, 127, 130, 199]
    check_rows(out, qkv, kv, btab, bs, H, hd, pos, slot, rows, p_half_step=2.0 ** -8)
    check_rows(one, qkv, kv, btab, bs, H, hd, pos, slot, rows)
    assert ops.error_word() == 0


@pytest.mark.parametrize("hd,H,lens", [(32, 6, [384]), (64, 6, [384, 200]), (64, 12, [600, 600, 600, 600]), (32, 12, [600, 600, 600, 600]), (128, 6, [384]), (128, 12, [600, 600, 600, 600]),
                                       (64, 6, [900]), (128, 6, [900])])
def test_scores_that_rise_fall_and_jump_along_the_context(hd, H, lens):
    """The running maximum moves in every tile, in none after the first, or in some rows of a warp alone; by one CTA for all keys and by clusters."""
    bs = 16
    kv, btab, pos, slot, qkv = make(hd + H, lens, H, hd, bs)
    n, d, g = len(pos), H * hd, torch.Generator().manual_seed(hd)
    j = pos.cpu().float()
    for h in range(H):
        u = torch.randint(0, 2, (hd,), generator=g) * 2.0 - 1
        level = {0: 0.3 * j, 1: -0.3 * j, 2: (j % 97) * 0.8, 3: 60.0 * (j == 333), 4: 40.0 * (j // 64 % 2), 5: 0.0 * j}[h % 6]      # of a score, in log2 units
        q = 0.5 * u + 0.02 * torch.randn(n, hd, generator=g)
        q[(j % 8 == 3) & (h % 6 > 1)] *= -1                       # rows for which the jumps go down
        qkv[:, h * hd:(h + 1) * hd] = q.bfloat16().to(DEV)
        qkv[:, d + h * hd:d + (h + 1) * hd] = (level[:, None] / (0.5 * math.sqrt(hd) * 1.4427) * u + 0.1 * torch.randn(n, hd, generator=g)).bfloat16().to(DEV)
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    out, one, at, runs = torch.zeros(n, d, device=DEV, dtype=torch.bfloat16), torch.zeros(n, d, device=DEV, dtype=torch.bfloat16), 0, []
    for m in lens:
        runs.append((at, m))
        at += m
    ops.paged_prefill8(qkv, kv, out, pos, slot, btab, bs, H, hd, runs, max(lens))
    ops.paged_attn8(qkv, kv, one, pos, slot, btab, bs, H, hd, n, max(lens))
    rows = [0, 63, 64, 127, 128, 131, 191, lens[0] - 6, lens[0] - 1, n - 1]
    check_rows(out, qkv, kv, btab, bs, H, hd, pos, slot, rows, p_half_step=2.0 ** -8)
    check_rows(one, qkv, kv, btab, bs, H, hd, pos, slot, rows)
    assert ((out.float() - one.float()).norm() / one.float().norm()).item() < 2 * 2.0 ** -8 and ops.error_word() == 0


def test_indices_out_of_range_are_recorded_and_skipped():
    H, hd, bs, lens = 2, 64, 4, [10, 6]
    kv, btab, pos, slot, qkv = make(5, lens, H, hd, bs)
    d, n = H * hd, len(pos)
    assert ops.error_word() == 0
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    assert ops.error_word() == 0
    before = kv.clone()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    far = btab.clone()
    far[0, 0] = kv.shape[0]
    for p, s, tab in ((-1, 0, btab), (btab.shape[1] * bs, 0, btab), (0, -1, btab), (0, 2, btab), (12, 0, btab), (1, 0, far)):      # position 12: a page of -1
        ops.append_kv8(qkv, kv, i32(p), i32(s), tab, bs, H, hd, 1)
        torch.cuda.synchronize()
        assert ops.error_word() == 8 and torch.equal(kv, before)
        k, v = torch.full((1, d), 3.0, device=DEV), torch.full((1, d), 3.0, device=DEV)
        ops.read_kv8(kv, k, v, i32(p), i32(s), tab, bs, H, hd, 1)
        torch.cuda.synchronize()
        assert ops.error_word() == 8 and float((k - 3).abs().max()) == 0 == float((v - 3).abs().max())
        for append in (False, True):
            out = torch.full((1, d), 3.0, device=DEV, dtype=torch.bfloat16)
            ops.paged_attn8(qkv, kv, out, i32(p), i32(s), tab, bs, H, hd, 1, 1 << 20, append=append)
            torch.cuda.synchronize()
            assert ops.error_word() == 8 and (torch.equal(kv, before) or (tab is far and append))
        out = torch.full((1, d), 3.0, device=DEV, dtype=torch.bfloat16)
        ops.paged_prefill8(qkv, kv, out, i32(p), i32(s), tab, bs, H, hd, [(0, 1)], 1 << 20)
        torch.cuda.synchronize()
        assert ops.error_word() == 8 and torch.equal(kv, before)
    # padding rows (position -1) between real ones, and a context beyond max_ctx: those rows are left, the others right
    p, s = i32(9, -1, 5), i32(0, 0, 1)
    out = torch.full((3, d), 3.0, device=DEV, dtype=torch.bfloat16)
    ops.paged_attn8(qkv[:3], kv, out, p, s, btab, bs, H, hd, 3, 10)
    torch.cuda.synchronize()
    assert ops.error_word() == 8 and float((out[1] - 3).abs().max()) == 0
    check_rows(out, qkv[:3], kv, btab, bs, H, hd, p, s, [0, 2])
    out = torch.full((10, d), 3.0, device=DEV, dtype=torch.bfloat16)
    ops.paged_prefill8(qkv, kv, out, pos[:10], slot[:10], btab, bs, H, hd, [(0, 10)], 7)
    torch.cuda.synchronize()
    assert ops.error_word() == 8 and float((out[7:] - 3).abs().max()) == 0
    check_rows(out, qkv, kv, btab, bs, H, hd, pos, slot, [0, 6], p_half_step=2.0 ** -8)


def test_offsets_beyond_32_bits():
    """A cache of more than 4 GB whose sequences lie at its end."""
    H, hd, bs, lens = 16, 128, 64, [130, 70]
    rec = ops.kv8_record_bytes(bs, hd)
    blocks = (5 << 30) // (H * rec)
    kv, btab, pos, slot, qkv = make(6, lens, H, hd, bs, blocks=blocks)
    btab[btab >= 0] = blocks - 1 - torch.arange(int((btab >= 0).sum()), device=DEV, dtype=torch.int32)
    d, n = H * hd, len(pos)
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    small, tab = kv[-8:].clone(), torch.where(btab >= 0, btab - (blocks - 8), btab)
    a, b, a2, b2 = (torch.zeros(n, d, device=DEV, dtype=torch.bfloat16) for _ in range(4))
    ops.read_kv8(kv, a, b, pos, slot, btab, bs, H, hd, n)
    ops.read_kv8(small, a2, b2, pos, slot, tab, bs, H, hd, n)
    assert torch.equal(a, a2) and torch.equal(b, b2) and float(a.float().std()) > 0.5
    ops.paged_attn8(qkv, kv, a, pos, slot, btab, bs, H, hd, n, 200)
    ops.paged_attn8(qkv, small, a2, pos, slot, tab, bs, H, hd, n, 200)
    assert torch.equal(a, a2)
    ops.paged_prefill8(qkv, kv, a, pos, slot, btab, bs, H, hd, [(0, 130), (130, 70)], 200)
    ops.paged_prefill8(qkv, small, a2, pos, slot, tab, bs, H, hd, [(0, 130), (130, 70)], 200)
    assert torch.equal(a, a2)
    pool = kv.view(1, *kv.shape)
    ops.copy_blocks8(pool, torch.tensor([blocks - 1, 1], dtype=torch.int32, device=DEV), 1)
    assert torch.equal(kv[1], kv[-1]) and bool(kv[1].any())
    torch.cuda.synchronize()
    assert ops.error_word() == 0


@pytest.mark.parametrize("hd,H,bs", [(64, 4, 16), (128, 2, 16), (32, 4, 2)])
def test_prompt_then_decode_steps_eager_captured_and_on_another_stream(hd, H, bs):
    """A prompt appended and attended to in two pieces, then decode steps: replays of one captured step with new inputs in place, two captured steps
    alive at once, launches on a side stream -- all the same bits as eager launches, and right."""
    lens, steps = [37, 90, 5], 3
    kv, btab, pos, slot, qkv = make(hd, [n + steps for n in lens], H, hd, bs)
    d = H * hd
    eager = {}
    first = torch.cat([torch.arange(n + steps) < n // 2 for n in lens]).to(DEV)
    second = torch.cat([(torch.arange(n + steps) >= n // 2) & (torch.arange(n + steps) < n) for n in lens]).to(DEV)

    def runs_of(m):
        at, r = 0, []
        for i in range(len(lens)):
            k = int((m & (slot == i)).sum())
            r.append((at, k))
            at += k
        return r

    def prefill(pool):
        outs = []
        for m in (first, second):
            q, p, s = qkv[m], pos[m].contiguous(), slot[m].contiguous()
            o = torch.zeros(len(p), d, device=DEV, dtype=torch.bfloat16)
            ops.append_kv8(q, pool, p, s, btab, bs, H, hd, len(p))
            ops.paged_prefill8(q, pool, o, p, s, btab, bs, H, hd, runs_of(m), 128)
            check_rows(o, q, pool, btab, bs, H, hd, p, s, [0, len(p) // 2, len(p) - 1], p_half_step=2.0 ** -8)
            outs.append(o)
        return outs

    prefill(kv)
    base = kv.clone()
    starts = torch.tensor([sum(n + steps for n in lens[:i]) + n for i, n in enumerate(lens)], device=DEV)
    q, p, s = torch.zeros(3, 3 * d, device=DEV, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32, device=DEV), torch.arange(3, dtype=torch.int32, device=DEV)
    out = torch.zeros(3, d, device=DEV, dtype=torch.bfloat16)

    def load(k):
        q.copy_(qkv[starts + k])
        p.copy_(pos[starts + k])

    def step(pool, o=out):
        ops.paged_attn8(q, pool, o, p, s, btab, bs, H, hd, 3, 128, append=True)

    for k in range(steps):
        load(k)
        step(kv)
        check_rows(out, q, kv, btab, bs, H, hd, p, s, range(3))
        eager[k] = out.clone()
    done = kv.clone()
    pool = base.clone()
    other, out2 = base.clone(), torch.zeros_like(out)
    load(0)
    step(pool)                                                     # warm-up outside the capture (it writes what the replay writes)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        step(pool)
    with torch.cuda.graph(g2):
        step(other, out2)
    pool.copy_(base)
    for k in range(steps):
        load(k)
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[k]) and torch.equal(out2, eager[k])
    assert torch.equal(pool, done) and torch.equal(other, done)
    pool.copy_(base)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for k in range(steps):
            load(k)
            step(pool)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(pool, done) and torch.equal(out, eager[steps - 1])
    assert ops.error_word() == 0


@pytest.mark.parametrize("hd,bs", [(16, 3), (32, 16), (64, 5), (128, 16)])
def test_infinite_queries_and_queries_near_the_types_ends(hd, bs):
    """An infinity in q leaves no finite row, be the scores +inf or -inf, at the first position too and with the token's own k taken from its registers;
    magnitudes of 1e19 beside keys of 1e-19, and of 1e-30, are ordinary."""
    H, lens = 6, [1, 2, 9, 70, 300]
    kv, btab, pos, slot, qkv = make(hd, lens, H, hd, bs)
    n, d = len(pos), H * hd
    qkv[:, 0] = float("inf")                       # head 0; what the others take comes after it
    qkv[:, hd + 1] = float("-inf")
    qkv[:, 2 * hd + 2] = float("nan")
    qkv[:, 3 * hd:4 * hd] *= 1e19
    qkv[:, d + 3 * hd:d + 4 * hd] *= 1e-19
    qkv[:, 4 * hd:5 * hd] *= 1e-30
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    last = torch.tensor([sum(lens[:i + 1]) - 1 for i in range(len(lens))], device=DEV)
    q, p, s = qkv[last], pos[last].contiguous(), slot[last].contiguous()
    outs = []
    for append in (False, True):
        out = torch.zeros(len(lens), d, device=DEV, dtype=torch.bfloat16)
        ops.paged_attn8(q, kv, out, p, s, btab, bs, H, hd, len(lens), max(lens), append=append)
        check_rows(out, q, kv, btab, bs, H, hd, p, s, range(len(lens)))
        outs.append(out)
    assert bool(outs[0][:, :3 * hd].isnan().all()) and not bool(outs[0][:, 3 * hd:].isnan().any())
    if hd > 16:
        out, at, runs = torch.zeros(n, d, device=DEV, dtype=torch.bfloat16), 0, []
        for k in lens:
            runs.append((at, k))
            at += k
        ops.paged_prefill8(qkv, kv, out, pos, slot, btab, bs, H, hd, runs, max(lens))
        check_rows(out, qkv, kv, btab, bs, H, hd, pos, slot, [0, 2, 11, 12, 40, 81, 82, 200, n - 1], p_half_step=2.0 ** -8)
    assert ops.error_word() == 0


def test_direct_calls_recorded_ones_and_unusual_arguments_agree():
    """Calls that the extension launches itself, the same calls recorded and replayed by a launch plan, and calls with arguments that it leaves to Python
    (NumPy numbers, runs as a tuple): the same bits, and each counted as one launch."""
    import numpy as np
    H, hd, bs, n = 3, 64, 5, 90
    kv, btab, pos, slot, qkv = make(4, [n], H, hd, bs, pad=8)
    d = H * hd
    new = lambda: torch.zeros(n, d, device=DEV, dtype=torch.bfloat16)

    def calls(kv, outs, num=int, runs=list):
        ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, num(n - 1))
        ops.paged_attn8(qkv[n - 1:], kv, outs[0], pos[n - 1:], slot[n - 1:], btab, bs, H, hd, num(1), num(n), append=True)
        ops.paged_prefill8(qkv, kv, outs[1], pos, slot, btab, bs, H, hd, runs([(0, 20), (20, 70)]), num(n))
        ops.read_kv8(kv, outs[2], outs[3], pos, slot, btab, bs, H, hd, num(n))
    results = []
    for kw in ({}, dict(num=np.int64), dict(runs=tuple)):
        c, outs = kv.clone(), [new() for _ in range(4)]
        before = ops.launch_count
        calls(c, outs, **kw)
        assert ops.launch_count == before + 4
        results.append([c] + outs)
    c, outs, plan = kv.clone(), [new() for _ in range(4)], ops.LaunchPlan()
    with plan.record():
        calls(c, outs)
    for t in [c] + outs:
        t.zero_()
    plan.replay()
    results.append([c] + outs)
    for r in results[1:]:
        assert all(torch.equal(x, y) for x, y in zip(results[0], r))
    assert bool(results[0][1][0].abs().max() > 0) and ops.error_word() == 0


def test_limits_beyond_the_table_and_calls_without_work():
    H, hd, bs = 2, 64, 16
    kv, btab, pos, slot, qkv = make(3, [40], H, hd, bs)
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, 40)
    a, b = torch.zeros(2, 40, H * hd, device=DEV, dtype=torch.bfloat16)
    ops.paged_attn8(qkv, kv, a, pos, slot, btab, bs, H, hd, 40, 40)
    ops.paged_attn8(qkv, kv, b, pos, slot, btab, bs, H, hd, 40, 1 << 40)
    assert torch.equal(a, b)
    ops.paged_prefill8(qkv, kv, a, pos, slot, btab, bs, H, hd, [(0, 40)], 40)
    ops.paged_prefill8(qkv, kv, b, pos, slot, btab, bs, H, hd, [(0, 40)], 1 << 40)
    assert torch.equal(a, b)
    before = kv.clone()
    ops.paged_prefill8(qkv, kv, b, pos, slot, btab, bs, H, hd, [], 40)
    ops.paged_attn8(qkv, kv, b, pos, slot, btab, bs, H, hd, 0, 40, append=True)
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, 0)
    ops.read_kv8(kv, a, a, pos, slot, btab, bs, H, hd, 0)
    ops.copy_blocks8(kv.unsqueeze(0), torch.zeros(0, dtype=torch.int32, device=DEV), 0)
    assert torch.equal(a, b) and torch.equal(kv, before) and ops.error_word() == 0
    long = torch.zeros(1, (1 << 26) + 1, dtype=torch.int32, device=DEV)      # 2^30 positions and sixteen
    with pytest.raises(ops.KernelError):
        ops.append_kv8(qkv, kv, pos, slot, long, bs, H, hd, 40)


def test_refused_on_a_gpu():
    H, hd, bs = 2, 64, 16
    kv, btab, pos, slot, qkv = make(1, [20], H, hd, bs)
    out = torch.zeros(20, H * hd, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.append_kv8(qkv.half(), kv, pos, slot, btab, bs, H, hd, 20)
    with pytest.raises(ValueError):
        ops.append_kv8(qkv[:, :-8], kv, pos, slot, btab, bs, H, hd, 20)
    with pytest.raises(ValueError):
        ops.append_kv8(qkv, kv, pos.cpu(), slot, btab, bs, H, hd, 20)
    with pytest.raises(ValueError):
        ops.paged_attn8(qkv, kv, out[:10], pos, slot, btab, bs, H, hd, 20, 64)
    with pytest.raises(ValueError):
        ops.paged_attn8(qkv, kv, out.float(), pos, slot, btab, bs, H, hd, 20, 64)
    odd = torch.zeros(20 * 400 + 1, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ops.KernelError):                           # rows that are not 16-byte aligned
        ops.append_kv8(odd[1:].view(20, 400), kv, pos, slot, btab, bs, H, hd, 20)
    with pytest.raises(ops.KernelError):
        ops.paged_attn8(torch.zeros(20, 387, device=DEV, dtype=torch.bfloat16), kv, out, pos, slot, btab, bs, H, hd, 20, 64)
    with pytest.raises(ops.KernelError):
        ops.paged_prefill8(qkv, kv, odd[1:1 + 20 * 128].view(20, 128), pos, slot, btab, bs, H, hd, [(0, 20)], 64)
    assert float(grid()[126]) == 448.0 and ops.error_word() == 0


def test_fp32_rows_on_a_gpu_take_the_plain_evaluation():
    H, hd, bs = 2, 32, 4
    kv, btab, pos, slot, qkv = make(2, [9], H, hd, bs)
    kv2, out, out2 = kv.clone(), torch.zeros(9, 64, device=DEV), torch.zeros(9, 64, device=DEV, dtype=torch.bfloat16)
    ops.append_kv8(qkv.float(), kv, pos, slot, btab, bs, H, hd, 9)
    ops.append_kv8(qkv, kv2, pos, slot, btab, bs, H, hd, 9)
    assert torch.equal(kv, kv2)
    ops.paged_attn8(qkv.float(), kv, out, pos, slot, btab, bs, H, hd, 9, 16)
    ops.paged_attn8(qkv, kv, out2, pos, slot, btab, bs, H, hd, 9, 16)
    assert float((out - out2.float()).abs().max()) <= 2.0 ** -7 * float(out.abs().max())


@pytest.mark.parametrize("L,d,heads,bs", [(2, 128, 4, 8), (2, 256, 4, 16), (2, 256, 2, 5), (1, 64, 4, 2)])
def test_engine_over_the_8bit_cache(L, d, heads, bs, monkeypatch):
    """Prompts that join a step beside decoding sequences (runs of many and of few tokens, single ones), captured and eager decode steps, a shared prefix;
    and the logits of a prefill and of a mixed step against the same engine with the plain evaluation of the cache's operators.  Both round at the
    same points; what differs is a bf16 step of some attention outputs, and codes that this moves: the bound of the engine's other tests, 3e-2."""
    cfg = Config(L, d, heads, 300, 200, 1)
    m = GPT(cfg, DEV, torch.bfloat16)
    m.init_weights(1234)
    m.sync_bf16()
    g = torch.Generator().manual_seed(d + bs)
    prompts = [torch.randint(0, 300, (n,), generator=g).tolist() for n in (5, 130, 1, 70, 17, 2, 40)]
    new = [20, 12, 25, 9, 14, 30, 8]
    outs = {}
    for graphs in (True, False):
        e = InferEngine(m, block_size=bs, max_seqs=4, max_tokens=264, use_graphs=graphs, kv8=True)
        assert e.kc is None and not e.persistent
        a, _, _ = e.generate(prompts, new, max_active=3)
        b, _, _ = e.generate(prompts, new, max_active=3)
        assert a == b and (len(e.graphs) > 0) == graphs
        outs[graphs] = a
    assert outs[True] == outs[False]
    e = InferEngine(m, block_size=bs, max_seqs=6, kv8=True)
    grp, st, _ = e.generate_group(prompts[4], 5, 12)
    assert all(x == grp[0] for x in grp) and st["prefix_blocks_saved"] == 4 * (17 // bs)

    def logits():
        e = InferEngine(m, block_size=bs, max_seqs=8, max_tokens=512, use_graphs=False, kv8=True)
        got = []
        run = e._run

        def spy(ntok, nseq, rep=1):
            r = run(ntok, nseq, rep).clone()
            got.append((ntok, e.logits[:nseq, :300].float().clone()))
            return r
        e._run = spy
        e.generate(prompts, 1)                                     # one step: every prompt
        e.generate([prompts[1], prompts[6]], [4, 1], max_active=2)
        return got
    native = logits()
    from kharon_b200.ops import reference as ref

    def attn(qkv, kv, out, pos, slot, btab, bs, H, hd, ntok, max_ctx, append=False):
        if append:
            ref.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, ntok)
        ref.paged_attn8(qkv, kv, out, pos, slot, btab, bs, H, hd, ntok, max_ctx)

    def prefill(qkv, kv, out, pos, slot, btab, bs, H, hd, runs, max_ctx):
        for r, n in runs:
            ref.paged_attn8(qkv[r:r + n], kv, out[r:r + n], pos[r:r + n], slot[r:r + n], btab, bs, H, hd, n, max_ctx)
    monkeypatch.setattr(ops, "append_kv8", ref.append_kv8)
    monkeypatch.setattr(ops, "paged_attn8", attn)
    monkeypatch.setattr(ops, "paged_prefill8", prefill)
    plain = logits()
    assert [n for n, _ in native] == [n for n, _ in plain]
    for (_, x), (_, y) in zip(native[:2], plain[:2]):              # (later steps follow from the tokens chosen)
        assert ((x - y).norm() / y.norm()).item() < 3e-2
    assert ops.error_word() == 0


def test_long_runs_leave_no_status_code():
    """Many key tiles and more items than SMs, so that every role of the kernel for long runs waits for every other."""
    for hd, H, runs in ((128, 16, [(2000, 256), (1500, 700), (0, 300), (60, 129)]), (64, 16, [(0, 1000), (0, 511), (3000, 65)]), (32, 8, [(5000, 300), (100, 100)])):
        lens = [p + n for p, n in runs]
        kv, btab, pos, slot, qkv = make(hd, lens, H, hd, 16)
        ops.append_kv8(qkv, kv, pos, slot, btab, 16, H, hd, len(pos))
        new = torch.cat([torch.arange(n) >= p for (p, _), n in zip(runs, lens)]).to(DEV)
        q, p, s = qkv[new], pos[new].contiguous(), slot[new].contiguous()
        out, one = (torch.zeros(len(p), H * hd, device=DEV, dtype=torch.bfloat16) for _ in range(2))
        starts, at = [], 0
        for _, k in runs:
            starts.append((at, k))
            at += k
        for _ in range(20):
            ops.paged_prefill8(q, kv, out, p, s, btab, 16, H, hd, starts, max(lens))
        first = out.clone()
        ops.paged_prefill8(q, kv, out, p, s, btab, 16, H, hd, starts, max(lens))
        ops.paged_attn8(q, kv, one, p, s, btab, 16, H, hd, len(p), max(lens))
        torch.cuda.synchronize()
        assert ops.error_word() == 0 and torch.equal(first, out)
        assert ((one.float() - out.float()).norm() / one.float().norm()).item() < 2 * 2.0 ** -8


@pytest.mark.parametrize("where", [22, 45, 63, 64, 127])
def test_nan_keys_at_every_place_of_a_tile(where):
    """A NaN in a key makes the score of its position, and with it every row that sees it, NaN."""
    H, hd, bs, n = 2, 64, 16, 300
    kv, btab, pos, slot, qkv = make(where, [n], H, hd, bs)
    qkv[where, H * hd + 5] = math.nan
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    for runs in ([(0, n)], [(0, 100), (100, 64), (164, 136)]):
        out = torch.zeros(n, H * hd, device=DEV, dtype=torch.bfloat16)
        ops.paged_prefill8(qkv, kv, out, pos, slot, btab, bs, H, hd, runs, n)
        torch.cuda.synchronize()
        assert bool(out[where:, :hd].isnan().all()) and not bool(out[:where].isnan().any()) and not bool(out[:, hd:].isnan().any())
    assert ops.error_word() == 0
