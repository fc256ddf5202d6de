"""The 8-bit cache's attention where queries, keys or values differ widely in size, against 64 bits with a bound for each key's own terms."""
import math

import pytest
import torch

from kharon_b200 import ops
from kv8_exact import attend_own, rows_of
from test_kv8_gpu import make

pytestmark = pytest.mark.gpu
DEV = "cuda"
# Rounding of the probabilities in runs of more than 64 tokens: they are f16, whose numbers in [1, 2) are 2^-10 apart, so half a step is 2^-11 of the value; half the smallest
# step is 2^-32 of the largest probability times 2^(difference of two value rows' exponents), 14 at most as `make` draws them.  Single tokens: two such terms, 2^-39.
RUN, RUN_FLOOR, ONE_FLOOR = torch.finfo(torch.float16).eps / 2, 2.0 ** -18, 2.0 ** -25
# What the single-token kernel leaves of it, or takes the positions again.
ONE_EACH = 2.0 ** -29
# What the kernel of long runs leaves of it, of the mean |v|, or computes the row again.
RUN_MEAN = 2.0 ** -9


def smallest_step(q, k, ev):
    """[H]: what half the smallest step of a probability in f16 may move o by, in the kernel of long runs, per unit of sum |v|.  Probabilities are 2^(s + EV - R) with EV the
    largest exponent of a tile of 128 values' rows (masked ones too) and R at most 7 below the largest s + EV, so the step is 2^-25 2^(R - EV) over sum 2^s."""
    n, s = k.shape[0], torch.einsum("he,jhe->hj", q, k) / math.sqrt(q.shape[-1]) / math.log(2)
    tiles = torch.stack([ev[a:a + 128].amax(0) for a in range(0, len(ev), 128)])            # [tiles, H]
    top = (s + tiles.repeat_interleave(128, 0)[:n].t()).amax(-1)
    return torch.exp2(-25 + top - 7 - tiles[:(n + 127) // 128].amin(0) - s.mul(math.log(2)).logsumexp(-1) / math.log(2))


def check(out, q, kv, btab, bs, H, hd, pos, slot, rows, p_half_step, floor, each=0.0, mean=0.0):
    kv, btab, pos, slot, q, out = kv.cpu(), btab.cpu(), pos.cpu(), slot.cpu(), q.double().cpu(), out.double().cpu()
    cache = {}
    for t in rows:
        s, n = int(slot[t]), int(pos[t]) + 1
        if s not in cache:
            cache[s] = rows_of(kv, btab[s], bs, hd, max(int(pos[u]) + 1 for u in rows if int(slot[u]) == s))
        if mean:
            ev = torch.stack([kv[int(btab[s][j // bs]), :, 2 * bs * hd + 2 * (j % bs) + 1].double() - 127 for j in range(len(cache[s][0]))])
            each = smallest_step(q[t, :H * hd].view(H, hd), cache[s][0][:n], ev).clamp(max=mean / n)[:, None]
        want, tol = attend_own(q[t, :H * hd].view(H, hd), cache[s][0][:n], cache[s][1][:n], p_half_step, floor, each)
        err = (out[t, :H * hd].view(H, hd) - want).abs()
        assert not bool(want.isnan().any()) and bool((err <= tol).all()), (t, n, float((err / tol).nan_to_num(1e30).max()))


def both(qkv, kv, pos, slot, btab, bs, H, hd, lens):
    """(runs, single tokens) of all rows."""
    out, one, at, runs = torch.zeros(len(pos), H * hd, device=DEV, dtype=torch.bfloat16), torch.zeros(len(pos), H * hd, device=DEV, dtype=torch.bfloat16), 0, []
    for n in lens:
        runs.append((at, n))
        at += n
    ops.paged_prefill8(qkv, kv, out, pos, slot, btab, bs, H, hd, runs, max(lens))
    ops.paged_attn8(qkv, kv, one, pos, slot, btab, bs, H, hd, len(pos), max(lens))
    torch.cuda.synchronize()
    assert ops.error_word() == 0
    return out, one


# (head width, heads, lengths): one group of rows, two groups with rows of their own, clusters with shared and with own rows
SHAPES = [(32, 2, [300]), (64, 2, [300]), (128, 2, [300]), (32, 2, [700]), (64, 2, [100, 700]), (128, 2, [700]), (128, 2, [520, 100]), (64, 12, [600, 600, 600, 600]), (128, 12, [600, 600, 600, 600])]


@pytest.mark.parametrize("hd,H,lens", [(16, 2, [90]), (32, 2, [300]), (64, 2, [40, 700]), (128, 2, [300])])
@pytest.mark.parametrize("power", [22, 25, 30, 45, 60])
def test_scores_beyond_the_integers_of_fp32(hd, H, lens, power):
    """Scores of some 2^power, where neighbouring numbers of fp32 are more than one apart: one position has all the weight, and no probability is out of range."""
    bs = 16
    kv, btab, pos, slot, qkv = make(hd + power, lens, H, hd, bs)
    n, d = len(pos), H * hd
    qkv[:, d:2 * d] *= 2.0 ** power
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    rows = list(range(0, n, 7)) + [n - 1]
    one = torch.zeros(n, d, device=DEV, dtype=torch.bfloat16)
    ops.paged_attn8(qkv, kv, one, pos, slot, btab, bs, H, hd, n, max(lens))
    check(one, qkv, kv, btab, bs, H, hd, pos, slot, rows, 0.0, ONE_FLOOR)
    assert ops.error_word() == 0


@pytest.mark.parametrize("hd,H,lens", SHAPES)
@pytest.mark.parametrize("power", [24, 30, 34, 70, 200])
def test_one_key_far_larger_than_the_others(hd, H, lens, power):
    """A key 2^power times the others (2^200: infinite) is as good as absent for the rows before it and for those whose product with it is negative; the others see
    it alone.  Its neighbours in a tile keep their own scores."""
    bs, at = 16, (40, 141)
    kv, btab, pos, slot, qkv = make(hd + power, lens, H, hd, bs)
    n, d = len(pos), H * hd
    for j in at:
        m = pos == j
        qkv[m, d:2 * d] = (qkv[m, d:2 * d].double() * 2.0 ** power).to(torch.bfloat16)
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    out, one = both(qkv, kv, pos, slot, btab, bs, H, hd, lens)
    rows = [0, 30, 39, 40, 41, 45, 99, 140, 141, 142, 150, 155, 200, lens[0] - 1, n - 1] if lens[0] > 200 else [5, 39, 40, 60, 99, 100 + 140, 100 + 141, 100 + 150, 100 + 155, 100 + 400, n - 1]
    check(out, qkv, kv, btab, bs, H, hd, pos, slot, rows, RUN, RUN_FLOOR)
    check(one, qkv, kv, btab, bs, H, hd, pos, slot, rows, 0.0, ONE_FLOOR)


@pytest.mark.parametrize("hd,H,lens", [(16, 2, [90]), (32, 2, [300]), (64, 2, [40, 700]), (128, 2, [300])])
@pytest.mark.parametrize("power", [50, 62, 66, 70])
def test_small_queries_beside_large_keys(hd, H, lens, power):
    """Queries of 2^-power and keys of 2^power give ordinary scores."""
    bs = 16
    kv, btab, pos, slot, qkv = make(hd + power, lens, H, hd, bs)
    n, d = len(pos), H * hd
    qkv[:, :d] *= 2.0 ** -power
    qkv[:, d:2 * d] *= 2.0 ** power / 4
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    rows = [0, 1, 39, 41, 80, n - 40, n - 1]
    if hd > 16:
        out, one = both(qkv, kv, pos, slot, btab, bs, H, hd, lens)
        check(out, qkv, kv, btab, bs, H, hd, pos, slot, rows, RUN, RUN_FLOOR)
    else:
        one = torch.zeros(n, d, device=DEV, dtype=torch.bfloat16)
        ops.paged_attn8(qkv, kv, one, pos, slot, btab, bs, H, hd, n, max(lens))
    check(one, qkv, kv, btab, bs, H, hd, pos, slot, rows, 0.0, ONE_FLOOR)



@pytest.mark.parametrize("hd,H,lens", [(16, 2, [90]), (32, 2, [300]), (64, 2, [40, 700]), (128, 2, [300])])
def test_queries_near_the_types_end_beside_small_keys(hd, H, lens):
    """Queries of 3e37 and keys of 1e-17: scores of some 1e20, finite, and one position has all the weight."""
    bs = 16
    kv, btab, pos, slot, qkv = make(hd, lens, H, hd, bs)
    n, d = len(pos), H * hd
    qkv[:, :d] *= 3e37
    qkv[:, d:2 * d] *= 1e-17
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    rows = [0, 1, 39, 41, 80, n - 40, n - 1]
    if hd > 16:
        out, one = both(qkv, kv, pos, slot, btab, bs, H, hd, lens)
        check(out, qkv, kv, btab, bs, H, hd, pos, slot, rows, RUN, RUN_FLOOR)
    else:
        one = torch.zeros(n, d, device=DEV, dtype=torch.bfloat16)
        ops.paged_attn8(qkv, kv, one, pos, slot, btab, bs, H, hd, n, max(lens))
    check(one, qkv, kv, btab, bs, H, hd, pos, slot, rows, 0.0, ONE_FLOOR)
    one.zero_()                                                   # the token's own key from its registers
    last = torch.tensor([sum(lens[:i + 1]) - 1 for i in range(len(lens))], device=DEV)
    k = len(lens)
    ops.paged_attn8(qkv[last], kv, one, pos[last].contiguous(), slot[last].contiguous(), btab, bs, H, hd, k, max(lens), append=True)
    check(one, qkv[last], kv, btab, bs, H, hd, pos[last], slot[last], range(k), 0.0, ONE_FLOOR)
    assert ops.error_word() == 0



@pytest.mark.parametrize("hd,H,bs,lens", [(16, 2, 16, [1, 2, 90]), (32, 4, 5, [40, 700]), (64, 2, 16, [33, 1000]), (128, 2, 24, [700, 5]), (64, 16, 16, [60] * 150), (128, 2, 16, [3000])])
@pytest.mark.parametrize("append", [False, True])
def test_single_tokens_with_an_infinite_value_or_scales_far_apart(hd, H, bs, lens, append):
    """An infinity in one element of a cached value (head 0: kept as the largest number) leaves the other elements to the other positions; head 1: scales from 2^-30 to 2^30."""
    kv, btab, pos, slot, qkv = make(hd, lens, H, hd, bs)
    n, d, g = len(pos), H * hd, torch.Generator().manual_seed(3)
    qkv[pos == min(lens[-1] - 1, 20), 2 * d + 2] = math.inf
    qkv[:, 2 * d + hd:2 * d + 2 * hd] *= (2.0 ** torch.randint(-30, 30, (n, 1), generator=g)).to(DEV)
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    last = torch.tensor([sum(lens[:i + 1]) - 1 for i in range(len(lens))], device=DEV)
    k = len(lens)
    q, p, s, out = qkv[last], pos[last].contiguous(), slot[last].contiguous(), torch.zeros(k, d, device=DEV, dtype=torch.bfloat16)
    ops.paged_attn8(q, kv, out, p, s, btab, bs, H, hd, k, max(lens), append=append)
    check(out, q, kv, btab, bs, H, hd, p, s, range(min(k, 4)), 0.0, 0.0, ONE_EACH)
    again = torch.zeros_like(out)
    ops.paged_attn8(q, kv, again, p, s, btab, bs, H, hd, k, max(lens), append=append)
    assert torch.equal(out, again) and ops.error_word() == 0


@pytest.mark.parametrize("hd,H,bs,lens", [(16, 2, 16, [1, 2, 90]), (32, 4, 5, [40, 700]), (64, 2, 16, [33, 1000]), (128, 2, 24, [700, 5]), (64, 16, 16, [60] * 150), (128, 2, 16, [3000])])
@pytest.mark.parametrize("append", [False, True])
def test_single_tokens_whose_query_has_one_element_far_larger_than_the_others(hd, H, bs, lens, append):
    """The keys are zero where the query is 2^60 times as large: the other elements make the scores."""
    kv, btab, pos, slot, qkv = make(hd, lens, H, hd, bs)
    n, d = len(pos), H * hd
    qkv[:, 3:d:hd] *= 2.0 ** 60
    qkv[:, d + 3:2 * d:hd] = 0.0
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    last = torch.tensor([sum(lens[:i + 1]) - 1 for i in range(len(lens))], device=DEV)
    k = len(lens)
    q, p, s, out = qkv[last], pos[last].contiguous(), slot[last].contiguous(), torch.zeros(k, d, device=DEV, dtype=torch.bfloat16)
    ops.paged_attn8(q, kv, out, p, s, btab, bs, H, hd, k, max(lens), append=append)
    check(out, q, kv, btab, bs, H, hd, p, s, range(min(k, 4)), 0.0, 0.0, ONE_EACH)
    assert ops.error_word() == 0


@pytest.mark.parametrize("hd,H,lens", SHAPES)
def test_values_of_the_smallest_scale_beside_ordinary_ones(hd, H, lens):
    """Position 0's values lie below 448 * 2^-63, where the exponent ends: the row that sees nothing else has them as they are.  Rows of zeros beside them change nothing."""
    bs = 16
    kv, btab, pos, slot, qkv = make(hd, lens, H, hd, bs)
    n, d = len(pos), H * hd
    qkv[pos == 0, 2 * d:] *= 2.0 ** -56
    qkv[(pos > 3) & (pos % 5 == 0), 2 * d:] = 0.0
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    out, one = both(qkv, kv, pos, slot, btab, bs, H, hd, lens)
    rows = [0, 1, 5, 80, lens[0] - 1, n - 1]
    check(out, qkv, kv, btab, bs, H, hd, pos, slot, rows, RUN, RUN_FLOOR)
    check(one, qkv, kv, btab, bs, H, hd, pos, slot, rows, 0.0, 0.0, ONE_EACH)



@pytest.mark.parametrize("hd,H,lens", SHAPES)
@pytest.mark.parametrize("power", [8, 12, 14, 17, 20, 22, 40])
@pytest.mark.parametrize("early", [True, False])
def test_one_value_row_far_larger_than_the_others(hd, H, lens, power, early):
    """One row of values 2^power times the others, in one element only: in the first tile, where all later rows see it with next to no weight, or further on, where some must
    not see it.  The other elements keep their bits."""
    bs, j = 16, 20 if early else max(lens) - 150
    kv, btab, pos, slot, qkv = make(hd + power, lens, H, hd, bs)
    n, d = len(pos), H * hd
    m = pos == j
    for h in range(H):
        qkv[m, 2 * d + h * hd:2 * d + (h + 1) * hd] = 0.0
        qkv[m, 2 * d + h * hd + 1] = 2.0 ** power
    qkv[m, d:2 * d] = 0.0
    qkv[pos > j, d:2 * d] *= 0.25
    if early:
        qkv[m, d:2 * d] = -qkv[:1, :d] * 4                         # (queries are alike: a score far below the others')
        qkv[:, :d] = (qkv[:1, :d].float() + 0.3 * qkv[:, :d].float()).bfloat16()
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    out, one = both(qkv, kv, pos, slot, btab, bs, H, hd, lens)
    first = n - lens[-1] if lens[-1] == max(lens) else 0
    rows = [first + t for t in (0, j - 20, j - 1, j, j + 1, j + 60, j + 149, max(lens) - 30, max(lens) - 1)]
    check(out, qkv, kv, btab, bs, H, hd, pos, slot, rows, RUN, 0.0, mean=RUN_MEAN)
    check(one, qkv, kv, btab, bs, H, hd, pos, slot, rows, 0.0, 0.0, ONE_EACH)


@pytest.mark.parametrize("hd,H,lens", [(32, 2, [700]), (64, 2, [700]), (128, 2, [700])])
def test_values_whose_scales_differ_between_tiles(hd, H, lens):
    """The first 256 positions' values are 0, the next ones' 2^-60 and the last ones' 2^62: the zeros have their weight."""
    bs = 16
    kv, btab, pos, slot, qkv = make(hd, lens, H, hd, bs)
    n, d = len(pos), H * hd
    qkv[pos < 256, 2 * d:] = 0.0
    qkv[(pos >= 256) & (pos < 512), 2 * d:] *= 2.0 ** -60
    qkv[pos >= 512, 2 * d:] *= 2.0 ** 62
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    out, one = both(qkv, kv, pos, slot, btab, bs, H, hd, lens)
    rows = [0, 255, 256, 300, 511, 512, 600, 699]
    check(out, qkv, kv, btab, bs, H, hd, pos, slot, rows, RUN, 0.0, mean=RUN_MEAN)
    check(one, qkv, kv, btab, bs, H, hd, pos, slot, rows, 0.0, 0.0, ONE_EACH)


@pytest.mark.parametrize("hd,H,lens", SHAPES)
@pytest.mark.parametrize("power", [18, 22, 25, 30, 45, 60])
def test_runs_with_scores_beyond_the_integers_of_fp32(hd, H, lens, power):
    """Scores of some 2^power, where neighbouring numbers of fp32 are far apart: one position has all the weight, and its values come out as they are."""
    bs = 16
    kv, btab, pos, slot, qkv = make(hd + power, lens, H, hd, bs)
    n, d = len(pos), H * hd
    qkv[:, d:2 * d] *= 2.0 ** power
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    out, _ = both(qkv, kv, pos, slot, btab, bs, H, hd, lens)
    check(out, qkv, kv, btab, bs, H, hd, pos, slot, list(range(0, min(n, 700), 17)) + [n - 1], RUN, 0.0, mean=RUN_MEAN)


@pytest.mark.parametrize("hd,H,lens", SHAPES)
def test_runs_whose_queries_have_one_element_far_larger_than_the_others(hd, H, lens):
    """The keys are zero where the query is 2^60 times as large: the other elements make the scores."""
    bs = 16
    kv, btab, pos, slot, qkv = make(hd, lens, H, hd, bs)
    n, d = len(pos), H * hd
    qkv[:, 3:d:hd] *= 2.0 ** 60
    qkv[:, d + 3:2 * d:hd] = 0.0
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    out, one = both(qkv, kv, pos, slot, btab, bs, H, hd, lens)
    rows = [0, 1, 39, 41, 80, n - 40, n - 1]
    check(out, qkv, kv, btab, bs, H, hd, pos, slot, rows, RUN, 0.0, mean=RUN_MEAN)
    check(one, qkv, kv, btab, bs, H, hd, pos, slot, rows, 0.0, 0.0, ONE_EACH)


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("n,half_step,mean", [(64, 0.0, 0.0), (300, RUN, RUN_MEAN), (700, RUN, RUN_MEAN)])
def test_probabilities_keep_the_bits_that_are_stated(hd, n, half_step, mean):
    """All keys but the first have the same score, whose probability over the first's lies halfway between two numbers of eight bits, and the first position's values
    cancel most of what the others add up to: a rounding of the probabilities is not averaged out, and not hidden by the output's."""
    H, bs = 2, 16
    kv, btab, pos, slot, qkv = make(hd, [n], H, hd, bs)
    x = qkv.zero_().view(n, 3, H, hd)
    gap = -math.log(194.5 / 256)                                   # of the scores
    x[:, 0, :, 0] = gap * math.sqrt(hd)
    x[0, 1, :, 0] = 1.0
    x[:, 2] = 1.0
    x[0, 2] = -math.exp(-gap) * (n - 1) * 0.97                     # the last row's sum is what is cancelled
    ops.append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, n)
    out, one = both(qkv, kv, pos, slot, btab, bs, H, hd, [n])
    rows = [n - 1, n - 2, n // 2]
    check(out, qkv, kv, btab, bs, H, hd, pos, slot, rows, half_step, 0.0, mean=mean)
    check(one, qkv, kv, btab, bs, H, hd, pos, slot, rows, 0.0, 0.0, ONE_EACH)
