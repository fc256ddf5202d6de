"""The 8-bit cache's operators from their definition, in 64 bits and without the package's code, and how far a kernel may be from them."""
import math

import torch

E_LO, E_HI = -63, 63


def grid():
    """Value of each of the 256 e4m3 codes."""
    v = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)]
    v[127] = math.nan
    return torch.tensor(v + [-x for x in v], dtype=torch.float64)


def quantise(x):
    """Rows [n, hd] -> (values on the grid times 2^e, e [n]); one number at a time."""
    g = grid()[:127].tolist()
    out, exps = [], []
    for row in x.double().tolist():
        a = max([abs(t) for t in row if t == t], default=0.0)
        e = next((k for k in range(E_LO, E_HI) if a <= 448.0 * 2.0 ** k), E_HI)
        vals = []
        for t in row:
            if t != t:
                vals.append(math.nan)
                continue
            y = min(abs(t) / 2.0 ** e, 448.0)
            i = min(range(127), key=lambda i: (abs(g[i] - y), i % 2))            # nearest, the even index of two
            vals.append(math.copysign(g[i] * 2.0 ** e, t))
        out.append(vals)
        exps.append(e)
    return torch.tensor(out, dtype=torch.float64), torch.tensor(exps)


def rows_of(kv, table, bs, hd, n):
    """Keys and values [n, H, hd] (float64) of a sequence's first n positions, from the bytes of a cache on the CPU."""
    g, out = grid(), []
    rec = kv.reshape(kv.shape[0], kv.shape[1], -1)
    for which in range(2):
        x = torch.empty(n, kv.shape[1], hd, dtype=torch.float64)
        for j in range(n):
            r, at = rec[int(table[j // bs])], j % bs
            code = r[:, (which * bs + at) * hd:(which * bs + at + 1) * hd].long()
            x[j] = g[code] * torch.pow(2.0, r[:, 2 * bs * hd + 2 * at + which].double() - 127)[:, None]
        out.append(x)
    return out


def attend(q, k, v, p_half_step=0.0):
    """One token: q [H, hd], k, v [ctx, H, hd], all float64.  Returns (o [H, hd], bound [H, hd] on a kernel's error).

    A kernel sums hd products for a score in fp32, in any order: off by at most hd * 2^-24 * sum |q k| (one more rounding each for the two scales and
    the reference, 2^-22 for the exponential), which moves p_j by that factor and o by twice it (numerator and normaliser).  The
    sums over ctx positions add ctx * 2^-24, counted on sum p |v|; `p_half_step` is a rounding of the probabilities before P V.  The output is
    rounded to bf16: half a step, 2^-8 of the value."""
    hd, ctx = q.shape[-1], k.shape[0]
    s = torch.einsum("he,jhe->hj", q, k) / math.sqrt(hd)
    p = torch.softmax(s, -1)
    o = torch.einsum("hj,jhe->he", p, v)
    mag = torch.einsum("hj,jhe->he", p, v.abs())
    top = torch.einsum("he,jhe->hj", q.abs(), k.abs()).amax(-1) / math.sqrt(hd)
    c = 2 * ((hd + 4) * 2.0 ** -24 * top + 2.0 ** -21) + 2 * (ctx + 8) * 2.0 ** -24 + p_half_step
    return o, 2.0 ** -8 * o.abs() + (1 + 2.0 ** -8) * c[:, None] * mag + 1e-30


def attend_own(q, k, v, p_half_step=0.0, floor=0.0, each=0.0):
    """``attend`` with a bound that counts each score by its own terms, so that one large key excuses nothing in the others.

    The score of key j is off by at most delta_j = (hd + 4) * 2^-24 * sum |q k_j| / sqrt(hd) + 2^-21 (exponential), so p_j lies between what it is with its own
    score moved one way and all others the other way; o is off by those differences times |v_j|, by ctx * 2^-24 of sum p |v| for the
    sums, and by `p_half_step` of it where the probabilities are rounded before P V.  `floor`: the smallest step of such a rounding, half of it, relative to the
    largest probability of the row, which every position may be off by; `each`: the same where the kernel bounds it by itself, as part of a whole.  Output in bf16."""
    hd, ctx = q.shape[-1], k.shape[0]
    s = torch.einsum("he,jhe->hj", q, k) / math.sqrt(hd)
    p = torch.softmax(s, -1)
    o = torch.einsum("hj,jhe->he", p, v)
    d = (hd + 4) * 2.0 ** -24 * torch.einsum("he,jhe->hj", q.abs(), k.abs()) / math.sqrt(hd) + 2.0 ** -21
    eye = torch.eye(ctx, dtype=torch.bool)
    others = lambda x: x[:, None, :].masked_fill(eye, -math.inf).logsumexp(-1)    # over the other keys
    hi = torch.sigmoid((s + d) - others(s - d)) if ctx > 1 else torch.ones_like(p)
    lo = torch.sigmoid((s - d) - others(s + d)) if ctx > 1 else torch.ones_like(p)
    dp = torch.maximum(hi - p, p - lo).clamp(min=0)
    mag = torch.einsum("hj,jhe->he", p, v.abs())
    err = torch.einsum("hj,jhe->he", dp, v.abs()) + ((ctx + 8) * 2.0 ** -24 + p_half_step) * mag + (floor * p.amax(-1)[:, None] + each) * v.abs().sum(0)
    return o, 2.0 ** -8 * o.abs() + (1 + 2.0 ** -8) * err + 1e-30


def quantising_oracle(cfg, model):
    """The PyTorch statement of the architecture, with keys and values replaced by what the 8-bit cache keeps of them (a row is a token and head)."""
    from kharon_b200.models.oracle import OracleGPT
    o = OracleGPT(cfg)
    o.load_from(model)
    g, hd = grid()[:127].float(), cfg.d_model // cfg.n_head

    def kept(x):
        rows = x.reshape(-1, hd)
        a = rows.abs().amax(-1)
        e = torch.zeros_like(a)
        for k in range(-40, 41):
            e = torch.where(a > 448.0 * 2.0 ** k, torch.full_like(a, 2.0 ** (k + 1)), e)
        e = e.clamp(min=2.0 ** -40)
        y = rows.abs() / e[:, None]
        up = torch.searchsorted(g, y.contiguous()).clamp(max=126)
        dn = (up - 1).clamp(min=0)
        lo, hi = y - g[dn], g[up] - y
        i = torch.where((lo < hi) | ((lo == hi) & (dn % 2 == 0)), dn, up)
        return (torch.sign(rows) * g[i] * e[:, None]).reshape(x.shape)

    def hook(module, args, out):
        q, k, v = out.split(cfg.d_model, dim=-1)
        return torch.cat([q, kept(k), kept(v)], -1)

    for b in o.blocks:
        b.qkv.register_forward_hook(hook)
    return o
