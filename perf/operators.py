"""Performance cases of the 8-bit paged KV cache: writing it, reading it back, and the attention over it.

A layer's cache is ``uint8 [n_blocks, H, record]``.  The record of a (block, head) holds the e4m3 codes of the block's keys
(``bs * hd`` bytes) and values (as many), then a pair of exponent bytes (key, value) for each position, and is padded to a multiple of 32
bytes.  A row of ``hd`` numbers x is kept as x = code * 2^(byte - 127), with the smallest exponent in [-63, 63] for which no magnitude
exceeds 448.

``own`` selects the framework's operators; otherwise ``run`` evaluates the same formulas with elementary torch operations.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
E_MIN, E_MAX, TOP = -63, 63, 448.0


# ------------------------------------------------------------------------------------------------ cases
def _append(name, seqs, lo, hi, H, hd, bs, mix):
    return dict(name=name, op="append", seqs=seqs, lo=lo, hi=hi, H=H, hd=hd, bs=bs, mix=mix)


def _read(name, seqs, lo, hi, H, hd, bs, mix):
    return dict(name=name, op="read", seqs=seqs, lo=lo, hi=hi, H=H, hd=hd, bs=bs, mix=mix)


def _decode(name, seqs, lo, hi, H, hd, bs, mix):
    return dict(name=name, op="decode", seqs=seqs, lo=lo, hi=hi, H=H, hd=hd, bs=bs, mix=mix)


def _chunk(name, seqs, lo, hi, nlo, nhi, H, hd, bs, mix):
    """``seqs`` pieces of nlo..nhi new tokens, each behind lo..hi cached positions."""
    return dict(name=name, op="chunk", seqs=seqs, lo=lo, hi=hi, nlo=nlo, nhi=nhi, H=H, hd=hd, bs=bs, mix=mix)


def listed():
    return [
        # the new tokens of one decode step of 32 users, by themselves: all latency
        _append("append-32", 32, 1, 1, 16, 64, 16, 1),
        # the prompts of a prefill step: 6 of ragged lengths, wide heads
        _append("append-prompts", 6, 403, 1900, 16, 128, 16, 2),
        # one cached conversation read back, to be handed to another engine
        _read("read-one", 1, 777, 777, 8, 64, 16, 3),
        # the cache of a batch of conversations read back
        _read("read-batch", 16, 1000, 4000, 16, 128, 16, 4),
        # one greedy completion of a byte-level policy: pages of two positions, a context of a few tokens
        _decode("decode-tiny", 1, 18, 18, 8, 32, 2, 5),
        # one user at the end of a long conversation: few rows, so the context itself has to be shared out
        _decode("decode-long", 1, 16300, 16300, 16, 64, 16, 6),
        # a server under load: ragged contexts
        _decode("decode-32", 32, 20, 1000, 16, 64, 16, 7),
        # a full server with wide heads and long contexts: all bandwidth
        _decode("decode-128", 128, 1000, 4096, 16, 128, 16, 8),
        # short pieces that join a step beside decoding users, narrow heads
        _chunk("chunk-short", 2, 200, 500, 24, 31, 8, 32, 16, 9),
        # six fresh prompts of odd lengths: time to first token
        _chunk("chunk-prompts", 6, 0, 0, 403, 1001, 16, 64, 16, 10),
        # the next turns of four conversations, wide heads
        _chunk("chunk-turns", 4, 1500, 4000, 384, 640, 16, 128, 16, 11),
        # one piece of a very long prompt
        _chunk("chunk-long", 1, 14300, 14300, 2048, 2048, 16, 128, 16, 12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "decode", "decode", "decode", "chunk", "chunk", "chunk"])
    H, hd, bs, mix = rng.choice([4, 8, 8, 16, 16]), rng.choice([32, 64, 64, 128]), rng.choice([2, 8, 16, 16, 24, 64]), rng.randrange(1 << 16)
    if op in ("append", "read"):
        seqs, hi = _log(rng, 1, 64), _log(rng, 1, 4000)
        hi = max(1, min(hi, (40000 if op == "read" else 8000) // seqs))
        c = (_append if op == "append" else _read)("", seqs, max(1, hi // rng.randint(1, 4)), hi, H, hd, bs, mix)
    elif op == "decode":
        seqs, hi = _log(rng, 1, 128), _log(rng, 1, 16384)
        hi = max(1, min(hi, 128 * 2500 * 16 * 128 // (seqs * H * hd)))
        c = _decode("", seqs, max(1, hi // rng.randint(1, 8)), hi, H, hd, bs, mix)
    else:
        seqs, nhi, hi = _log(rng, 1, 12), _log(rng, 16, 2048), rng.choice([0, _log(rng, 1, 14000)])
        while seqs * nhi * (hi + nhi) * H * hd > 2048 * 15000 * 16 * 128:      # at most the largest listed one
            seqs, nhi, hi = max(1, seqs // 2), nhi if seqs > 1 else max(1, nhi // 2), hi if seqs > 1 else hi // 2
        c = _chunk("", seqs, hi // rng.randint(1, 4), hi, max(1, nhi // rng.randint(1, 3)), nhi, H, hd, bs, mix)
    c.pop("name")
    return c


def _lengths(c):
    """(cached positions before the call, new tokens) of each sequence, from the case alone."""
    r = random.Random(c["mix"])
    lens = [r.randint(c["lo"], c["hi"]) for _ in range(c["seqs"])]
    if c["op"] == "append":
        return [(0, n) for n in lens]
    if c["op"] == "read":
        return [(n, n) for n in lens]
    if c["op"] == "decode":                       # ``lens`` counts the new token
        return [(n - 1, 1) for n in lens]
    return [(n, r.randint(c["nlo"], c["nhi"])) for n in lens]


def work(c):
    H, hd, ls = c["H"], c["hd"], _lengths(c)
    d, new = H * hd, sum(n for _, n in ls)
    stored = 2 * d + 2 * H                         # bytes of a cached position
    if c["op"] == "append":
        return {"bytes": new * (4 * d + stored + 8), "flops": new * 4 * d}
    if c["op"] == "read":
        return {"bytes": new * (4 * d + stored + 8), "flops": new * 2 * d}
    if c["op"] == "decode":
        return {"bytes": sum(p * stored + 8 * d + stored + 8 for p, _ in ls), "flops": sum(4 * d * (p + 1) for p, _ in ls)}
    return {"bytes": sum((p + n) * stored + n * (4 * d + 8) for p, n in ls), "flops": sum(4 * d * (n * p + n * (n + 1) // 2) for p, n in ls)}


# ------------------------------------------------------------------------------------------------ the cache's format
def _power(e):
    """2^e of integers, exactly (its bits)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x):
    """Rows [..., hd] -> (e4m3 values, exponent bytes [...])."""
    x = x.float()
    a = x.abs().amax(-1)
    e = torch.frexp(a / TOP)
    e = (e.exponent - (e.mantissa == 0.5).int()).clamp(E_MIN, E_MAX)            # smallest e with amax / 448 <= 2^e
    e = e.masked_fill(a == 0, E_MIN)
    return (x * _power(-e)[..., None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _views(kv, bs, hd):
    """(key codes, value codes, exponent bytes) of a cache [n_blocks, H, record]: [n_blocks, H, bs, hd] twice and [n_blocks, H, bs, 2]."""
    n = bs * hd
    return (kv[..., :n].unflatten(-1, (bs, hd)).view(torch.float8_e4m3fn), kv[..., n:2 * n].unflatten(-1, (bs, hd)).view(torch.float8_e4m3fn),
            kv[..., 2 * n:2 * n + 2 * bs].unflatten(-1, (bs, 2)))


def _store(kv, bs, hd, blk, at, k, v):
    """Rows k, v [n, H, hd] into block ``blk[i]``, position ``at[i]``."""
    ck, cv, ce = _views(kv, bs, hd)
    (qk, ek), (qv, ev) = _quantise(k), _quantise(v)
    ck.view(torch.uint8)[blk, :, at] = qk.view(torch.uint8)
    cv.view(torch.uint8)[blk, :, at] = qv.view(torch.uint8)
    ce[blk, :, at] = torch.stack([ek, ev], -1)


def _load(kv, bs, hd, blk, at):
    """Keys and values [*blk.shape, H, hd] of the listed places."""
    ck, cv, ce = _views(kv, bs, hd)
    s = _power(ce[blk, :, at].int() - 127)
    return (ck.view(torch.uint8)[blk, :, at].view(torch.float8_e4m3fn).float() * s[..., 0, None],
            cv.view(torch.uint8)[blk, :, at].view(torch.float8_e4m3fn).float() * s[..., 1, None])


# ------------------------------------------------------------------------------------------------ preparation
def prepare(c, seed):
    H, hd, bs = c["H"], c["hd"], c["bs"]
    d, ls = H * hd, _lengths(c)
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    total = [p + n if c["op"] != "read" else n for p, n in ls]
    pages = [(t + bs - 1) // bs for t in total]
    n_blocks, max_lb = sum(pages) + 3, max(pages) + 2
    order = torch.randperm(n_blocks, generator=g, device=DEV).int()
    btab = torch.full((c["seqs"], max_lb), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(pages):
        btab[i, :n] = order[at:at + n]
        at += n
    rec = (2 * bs * hd + 2 * bs + 31) // 32 * 32
    kv = torch.zeros(n_blocks, H, rec, dtype=torch.uint8, device=DEV)
    if c["op"] != "append":                        # keys of about unit size, values whose size differs from position to position
        ck, cv, ce = _views(kv, bs, hd)
        for b in range(0, n_blocks, max(1, (1 << 27) // (bs * d))):
            part = slice(b, b + max(1, (1 << 27) // (bs * d)))
            shape = ck[part].shape
            for codes, which, spread in ((ck, 0, 0.2), (cv, 1, 0.7)):
                q, e = _quantise((rand(*shape) * torch.exp(spread * rand(*shape[:3], 1))).bfloat16())
                codes.view(torch.uint8)[part] = q.view(torch.uint8)
                ce[part][..., which] = e
    first = [0 if c["op"] == "read" else p for p, _ in ls]
    slot = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, (_, n) in enumerate(ls)]).to(DEV)
    pos = torch.cat([torch.arange(p, p + n, dtype=torch.int32) for p, (_, n) in zip(first, ls)]).to(DEV)
    ntok = pos.numel()
    s = dict(case=dict(c), kv=kv, pos=pos, slot=slot, btab=btab, ntok=ntok, max_ctx=max_lb * bs)
    if c["op"] == "read":
        s["k"], s["v"] = (torch.empty(ntok, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        return s
    qkv = rand(ntok, 3 * d)
    qkv[:, :d] *= 1.5                              # scores with a standard deviation of about 1.5
    s["qkv"] = qkv.bfloat16()
    s["out"] = torch.zeros(ntok, d, dtype=torch.bfloat16, device=DEV)
    if c["op"] == "chunk":                         # the new tokens' keys and values are in the cache already, as after an append
        k, v = s["qkv"][:, d:2 * d].reshape(ntok, H, hd), s["qkv"][:, 2 * d:].reshape(ntok, H, hd)
        p = pos.long()
        _store(kv, bs, hd, btab[slot.long(), p // bs].long(), p % bs, k, v)
        starts, at = [], 0
        for _, n in ls:
            starts.append((at, n))
            at += n
        s["runs"] = starts
        n_max = max(n for _, n in ls)              # the runs as rows of a rectangle, for the plain form
        t = torch.arange(n_max, device=DEV)
        s["row"] = torch.tensor([a for a, _ in starts], device=DEV)[:, None] + torch.minimum(t, torch.tensor([n - 1 for _, n in ls], device=DEV)[:, None])
        s["real"] = t < torch.tensor([n for _, n in ls], device=DEV)[:, None]
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    H, hd, bs, op = c["H"], c["hd"], c["bs"], c["op"]
    kv, pos, slot, btab, ntok = s["kv"], s["pos"], s["slot"], s["btab"], s["ntok"]
    if own:
        from kharon_b200 import ops
        if op == "append":
            ops.append_kv8(s["qkv"], kv, pos, slot, btab, bs, H, hd, ntok)
        elif op == "read":
            ops.read_kv8(kv, s["k"], s["v"], pos, slot, btab, bs, H, hd, ntok)
        elif op == "decode":
            ops.paged_attn8(s["qkv"], kv, s["out"], pos, slot, btab, bs, H, hd, ntok, s["max_ctx"], append=True)
        else:
            ops.paged_prefill8(s["qkv"], kv, s["out"], pos, slot, btab, bs, H, hd, s["runs"], s["max_ctx"])
    else:
        d, p = H * hd, pos.long()
        if op in ("append", "decode"):
            _store(kv, bs, hd, btab[slot.long(), p // bs].long(), p % bs, s["qkv"][:, d:2 * d].reshape(ntok, H, hd), s["qkv"][:, 2 * d:].reshape(ntok, H, hd))
        if op == "read":
            k, v = _load(kv, bs, hd, btab[slot.long(), p // bs].long(), p % bs)
            s["k"], s["v"] = k.reshape(ntok, d).bfloat16(), v.reshape(ntok, d).bfloat16()
        elif op == "decode":
            s["out"] = _attend(s, kv, slot[:, None], p[:, None], s["qkv"][:, None, :d])[:, 0].to(torch.bfloat16)
        elif op == "chunk":
            row = s["row"]
            o = _attend(s, kv, slot[row], p[row], s["qkv"][row, :d])
            s["out"] = o[s["real"]].to(torch.bfloat16)
    if op == "read":
        return {"k": s["k"], "v": s["v"]}
    ck, cv, ce = _views(kv, bs, hd)
    if op == "append":
        return {"k": ck, "v": cv, "e": ce}
    if op == "decode":
        return {"out": s["out"], "k": ck, "v": cv, "e": ce}
    return {"out": s["out"]}


def _attend(s, kv, slot, pos, q):
    """Sequences of equally many queries: q [S, n, H * hd] at positions pos [S, n] of the sequences slot [S, n]."""
    c = s["case"]
    H, hd, bs = c["H"], c["hd"], c["bs"]
    S, n = pos.shape
    j = torch.arange(max(p + m for p, m in _lengths(c)), device=DEV)
    blk = s["btab"][slot[:, 0].long()][:, j // bs].long().clamp(min=0)
    k, v = _load(kv, bs, hd, blk, (j % bs).expand_as(blk))                      # [S, ctx, H, hd]
    sc = q.float().reshape(S, n, H, hd).transpose(1, 2) @ k.permute(0, 2, 3, 1) / math.sqrt(hd)
    sc = sc.masked_fill((j > pos[..., None])[:, None], float("-inf"))           # [S, H, n, ctx]
    sc = torch.exp(sc - sc.amax(-1, keepdim=True))
    o = (sc / sc.sum(-1, keepdim=True)) @ v.transpose(1, 2)
    return o.transpose(1, 2).reshape(S, n, H * hd)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _powers():
    """2^k for k = E_MIN .. E_MAX."""
    return torch.tensor([2.0 ** k for k in range(E_MIN, E_MAX + 1)], dtype=torch.float64, device=DEV)


def _grid():
    """The 127 magnitudes of e4m3 in order: eight steps of 2^-9, then eight to each power of two, up to 448."""
    return torch.tensor([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1],
                        dtype=torch.float64, device=DEV)


def _exact_rows(x):
    """Index into the grid, sign and exponent of every number of the rows x: the nearest magnitude, the even index of two."""
    x, powers, grid = x.double(), _powers(), _grid()
    e = torch.searchsorted(TOP * powers, x.abs().amax(-1).contiguous()).clamp(max=E_MAX - E_MIN)       # first k with amax <= 448 2^k
    y = (x.abs() / powers[e][..., None]).clamp(max=TOP)
    up = torch.searchsorted(grid, y.contiguous()).clamp(max=126)
    dn = (up - 1).clamp(min=0)
    a, b = y - grid[dn], grid[up] - y
    i = torch.where((a < b) | ((a == b) & (dn % 2 == 0)), dn, up)
    return torch.where(x < 0, -grid[i], grid[i]), e + E_MIN


def _exact_cache(kv, table, bs, hd, n):
    """Keys and values [n, H, hd] of a sequence's first n positions, from the bytes."""
    grid, powers, place = _grid(), _powers(), torch.arange(n)
    both = torch.cat([grid, grid.new_full((1,), math.nan)])
    both = torch.cat([both, -both])
    rec = kv[table[place // bs].to(DEV)]                                        # [n, H, record]
    off = (place % bs).to(DEV)[:, None, None]
    cols = torch.arange(hd, device=DEV)
    out = []
    for which in range(2):
        code = rec.gather(-1, ((which * bs + off) * hd + cols).expand(n, rec.shape[1], hd))
        e = rec.gather(-1, (2 * bs * hd + 2 * off + which).expand(n, rec.shape[1], 1))
        out.append(both[code.long()] * powers[(e.long() - 127 - E_MIN).clamp(0, E_MAX - E_MIN)])
    return out


def exact(c, seed):
    H, hd, bs = c["H"], c["hd"], c["bs"]
    s = prepare(c, seed)
    d, ls = H * hd, _lengths(c)
    kv, btab = s["kv"], s["btab"].cpu().long()
    if c["op"] == "append":
        out = {"k": torch.zeros(kv.shape[0], H, bs, hd, dtype=torch.float64, device=DEV)}
        out["v"], out["e"] = torch.zeros_like(out["k"]), torch.zeros(kv.shape[0], H, bs, 2, dtype=torch.uint8, device=DEV)
        at = 0
        for i, (_, n) in enumerate(ls):
            place = torch.arange(n)
            blk, off = btab[i, place // bs].to(DEV), (place % bs).to(DEV)
            for which, name in enumerate("kv"):
                y, e = _exact_rows(s["qkv"][at:at + n, (which + 1) * d:(which + 2) * d].reshape(n, H, hd))
                out[name][blk, :, off] = y
                out["e"][..., which][blk, :, off] = (e + 127).to(torch.uint8)
            at += n
        return out
    rows, at = [], 0
    for i, (p, n) in enumerate(ls):
        have = n if c["op"] == "read" else p + n
        if c["op"] == "read":
            k, v = _exact_cache(kv, btab[i], bs, hd, n)
            rows.append((k.reshape(n, d), v.reshape(n, d)))
            continue
        new = s["qkv"][at:at + n]
        k, v = _exact_cache(kv, btab[i], bs, hd, have)
        if c["op"] == "decode":
            for x, col in ((k, 1), (v, 2)):
                y, e = _exact_rows(new[:, col * d:(col + 1) * d].reshape(n, H, hd))
                x[p:] = y * _powers()[e - E_MIN][..., None]
        at += n
        outs = []
        for h in range(H):
            sc = new[:, h * hd:(h + 1) * hd].double() @ k[:, h].t() / math.sqrt(hd)
            sc = sc.masked_fill(torch.arange(have, device=DEV) > p + torch.arange(n, device=DEV)[:, None], float("-inf"))
            outs.append(torch.softmax(sc, -1) @ v[:, h])
        rows.append(torch.cat(outs, -1))
    if c["op"] == "read":
        return {"k": torch.cat([a for a, _ in rows]), "v": torch.cat([b for _, b in rows])}
    out = {"out": torch.cat(rows)}
    return out if c["op"] == "chunk" else {**out, "k": None, "v": None, "e": None}
