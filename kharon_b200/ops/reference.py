"""PyTorch evaluation of every operator, in fp32 math, writing into the caller's buffers.

Used (a) on CPU tensors, where it is the execution path of the CPU test tier and of the
fp32 oracle model, and (b) by the GPU tests as the plain-PyTorch reference each CUDA kernel
is compared against.  Storage dtype follows the tensors passed in (fp32 or bf16).
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F

EPI_NONE, EPI_BIAS, EPI_BIAS_GELU, EPI_BIAS_RESID, EPI_DGELU, EPI_RESID, EPI_GELU = range(7)

_K = 0.79788456
_C = 0.044715


def gelu(x):
    return 0.5 * x * (1.0 + torch.tanh(_K * (x + _C * x * x * x)))


def gelu_grad(x):
    u = _K * (x + _C * x * x * x)
    t = torch.tanh(u)
    return 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * _K * (1.0 + 3.0 * _C * x * x)


#: fp32 matrix product used by ``gemm``; the operator layer installs the native CUDA-core kernel
#: for GPU tensors (see ``ops._matmul_f32``), CPU tensors use torch.
matmul_f32 = None


def _mm(A, B):
    if matmul_f32 is not None and A.is_cuda:
        return matmul_f32(A, B)
    return A @ B


def gemm(a, b, out, a_mn, b_mn, accumulate, epi, bias, aux, alpha):
    A = a.float().t() if a_mn else a.float()
    Bm = b.float() if b_mn else b.float().t()
    acc = _mm(A, Bm) * alpha
    if epi in (EPI_BIAS, EPI_BIAS_GELU, EPI_BIAS_RESID, EPI_GELU):
        acc = acc + bias.float()
    if epi == EPI_BIAS_GELU:
        aux.copy_(acc)
        acc = gelu(aux.float())
    elif epi == EPI_GELU:
        acc = gelu(acc.to(out.dtype).float())
    elif epi in (EPI_BIAS_RESID, EPI_RESID):
        acc = acc + aux.float()
    elif epi == EPI_DGELU:
        acc = acc * gelu_grad(aux.float())
    if accumulate:
        out.add_(acc.to(out.dtype))
    else:
        out.copy_(acc)
    return out


def embed_fwd(tok, pos, wte, wpe, out, T):
    rows = out.shape[0]
    p = pos.long() if pos is not None else (torch.arange(rows, device=out.device) % T)
    out.copy_(wte.float()[tok.long()] + wpe.float()[p])
    return out


def embed_bwd(tok, dx, dwte, dwpe, B, T):
    d = dx.shape[1]
    if dwte is not None:
        dwte.index_add_(0, tok.long().reshape(-1), dx.float())
    if dwpe is not None:
        dwpe[:T].add_(dx.float().reshape(B, T, d).sum(0))


def colsum(x, out, accumulate):
    s = x.float().sum(0)
    if accumulate:
        out.add_(s)
    else:
        out.copy_(s)


def layernorm_fwd(x, w, b, y, mean, rstd):
    xf = x.float()
    mu = xf.mean(-1, keepdim=True)
    var = ((xf - mu) ** 2).mean(-1, keepdim=True)
    rs = torch.rsqrt(var + 1e-5)
    y.copy_((xf - mu) * rs * w.float() + b.float())
    if mean is not None:
        mean.copy_(mu.squeeze(-1))
    if rstd is not None:
        rstd.copy_(rs.squeeze(-1))
    return y


def layernorm_bwd(dy, x, w, mean, rstd, dres, dx, dw, db):
    g = dy.float()
    xh = (x.float() - mean.float()[:, None]) * rstd.float()[:, None]
    gw = g * w.float()
    s1 = gw.mean(-1, keepdim=True)
    s2 = (gw * xh).mean(-1, keepdim=True)
    o = rstd.float()[:, None] * (gw - s1 - xh * s2)
    if dres is not None:
        o = o + dres.float()
    dw.add_((g * xh).sum(0))
    db.add_(g.sum(0))
    dx.copy_(o)


def xent(logits, V, target, coef, uniform, rowloss, prob, write_grad):
    R = logits.shape[0]
    lg = logits[:, :V].float()
    lse = torch.logsumexp(lg, -1)
    t = target.long()
    valid = (t >= 0) & (t < V)
    ts = t.clamp(0, V - 1)
    xt = lg.gather(1, ts[:, None]).squeeze(1)
    if rowloss is not None:
        rowloss.copy_(torch.where(valid, lse - xt, torch.zeros_like(xt)))
    if prob is not None:
        prob.copy_(torch.where(valid, torch.exp(xt - lse), torch.zeros_like(xt)))
    if write_grad:
        sc = coef.float() if coef is not None else torch.full((R,), float(uniform), device=logits.device)
        sc = torch.where(valid, sc, torch.zeros_like(sc))
        p = torch.exp(lg - lse[:, None])
        onehot = F.one_hot(ts, V).float()
        logits.zero_()
        logits[:, :V] = ((p - onehot) * sc[:, None]).to(logits.dtype)


def xent_stats(logits, V, target, v0, stats):
    lg = logits[:, :V].float()
    m = lg.max(-1).values
    s = torch.exp(lg - m[:, None]).sum(-1)
    t = target.long() - v0
    inside = (t >= 0) & (t < V)
    xt = lg.gather(1, t.clamp(0, V - 1)[:, None]).squeeze(1)
    stats[:, 0] = m
    stats[:, 1] = s
    stats[:, 2] = torch.where(inside, xt, torch.full_like(xt, float("-inf")))


def xent_grad(logits, V, target, v0, gmax, gsum, coef, uniform):
    R = logits.shape[0]
    lg = logits[:, :V].float()
    tg = target.long()
    sc = coef.float() if coef is not None else torch.full((R,), float(uniform), device=logits.device)
    sc = torch.where(tg >= 0, sc, torch.zeros_like(sc))
    p = torch.exp(lg - gmax.float()[:, None]) / gsum.float()[:, None]
    t = tg - v0
    inside = (t >= 0) & (t < V)
    onehot = F.one_hot(t.clamp(0, V - 1), V).float() * inside[:, None].float()
    logits.zero_()
    logits[:, :V] = ((p - onehot) * sc[:, None]).to(logits.dtype)


def _log_probs(logits, V, target, on):
    """log softmax(x)[target] of the rows that count, else 0 (fp64), and the softmax."""
    lg = torch.where(on[:, None], logits[:, :V].double(), 0.0)
    ts = target.long().clamp(0, V - 1)
    lse = torch.logsumexp(lg, -1)
    lse = torch.where(lse == math.inf, math.nan, lse)              # of a row with an infinite logit, whose softmax has inf - inf
    lp = lg.gather(1, ts[:, None])[:, 0] - lse
    return torch.where(on, lp, 0.0), lg, lse, ts


def _put_gradient(dlogits, V, on, slope, lg, lse, ts):
    """slope (onehot - softmax) into the rows that count, zeros into the other rows' columns."""
    p = torch.exp(lg - lse[:, None])
    rest = p.scatter(1, ts[:, None], 0.0)
    p = -p
    p.scatter_(1, ts[:, None], rest.sum(-1, keepdim=True))         # 1 - p_t without the cancellation
    dlogits[:, V:] = 0
    dlogits[:, :V] = torch.where(on[:, None], p * slope[:, None], 0.0).to(dlogits.dtype)


def policy_loss(logits, V, target, adv, old_logp, ref_logp, lo, hi, beta, weight, uniform, rowloss, logp, kl, clipped, dlogits):
    R = logits.shape[0]
    if R == 0:
        return
    w = weight.double() if weight is not None else torch.full((R,), float(uniform), dtype=torch.float64, device=logits.device)
    on = (target >= 0) & (target < V) & (w != 0)
    lp, lg, lse, ts = _log_probs(logits, V, target, on)
    loss = torch.zeros_like(lp)
    slope, k, cl = torch.zeros_like(lp), torch.zeros_like(lp), torch.zeros_like(lp)
    if adv is not None:
        A = adv.double().reshape(-1).repeat_interleave(R // adv.numel())
        ratio = torch.exp(lp - old_logp.double()) if old_logp is not None else torch.where(torch.isnan(lp), lp, 1.0)
        raw, held = ratio * A, ratio.clamp(1.0 - lo, 1.0 + hi) * A
        cl = (raw > held).double()
        loss = -torch.where(raw > held, held, raw)
        slope = torch.where(raw > held, 0.0, -raw)
    if ref_logp is not None:
        d = ref_logp.double() - lp
        k = torch.expm1(d) - d
        if beta != 0:
            loss = loss + beta * k
            slope = slope - beta * torch.expm1(d)
    for out, value in ((rowloss, w * loss), (logp, lp), (kl, k), (clipped, cl)):
        if out is not None:
            out.view(-1).copy_(torch.where(on, value, 0.0))
    if dlogits is not None:
        _put_gradient(dlogits, V, on, w * slope, lg, lse, ts)


def preference_loss(logits, V, target, starts, ref_logp, beta, smoothing, weight, uniform, loss, margin, log_ratio, logp, dlogits):
    at, R = starts.tolist(), logits.shape[0]
    P = len(at) // 2
    if any(not 0 <= a <= b <= R for a, b in zip(at, at[1:])):
        raise IndexError("sequences outside the rows, or out of order")
    if P == 0:
        return
    a, b = at[0], at[-1]
    w = weight.double() if weight is not None else torch.full((P,), float(uniform), dtype=torch.float64, device=logits.device)
    seq = torch.repeat_interleave(torch.arange(2 * P, device=logits.device), starts.long().diff())
    tgt = target[a:b]
    on = (tgt >= 0) & (tgt < V) & (w != 0)[seq // 2]
    lp, lg, lse, ts = _log_probs(logits[a:b], V, tgt, on)
    over = lp if ref_logp is None else torch.where(on, lp - ref_logp[a:b].double(), 0.0)
    q = torch.zeros(2 * P, dtype=torch.float64, device=logits.device).index_add_(0, seq, over)
    m = beta * (q[0::2] - q[1::2])
    value = w * ((1.0 - smoothing) * F.softplus(-m) + smoothing * F.softplus(m))
    slope = torch.where(w != 0, w * beta * (smoothing * torch.sigmoid(m) - (1.0 - smoothing) * torch.sigmoid(-m)), 0.0)
    for out, v in ((loss, torch.where(w != 0, value, 0.0)), (margin, m), (log_ratio, q)):
        if out is not None:
            out.view(-1).copy_(v)
    if logp is not None:
        logp.view(-1)[a:b] = lp.to(logp.dtype)
    if dlogits is not None:
        _put_gradient(dlogits[a:b], V, on, torch.stack([slope, -slope], 1).view(-1)[seq], lg, lse, ts)


def clip_factor(sumsq, out, max_norm, left_out=None):
    norm = math.sqrt(float(sumsq)) if float(sumsq) >= 0 else math.nan
    factor = math.nan if not math.isfinite(norm) else 1.0 if norm <= max_norm else max_norm / norm
    out.view(-1).copy_(torch.tensor([norm, factor], dtype=torch.float64))         # (a norm beyond fp32's range shows as inf)
    if left_out is not None and math.isnan(factor):
        left_out += 1


def grad_norm(tensors, out, max_norm, sumsq, left_out=None):
    total = torch.tensor([sum(float(t.double().square().sum()) for t in tensors)], dtype=torch.float64)
    if sumsq is not None:
        sumsq.copy_(total)
    if out is not None:
        clip_factor(total, out, max_norm, left_out)


def scale(src, dst, out):
    f = float(out.view(-1)[1])
    for s, d in zip(src, dst):
        d.view(-1).copy_(s.view(-1) if math.isnan(f) else s.view(-1).float() * f)


def adamw(p, g, m, v, pb, lr, b1, b2, eps, wd, bc1, bc2, grad_scale, zero_grad):
    gk = g * grad_scale
    m.mul_(b1).add_(gk, alpha=1.0 - b1)
    v.mul_(b2).addcmul_(gk, gk, value=1.0 - b2)
    p.mul_(1.0 - lr * wd).sub_(lr * (m / bc1) / (torch.sqrt(v / bc2) + eps))
    if pb is not None:
        pb.copy_(p)
    if zero_grad:
        g.zero_()


def _heads(qkv, B, T, H, hd):
    d = H * hd
    x = qkv[:, : 3 * d].float().reshape(B, T, 3, H, hd)
    q, k, v = x[:, :, 0], x[:, :, 1], x[:, :, 2]
    return q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)   # [B,H,T,hd]


def flash_fwd(qkv, out, lse, B, T, H, hd):
    q, k, v = _heads(qkv, B, T, H, hd)
    s = (q @ k.transpose(-1, -2)) / math.sqrt(hd)
    mask = torch.ones(T, T, dtype=torch.bool, device=qkv.device).tril()
    s = s.masked_fill(~mask, float("-inf"))
    l = torch.logsumexp(s, -1)
    p = torch.exp(s - l[..., None])
    o = p @ v
    out.copy_(o.transpose(1, 2).reshape(B * T, H * hd))
    if lse is not None:
        lse.copy_(l)


def flash_bwd(qkv, out, dout, lse, dqkv, B, T, H, hd):
    q, k, v = _heads(qkv, B, T, H, hd)
    d = H * hd
    do = dout.float().reshape(B, T, H, hd).transpose(1, 2)
    s = (q @ k.transpose(-1, -2)) / math.sqrt(hd)
    mask = torch.ones(T, T, dtype=torch.bool, device=qkv.device).tril()
    s = s.masked_fill(~mask, float("-inf"))
    p = torch.softmax(s, -1)
    dv = p.transpose(-1, -2) @ do
    dp = do @ v.transpose(-1, -2)
    ds = p * (dp - (dp * p).sum(-1, keepdim=True)) / math.sqrt(hd)
    dq = ds @ k
    dk = ds.transpose(-1, -2) @ q
    res = torch.stack([dq, dk, dv], 0).permute(1, 3, 0, 2, 4).reshape(B * T, 3 * d)
    dqkv[:, : 3 * d] = res.to(dqkv.dtype)


def append_kv(qkv, kc, vc, pos, slot, btab, bs, H, hd, ntok):
    d = H * hd
    p = pos[:ntok].long()
    blk = btab[slot[:ntok].long(), p // bs].long()
    kc[blk, p % bs] = qkv[:ntok, d:2 * d].reshape(ntok, H, hd).to(kc.dtype)
    vc[blk, p % bs] = qkv[:ntok, 2 * d:3 * d].reshape(ntok, H, hd).to(vc.dtype)


def paged_attn(qkv, kc, vc, out, pos, slot, btab, bs, H, hd, ntok):
    d = H * hd
    p = pos[:ntok].long()
    ctx = int(p.max()) + 1
    j = torch.arange(ctx, device=qkv.device)
    blk = btab[slot[:ntok].long()][:, j // bs].long().clamp_(min=0)          # [ntok, ctx]
    K = kc[blk, (j % bs)[None, :]].float()                                   # [ntok, ctx, H, hd]
    Vv = vc[blk, (j % bs)[None, :]].float()
    q = qkv[:ntok, :d].float().reshape(ntok, H, hd)
    s = torch.einsum("the,tjhe->thj", q, K) / math.sqrt(hd)
    s = s.masked_fill((j[None, :] > p[:, None])[:, None, :], float("-inf"))
    out[:ntok] = torch.einsum("thj,tjhe->the", torch.softmax(s, -1), Vv).reshape(ntok, d).to(out.dtype)


def kv8_views(kv, bs, hd):
    """(codes of k, codes of v [..., bs, hd], exponent bytes [..., bs, 2]) of records [..., record]."""
    n = bs * hd
    return kv[..., :n].unflatten(-1, (bs, hd)), kv[..., n:2 * n].unflatten(-1, (bs, hd)), kv[..., 2 * n:2 * n + 2 * bs].unflatten(-1, (bs, 2))


def kv8_quantise(x):
    """Rows [..., hd] -> (e4m3 codes, exponent bytes [...]): the smallest exponent in [-63, 63] for which no magnitude exceeds 448."""
    x = x.float()
    a = x.abs().nan_to_num(nan=0.0, posinf=math.inf).amax(-1)
    m, e = torch.frexp(a.clamp(max=2.0 ** 100))                                  # a = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(a > 0, e - 9 + (m > 0.875).int(), torch.full_like(e, -63)).clamp(-63, 63)
    y = x * ((127 - e) << 23).view(torch.float32)[..., None]
    return y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)


def _kv8_places(kv, pos, slot, btab, bs, ntok):
    p, s = pos[:ntok].long(), slot[:ntok].long()
    if ntok and (int(p.min()) < 0 or int(p.max()) >= btab.shape[1] * bs or int(s.min()) < 0 or int(s.max()) >= btab.shape[0]):
        raise IndexError("a position or a sequence outside the block table")
    blk = btab[s, p // bs].long()
    if ntok and (int(blk.min()) < 0 or int(blk.max()) >= kv.shape[0]):
        raise IndexError("a block outside the cache")
    return blk, p % bs


def append_kv8(qkv, kv, pos, slot, btab, bs, H, hd, ntok):
    d = H * hd
    blk, at = _kv8_places(kv, pos, slot, btab, bs, ntok)
    ck, cv, ce = kv8_views(kv, bs, hd)
    for codes, which in ((ck, 0), (cv, 1)):
        q, e = kv8_quantise(qkv[:ntok, (which + 1) * d:(which + 2) * d].reshape(ntok, H, hd))
        codes[blk, :, at] = q
        ce[..., which][blk, :, at] = e


def _kv8_load(kv, blk, at, bs, hd):
    """k, v [*blk.shape, H, hd] in fp32."""
    ck, cv, ce = kv8_views(kv, bs, hd)
    s = (ce[blk, :, at].int() << 23).view(torch.float32)
    f = lambda c, which: c[blk, :, at].view(torch.float8_e4m3fn).float() * s[..., which, None]
    return f(ck, 0), f(cv, 1)


def read_kv8(kv, k, v, pos, slot, btab, bs, H, hd, ntok):
    blk, at = _kv8_places(kv, pos, slot, btab, bs, ntok)
    x, y = _kv8_load(kv, blk, at, bs, hd)
    k[:ntok, :H * hd] = x.reshape(ntok, H * hd).to(k.dtype)
    v[:ntok, :H * hd] = y.reshape(ntok, H * hd).to(v.dtype)


def paged_attn8(qkv, kv, out, pos, slot, btab, bs, H, hd, ntok, max_ctx):
    if ntok == 0:
        return
    d = H * hd
    _kv8_places(kv, pos, slot, btab, bs, ntok)
    p = pos[:ntok].long()
    if int(p.max()) >= max_ctx:
        raise IndexError("a position beyond max_ctx")
    for t in range(ntok):
        j = torch.arange(int(p[t]) + 1, device=kv.device)
        blk = btab[slot[t].long(), j // bs].long()
        if int(blk.min()) < 0 or int(blk.max()) >= kv.shape[0]:
            raise IndexError("a block outside the cache")
        k, v = _kv8_load(kv, blk, j % bs, bs, hd)                                # [ctx, H, hd]
        s = torch.einsum("he,jhe->hj", qkv[t, :d].float().reshape(H, hd), k) / math.sqrt(hd)
        out[t, :d] = torch.einsum("hj,jhe->he", torch.softmax(s, -1), v).reshape(d).to(out.dtype)


def sample(logits, V, temperature, seed, step, rep, out, nseq):
    lg = logits[:nseq, :V].float()
    if temperature <= 0:
        idx = lg.argmax(-1)
        out[:nseq * rep].copy_(idx.repeat_interleave(rep).to(out.dtype))
        return
    g = torch.Generator().manual_seed((int(seed) * 1000003 + int(step)) & 0x7FFFFFFF)
    p = torch.softmax(lg / temperature, -1).cpu()
    idx = torch.multinomial(p, rep, replacement=True, generator=g).to(out.device)
    out[:nseq * rep].copy_(idx.reshape(-1).to(out.dtype))
