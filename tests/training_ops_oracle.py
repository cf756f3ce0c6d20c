"""64-bit formulas of the decoder-training operators, with the error bounds their tests use.

Every function returns (reference, slack) pairs: ``slack`` bounds the fp32 arithmetic of the kernel
or restatement under test, before the one rounding to the output's type that ``close`` adds.
"""

import math

import numpy as np
import torch

U = 2.0 ** -24  # half a step of fp32
WORK = "cuda" if torch.cuda.is_available() else "cpu"  # where the 64-bit arithmetic runs


def w64(t):
    return t.detach().to(WORK).double()


def close(got, ref, slack, what=""):
    """|got - ref| <= half a step of got's type at ref, plus slack; equal NaN and infinities."""
    info = torch.finfo(got.dtype)
    g, r = w64(got), w64(ref)
    assert g.shape == r.shape, (what, g.shape, r.shape)
    odd = ~torch.isfinite(r)
    assert torch.equal(g[odd].nan_to_num(0.5), r[odd].nan_to_num(0.5)), f"{what}: infinities or NaN differ"
    bound = r.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2 + w64(slack)
    bad = ((g - r).abs() > bound) & ~odd | (~torch.isfinite(g) & ~odd)
    if bad.any():
        i = tuple(torch.nonzero(bad)[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; at {i} got {g[i]}, want {r[i]}, "
                             f"bound {bound[i]}")


# ------------------------------------------------------------------ head norms and rotation

def _rotation(rows, seq, hd, theta):
    pos = torch.arange(rows, dtype=torch.float64, device=WORK) % seq
    freq = torch.exp(torch.arange(hd // 2, dtype=torch.float64, device=WORK) * (-2.0 * math.log(theta) / hd))
    ang = torch.outer(pos, freq)
    return ang.cos()[:, None], ang.sin()[:, None]


def heads_forward(qkv, gq, gk, seq, H, HK, hd, theta, eps):
    T = qkv.shape[0]
    x = w64(qkv[:, :(H + HK) * hd]).view(T, H + HK, hd)
    g = torch.cat([w64(gq).expand(H, -1), w64(gk).expand(HK, -1)])
    u = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * g
    cs, sn = _rotation(T, seq, hd, theta)
    a, b = u[..., :hd // 2], u[..., hd // 2:]
    y = torch.cat([a * cs - b * sn, b * cs + a * sn], -1)
    # a norm (a sum of depth <= 24, a root) and two products of 1-2 ulp sines: < 32 half steps of the terms
    slack = 32 * U * (torch.cat([a.abs() + b.abs()] * 2, -1))
    return y.view(T, -1), slack.view(T, -1)


def heads_backward(dqk, qkv, gq, gk, seq, H, HK, hd, theta, eps):
    """((dx, slack), (dq_gain, slack), (dk_gain, slack))"""
    T = qkv.shape[0]
    x = w64(qkv[:, :(H + HK) * hd]).view(T, H + HK, hd)
    dy = w64(dqk[:, :(H + HK) * hd]).view(T, H + HK, hd)
    g = torch.cat([w64(gq).expand(H, -1), w64(gk).expand(HK, -1)])
    cs, sn = _rotation(T, seq, hd, theta)
    a, b = dy[..., :hd // 2], dy[..., hd // 2:]
    du = torch.cat([a * cs + b * sn, b * cs - a * sn], -1)
    big = torch.cat([a.abs() + b.abs()] * 2, -1)  # what du's terms can lose
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    w, xh = du * g, x * r
    dx = r * (w - xh * (w * xh).mean(-1, keepdim=True))
    wide = big * g.abs()
    slack = 64 * U * r * (wide + xh.abs() * (wide * xh.abs()).mean(-1, keepdim=True))
    terms, many = du * xh, big * xh.abs()
    # sums of depth <= 128 over a block's rows and heads, its lanes and warps, and the blocks
    gains = [(terms[:, s].sum((0, 1)), 160 * U * many[:, s].sum((0, 1))) for s in (slice(0, H), slice(H, H + HK))]
    return [(dx.view(T, -1), slack.view(T, -1))] + gains


# ------------------------------------------------------------------ dropout

def keep_bits(n, seed, offset):
    """The 16 random bits of elements 0 .. n-1: Philox4x32-10 in numpy's 64-bit words."""
    c = [np.zeros((n + 7) // 8, np.uint64) for _ in range(4)]
    c[0] += np.arange(len(c[0]), dtype=np.uint64)
    c[2] += np.uint64(offset % 2 ** 32)
    c[3] += np.uint64(offset // 2 ** 32)
    key = [seed % 2 ** 32, seed // 2 ** 32]
    low, half = np.uint64(2 ** 32 - 1), np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ np.uint64(key[0]), b & low, (a >> half) ^ c[3] ^ np.uint64(key[1]), a & low]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    return np.stack([w.astype("<u4") for w in c], 1).view("<u2").reshape(-1)[:n]


def dropout(x, p, seed, offset, residual=None):
    cut = round(p * 65536)
    keep = torch.from_numpy((keep_bits(x.numel(), seed, offset) >= cut).reshape(x.shape)).to(WORK)
    y = torch.where(keep, w64(x) * 65536 / (65536 - cut), 0.0)
    r = torch.zeros_like(y) if residual is None else w64(residual)
    return y + r, 2 * U * y.abs() + (0 if residual is None else U * (y.abs() + r.abs())), keep


# ------------------------------------------------------------------ losses over logits

def logprobs(logits, vocab, targets):
    """((logps, slack), (stats, slack), softmax, valid) in 64 bits; stats are [T, 2], a row's maximum and its sum."""
    x = w64(logits[:, :vocab])
    t = targets.to(WORK)
    valid = (t >= 0) & (t < vocab)
    m = x.nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf).amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    s = e.sum(-1, keepdim=True)
    empty = ((m == -math.inf) & (s == 0))[:, 0]
    p = e / s
    lp = (x.gather(1, t.clamp(0, vocab - 1)[:, None]) - m - s.log())[:, 0]
    lp = torch.where(valid, torch.where(empty, -math.inf, lp), 0.0)
    # each exponential is within 2 + 1.2 |x - m| steps; weighted by itself |x - m| averages below
    # log V + 1; running sums add a depth below 600
    slack = torch.full_like(lp, (2 * (2 + 1.2 * (math.log(vocab) + 1)) + 64) * U)
    stats = torch.cat([m, s], 1)
    return (lp, slack), (stats, torch.stack([torch.zeros_like(lp), s[:, 0].nan_to_num(0.0) * slack], 1)), torch.where(empty[:, None], 0.0, p), valid & ~empty


def dlogits(logits, vocab, targets, dlogps, dslack=0.0):
    (_, ls), (stats, _), p, valid = logprobs(logits, vocab, targets)
    up = torch.where(valid, w64(dlogps), 0.0)
    hot = torch.zeros_like(p).scatter_(1, targets.to(WORK).clamp(0, vocab - 1)[:, None], 1.0)
    zero = (up == 0)[:, None]
    d = torch.where(zero, 0.0, (hot - p) * up[:, None])
    x = w64(logits[:, :vocab])
    # the exponential's own steps, and those of the sum
    far = (x - stats[:, :1]).abs().nan_to_num(0.0, 0.0, 0.0)
    rel = 2 * (2 + 1.2 * far) * U + ls[:, None]
    slack = torch.where(zero, 0.0, up.abs()[:, None] * (p * rel + 4 * U * (hot + p)) + (hot - p).abs() * dslack)
    return d, slack.nan_to_num(0.0)


def policy(logits, vocab, targets, old, adv, w, ref, low, high, kl, scale):
    """((losses, slack), (logps, slack), (dlogits, slack))"""
    (lp, ls), _, _, valid = logprobs(logits, vocab, targets)
    tg = targets.to(WORK)
    has = (tg >= 0) & (tg < vocab)
    w = torch.ones_like(lp) if w is None else w64(w)
    A, ratio = w64(adv), torch.exp(lp - w64(old))
    gained = torch.where(A >= 0, A * ratio.clamp(max=1 + high), A * ratio.clamp(min=1 - low))
    inside = torch.where(A >= 0, ratio <= 1 + high, ratio >= 1 - low)
    loss, d = -gained, -torch.where(inside, A * ratio, 0.0)
    big = A.abs() * ratio.clamp(min=1)
    if ref is not None and kl:
        back = w64(ref) - lp
        loss, d = loss + kl * (torch.exp(back) - 1 - back), d + kl * (1 - torch.exp(back))
        big = big + kl * (torch.exp(back) + 1)
    used = has & (w != 0)
    loss, d, big = (torch.where(used, v * w, 0.0) for v in (loss, d, big))
    slack = big.abs() * (ls + 4 * U)
    dl, dls = dlogits(logits, vocab, targets, d * scale, (slack * abs(scale))[:, None])
    return (loss, slack), (lp, ls), (dl, dls)


def preference(logps, ref, mask, beta, form, smoothing, scale):
    """(losses, rewards, dlogps): fp64 inside, so their slack is nothing but the last rounding."""
    m = mask.to(WORK)
    diff = torch.where(m, w64(logps) - w64(ref), 0.0)
    r, n = diff.sum(1), m.sum(1).clamp(min=1)
    c, j = r[0::2], r[1::2]
    if form == "sigmoid":
        h = beta * (c - j)
        losses = (1 - smoothing) * torch.logaddexp(torch.zeros_like(h), -h) \
            + smoothing * torch.logaddexp(torch.zeros_like(h), h)
        slope = -(1 - smoothing) * torch.sigmoid(-h) + smoothing * torch.sigmoid(h)
        up = torch.stack([beta * slope, -beta * slope], 1).view(-1)
    else:
        gap = c / n[0::2] - j / n[1::2] - 1 / (2 * beta)
        losses = gap ** 2
        up = torch.stack([2 * gap / n[0::2], -2 * gap / n[1::2]], 1).view(-1)
    return losses, beta * r, torch.where(m, (up * scale)[:, None], 0.0)
