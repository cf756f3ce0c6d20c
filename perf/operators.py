"""Workloads of the decoder-training operators: head norms with rotation, dropout, preference and policy losses.

Each case is one call, or one run of calls, as a training step makes them.  ``run`` computes a case
with the framework's operators (``own``) or in plain torch; ``exact`` computes it in 64 bits.
"""

import functools
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
MOST_QKV = 16384 * 48 * 128      # elements of the largest packed query/key/value rows
MOST_DROPOUT = 16384 * 4096
MOST_LOGITS = 4096 * 128256


def listed():
    return [
        # one short sequence through an 8B-class block: a call whose launch is most of its time
        dict(name="heads_fwd_short", op="heads_fwd", batch=1, seq=64, heads=32, kv_heads=8, dim=128, theta=500000.0,
             dtype="bf16"),
        # four sequences of 4096 tokens through the same block
        dict(name="heads_fwd_8b", op="heads_fwd", batch=4, seq=4096, heads=32, kv_heads=8, dim=128, theta=500000.0,
             dtype="bf16"),
        # backward of the same
        dict(name="heads_bwd_8b", op="heads_bwd", batch=4, seq=4096, heads=32, kv_heads=8, dim=128, theta=500000.0,
             dtype="bf16"),
        # ragged length, an odd head count and a head dimension that is no power of two, in 32 bits
        dict(name="heads_bwd_odd", op="heads_bwd", batch=3, seq=1021, heads=9, kv_heads=3, dim=80, theta=10000.0,
             dtype="fp32"),
        # a tiny transformer's residual branch, forward and gradient: latency
        dict(name="dropout_tiny", op="dropout", rows=512, cols=128, residual=True, p=0.1, dtype="fp32"),
        # residual branch of an 8B-class block, forward and gradient
        dict(name="dropout_8b", op="dropout", rows=16384, cols=4096, residual=True, p=0.1, dtype="bf16"),
        # embedding output of odd shape, no residual
        dict(name="dropout_odd", op="dropout", rows=4099, cols=1283, residual=False, p=0.25, dtype="fp16"),
        # log probabilities of a frozen reference model's tokens, GPT vocabulary
        dict(name="logprobs_gpt", op="logprobs", rows=4096, vocab=50257, dtype="bf16"),
        # preference step on four pairs, GPT vocabulary: log probabilities, loss, gradient of the logits
        dict(name="preference_gpt", op="preference", pairs=4, seq=1024, vocab=50257, form="sigmoid", dtype="bf16"),
        # the same on the tiny transformer's vocabulary, squared form
        dict(name="preference_tiny", op="preference", pairs=2, seq=61, vocab=1024, form="squared", dtype="fp32"),
        # clipped policy loss over 4096 sampled tokens, 8B-class vocabulary, logits to their gradient
        dict(name="policy_8b", op="policy", rows=4096, vocab=128256, dtype="bf16"),
        # a short ragged chunk of an odd vocabulary
        dict(name="policy_odd", op="policy", rows=333, vocab=5003, dtype="fp16"),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["heads_fwd", "heads_bwd", "dropout", "logprobs", "preference", "policy"])
    case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    if op in ("heads_fwd", "heads_bwd"):
        kv = rng.choice([1, 2, 3, 4, 8])
        case.update(heads=kv * rng.choice([1, 3, 4, 8]), kv_heads=kv, dim=rng.choice([32, 64, 80, 96, 128, 256]),
                    theta=rng.choice([10000.0, 500000.0]))
        width = (case["heads"] + 2 * kv) * case["dim"] * BYTES[case["dtype"]] // 2
        tokens = _log_uniform(rng, 1, max(1, min(32768, MOST_QKV // width)))
        batch = rng.choice([b for b in (1, 2, 3, 5) if b <= tokens])
        case.update(batch=batch, seq=tokens // batch)
    elif op == "dropout":
        cols = _log_uniform(rng, 8, 8192)
        case.update(cols=cols, rows=_log_uniform(rng, 1, MOST_DROPOUT * 2 // BYTES[case["dtype"]] // cols),
                    residual=rng.random() < 0.6, p=rng.choice([0.0, 0.05, 0.1, 0.25, 0.5]))
    else:
        vocab = _log_uniform(rng, 32, 131072)
        rows = _log_uniform(rng, 2, min(16384, MOST_LOGITS * 2 // BYTES[case["dtype"]] // vocab))
        case["vocab"] = vocab
        if op == "preference":
            pairs = rng.choice([n for n in (1, 2, 4) if 2 * n <= rows])
            case.update(pairs=pairs, seq=rows // (2 * pairs), form=rng.choice(["sigmoid", "squared"]))
        else:
            case["rows"] = rows
    return case


# ------------------------------------------------------------------ inputs

def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _logits(g, rows, vocab, dtype):
    """Logits as a vocabulary projection leaves them: rows padded to a multiple of 8 columns, the
    sampled token a few units above the rest."""
    width = (vocab + 7) // 8 * 8
    logits = (_normal(g, rows, width) * 2.0).to(dtype)
    targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    logits[torch.arange(rows, device="cuda"), targets] += 4.0
    return logits, targets


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    s = dict(case=case)
    if op in ("heads_fwd", "heads_bwd"):
        T, n, dim = case["batch"] * case["seq"], case["heads"] + case["kv_heads"], case["dim"]
        s["qkv"] = _normal(g, T, (n + case["kv_heads"]) * dim).to(dtype)
        s["gains"] = [(1.0 + 0.1 * _normal(g, dim)).to(dtype) for _ in range(2)]
        if op == "heads_bwd":  # the attention's gradients, packed as the projection's output is
            s["dqkv"] = (0.1 * _normal(g, T, (n + case["kv_heads"]) * dim)).to(dtype)
    elif op == "dropout":
        shape = (case["rows"], case["cols"])
        s["x"] = _normal(g, *shape).to(dtype)
        if case["residual"]:
            s["residual"], s["dy"] = _normal(g, *shape).to(dtype), (0.1 * _normal(g, *shape)).to(dtype)
        s["seed"], s["offset"] = 1234 + seed, (seed % 2 ** 30 << 33) + 7
    else:
        rows = 2 * case["pairs"] * case["seq"] if op == "preference" else case["rows"]
        V = case["vocab"]
        s["logits"], s["targets"] = _logits(g, rows, V, dtype)
        if op == "logprobs":
            return s
        logps = torch.empty(rows, device="cuda")
        for a in range(0, rows, 1024):
            lp = torch.log_softmax(s["logits"][a:a + 1024, :V].float(), -1)
            logps[a:a + 1024] = lp.gather(1, s["targets"][a:a + 1024, None])[:, 0]
        s["ref"] = logps + 0.1 * _normal(g, rows)
        if op == "preference":  # answers of ragged length behind a prompt; the rest is masked
            S, n = case["seq"], 2 * case["pairs"]
            at = torch.arange(S, device="cuda")[None]
            first = torch.randint(0, S // 4 + 1, (n, 1), generator=g, device="cuda")
            last = torch.randint(S // 2, S + 1, (n, 1), generator=g, device="cuda")
            s["mask"] = (at >= first) & (at < last.clamp(min=1))
            s["ref"] = s["ref"].view(n, S)
        else:
            # log ratios of a policy some updates old, none next to a border of the clip, where the
            # gradient jumps and neither side of a rounding is wrong
            r = 0.15 * _normal(g, rows)
            for border in (math.log(0.8), math.log(1.2)):
                r = torch.where((r - border).abs() < 1e-3, r + 4e-3, r)
            s["old"] = logps - r
            s["advantages"] = _normal(g, rows)
            kept = torch.rand(rows, generator=g, device="cuda") < 0.9  # the others are prompt or padding
            s["weights"] = kept.float() / kept.sum().clamp(min=1)
    return s


# ------------------------------------------------------------------ plain form

def _turn(case, device):
    """Cosine and sine of each position's angles; the angles in 64 bits."""
    T, half = case["batch"] * case["seq"], case["dim"] // 2
    inverse = case["theta"] ** (torch.arange(half, device=device, dtype=torch.float64) * (-2.0 / case["dim"]))
    angle = (torch.arange(T, device=device) % case["seq"]).double()[:, None] * inverse
    return angle.cos().float()[:, None], angle.sin().float()[:, None]


def _plain_heads(s):
    c = s["case"]
    T, n, half = s["qkv"].shape[0], c["heads"] + c["kv_heads"], c["dim"] // 2
    x = s["qkv"][:, :n * c["dim"]].float().view(T, n, c["dim"])
    gain = torch.cat([s["gains"][0].float().expand(c["heads"], -1), s["gains"][1].float().expand(c["kv_heads"], -1)])
    cos, sin = _turn(c, x.device)
    r = (x.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    if c["op"] == "heads_fwd":
        u = x * r * gain
        a, b = u[..., :half], u[..., half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(s["qkv"].dtype).view(T, -1)
    dy = s["dqkv"][:, :n * c["dim"]].float().view(T, n, c["dim"])
    a, b = dy[..., :half], dy[..., half:]
    du = torch.cat([a * cos + b * sin, b * cos - a * sin], -1)
    xhat = x * r
    dgain = (du * xhat).sum(0)
    w = du * gain
    dx = r * (w - xhat * (w * xhat).mean(-1, keepdim=True))
    return {"dx": dx.to(s["qkv"].dtype).view(T, -1), "dq_gain": dgain[:c["heads"]].sum(0),
            "dk_gain": dgain[c["heads"]:].sum(0)}


LOW = 0xFFFFFFFF


def _multiply(a, m):
    """High and low words of the product of 32-bit values held in 64-bit integers."""
    return (a * (m >> 16) + (a * (m & 0xFFFF) >> 16)) >> 16, (a * m) & LOW


def _round(state, i, seed):
    """One round of Philox4x32 (Salmon, Moraes, Dror, Shaw 2011)."""
    c0, c1, c2, c3 = state
    k0, k1 = (seed + i * 0x9E3779B9) & LOW, ((seed >> 32) + i * 0xBB67AE85) & LOW
    h0, l0 = _multiply(c0, 0xD2511F53)
    h1, l1 = _multiply(c2, 0xCD9E8D57)
    return h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0


def _plain_keep(shape, p, seed, offset):
    """The kept elements: 16 random bits for each, of generator output (element // 8, offset) under the key ``seed``."""
    n = math.prod(shape)
    group = torch.arange((n + 7) // 8, device="cuda")
    start = (group & LOW, group >> 32, torch.full_like(group, offset & LOW), torch.full_like(group, offset >> 32))
    words = torch.stack(functools.reduce(lambda c, i: _round(c, i, seed), range(10), start), -1)
    bits = torch.stack([words & 0xFFFF, words >> 16], -1).view(-1)[:n]
    return (bits >= round(p * 65536)).view(shape)


def _plain_dropout(s):
    x, p = s["x"], s["case"]["p"]
    keep, scale = _plain_keep(x.shape, p, s["seed"], s["offset"]), 65536 / (65536 - round(p * 65536))
    y = torch.where(keep, x.float() * scale, 0.0)
    if not s["case"]["residual"]:
        return {"y": y.to(x.dtype)}
    dx = torch.where(keep, s["dy"].float() * scale, 0.0)
    return {"y": (y + s["residual"].float()).to(x.dtype), "dx": dx.to(x.dtype)}


def _plain_logprobs(s):
    x = s["logits"][:, :s["case"]["vocab"]].float()
    top = x.amax(-1, keepdim=True)
    e = (x - top).exp()
    total = e.sum(-1, keepdim=True)
    at = s["targets"][:, None]
    logps = (x.gather(1, at) - top - total.log())[:, 0]
    return e, total, top, logps


def _plain_dlogits(s, e, total, dlogps):
    d = e.mul_(-(dlogps[:, None] / total))
    d.scatter_add_(1, s["targets"][:, None], dlogps[:, None])
    return d.to(s["logits"].dtype)


def _plain_preference(s):
    c = s["case"]
    e, total, _, logps = _plain_logprobs(s)
    ratio = torch.where(s["mask"], logps.view(s["ref"].shape).double() - s["ref"], 0.0)
    r = ratio.sum(-1)
    if c["form"] == "sigmoid":
        h = 0.1 * (r[0::2] - r[1::2])
        loss = (1 + (-h.abs()).exp()).log() + (-h).clamp(min=0)
        slope = -0.1 / (1 + h.exp())
        up = torch.stack([slope, -slope], -1).view(-1)
    else:
        count = s["mask"].sum(-1).clamp(min=1)
        mean = r / count
        gap = mean[0::2] - mean[1::2] - 1 / (2 * 0.1)
        loss = gap.square()
        up = torch.stack([2 * gap, -2 * gap], -1).view(-1) / count
    dlogps = torch.where(s["mask"], (up / c["pairs"])[:, None], 0.0).float()
    return {"loss": loss.float(), "rewards": (0.1 * r).float(), "logps": logps,
            "dlogits": _plain_dlogits(s, e, total, dlogps.view(-1))}


def _plain_policy(s):
    e, total, _, logps = _plain_logprobs(s)
    A, w = s["advantages"], s["weights"]
    ratio = (logps - s["old"]).exp()
    free, bound = -A * ratio, -A * ratio.clamp(0.8, 1.2)
    d = s["ref"] - logps
    loss = w * (torch.maximum(free, bound) + 0.05 * (d.expm1() - d))
    dlogps = w * (torch.where(free >= bound, free, 0.0) - 0.05 * d.expm1())
    return {"loss": loss, "logps": logps, "dlogits": _plain_dlogits(s, e, total, dlogps)}


# ------------------------------------------------------------------ the framework's operators

def _own_heads(s):
    from meshtrain_b200 import ops

    c = s["case"]
    shape = (c["seq"], c["heads"], c["kv_heads"], c["dim"], c["theta"])
    if c["op"] == "heads_fwd":
        return ops.qk_norm_rope(s["qkv"], *s["gains"], *shape)
    dgains = torch.zeros(2, c["dim"], device="cuda")
    dx = ops.qk_norm_rope_bwd(s["dqkv"], s["qkv"], *s["gains"], *shape, dgains[0], dgains[1])
    return {"dx": dx, "dq_gain": dgains[0], "dk_gain": dgains[1]}


def _own_dropout(s):
    from meshtrain_b200 import ops

    args = (s["case"]["p"], s["seed"], s["offset"])
    if not s["case"]["residual"]:
        return {"y": ops.dropout(s["x"], *args)}
    return {"y": ops.dropout(s["x"], *args, residual=s["residual"]), "dx": ops.dropout(s["dy"], *args)}


def _own_loss(s):
    from meshtrain_b200 import ops

    c = s["case"]
    V = c["vocab"]
    if c["op"] == "logprobs":
        logps, stats = ops.token_logprobs(s["logits"], V, s["targets"])
        return {"logps": logps, "stats": stats}
    if c["op"] == "policy":
        loss, logps, dlogits = ops.policy_loss_chunk(
            s["logits"], V, s["targets"], s["old"], s["advantages"], s["weights"], ref_logps=s["ref"], clip_low=0.2,
            clip_high=0.2, kl_coef=0.05)
        return {"loss": loss, "logps": logps, "dlogits": dlogits[:, :V]}
    logps, stats = ops.token_logprobs(s["logits"], V, s["targets"])
    loss, rewards, dlogps = ops.preference_loss(logps.view(s["ref"].shape), s["ref"], s["mask"], beta=0.1,
                                                form=c["form"], grad_scale=1.0 / c["pairs"])
    dlogits = ops.token_logprobs_bwd(s["logits"], V, s["targets"], stats, dlogps)
    return {"loss": loss, "rewards": rewards, "logps": logps, "dlogits": dlogits[:, :V]}


def run(state):
    op = state["case"]["op"]
    if own:
        return (_own_heads if op.startswith("heads") else _own_dropout if op == "dropout" else _own_loss)(state)
    if op == "logprobs":
        _, total, top, logps = _plain_logprobs(state)
        return {"logps": logps, "stats": torch.cat([top, total], 1)}
    return {"heads_fwd": _plain_heads, "heads_bwd": _plain_heads, "dropout": _plain_dropout,
            "preference": _plain_preference, "policy": _plain_policy}[op](state)


def work(case):
    op, e = case["op"], BYTES[case["dtype"]]
    if op in ("heads_fwd", "heads_bwd"):
        n = case["batch"] * case["seq"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": (2 if op == "heads_fwd" else 3) * n * e, "flops": (8 if op == "heads_fwd" else 17) * n}
    if op == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": (5 if case["residual"] else 2) * n * e, "flops": (3 if case["residual"] else 1) * n}
    rows = 2 * case["pairs"] * case["seq"] if op == "preference" else case["rows"]
    n = rows * case["vocab"]
    if op == "logprobs":
        return {"bytes": n * e + 20 * rows, "flops": 4 * n}
    return {"bytes": 2 * n * e + (28 if op == "policy" else 17) * rows, "flops": 7 * n}


# ------------------------------------------------------------------ 64 bits

def _exact_heads(s):
    c = s["case"]
    H, K, n = c["heads"], c["kv_heads"], c["dim"]
    T = s["qkv"].shape[0]
    pos = torch.arange(c["seq"], dtype=torch.float64, device="cuda").repeat(c["batch"])
    freq = torch.exp(torch.arange(n // 2, dtype=torch.float64, device="cuda") * (-2.0 * math.log(c["theta"]) / n))
    spin = torch.polar(torch.ones_like(pos)[:, None].expand(T, n // 2), torch.outer(pos, freq))
    out, dgains = [], []
    for h in range(H + K):  # one head at a time, the two halves of it as one complex number
        x, g = s["qkv"][:, h * n:(h + 1) * n].double(), s["gains"][h >= H].double()
        norm = torch.sqrt(torch.sum(x * x, 1, keepdim=True) / n + 1e-5)
        if c["op"] == "heads_fwd":
            u = x / norm * g
            z = torch.complex(u[:, :n // 2], u[:, n // 2:]) * spin
            out.append(torch.cat([z.real, z.imag], 1))
            continue
        dy = s["dqkv"][:, h * n:(h + 1) * n].double()
        z = torch.complex(dy[:, :n // 2], dy[:, n // 2:]) * spin.conj()
        du = torch.cat([z.real, z.imag], 1)
        dgains.append(torch.sum(du * x / norm, 0))
        out.append(du * g / norm - x * torch.sum(du * g * x, 1, keepdim=True) / (n * norm ** 3))
    if c["op"] == "heads_fwd":
        return torch.cat(out, 1)
    return {"dx": torch.cat(out, 1), "dq_gain": torch.stack(dgains[:H]).sum(0), "dk_gain": torch.stack(dgains[H:]).sum(0)}


def _exact_dropout(s):
    rows, cols = s["x"].shape
    n, p = rows * cols, s["case"]["p"]
    c = [np.zeros((n + 7) // 8, np.uint64) for _ in range(4)]
    c[0] += np.arange(len(c[0]), dtype=np.uint64)
    c[2] += np.uint64(s["offset"] % 2 ** 32)
    c[3] += np.uint64(s["offset"] // 2 ** 32)
    key = [s["seed"] % 2 ** 32, s["seed"] // 2 ** 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        half, low = np.uint64(32), np.uint64(2 ** 32 - 1)
        c = [(b >> half) ^ c[1] ^ np.uint64(key[0]), b & low, (a >> half) ^ c[3] ^ np.uint64(key[1]), a & low]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    bits = np.stack([w.astype("<u4") for w in c], 1).view("<u2").reshape(-1)[:n]
    cut = round(p * 2 ** 16)
    keep = torch.from_numpy(bits >= cut).cuda().view(rows, cols)
    scale = 1.0 / (1.0 - cut / 2 ** 16)
    y = s["x"].double().masked_fill(~keep, 0.0) * scale
    if not s["case"]["residual"]:
        return {"y": y}
    return {"y": s["residual"].double() + y, "dx": s["dy"].double().masked_fill(~keep, 0.0) * scale}


def _exact_loss(s):
    c = s["case"]
    op, V, rows = c["op"], c["vocab"], s["targets"].shape[0]
    block = max(1, (1 << 26) // V)
    logps, lse = (torch.empty(rows, dtype=torch.float64, device="cuda") for _ in range(2))
    for a in range(0, rows, block):
        x = s["logits"][a:a + block, :V].double()
        lse[a:a + block] = torch.logsumexp(x, -1)
        logps[a:a + block] = x[torch.arange(len(x)), s["targets"][a:a + block]] - lse[a:a + block]
    if op == "logprobs":
        top = s["logits"][:, :V].amax(1).double()
        return {"logps": logps, "stats": torch.stack([top, torch.exp(lse - top)], 1)}
    if op == "policy":
        A, w, k = s["advantages"].double(), s["weights"].double(), 0.05
        ratio, back = torch.exp(logps - s["old"].double()), torch.exp(s["ref"].double() - logps)
        inside = torch.where(A >= 0, ratio <= 1.2, ratio >= 0.8)
        gained = torch.where(A >= 0, A * ratio.clamp(max=1.2), A * ratio.clamp(min=0.8))
        out = {"loss": w * (k * (back - 1 - s["ref"].double() + logps) - gained), "logps": logps}
        dlogps = w * (k * (1 - back) - torch.where(inside, A * ratio, 0.0))
    else:
        m = s["mask"].double()
        r = (m * (logps.view(m.shape) - s["ref"].double())).sum(1)
        sign = torch.tensor([1.0, -1.0], dtype=torch.float64, device="cuda").repeat(c["pairs"])
        if c["form"] == "sigmoid":
            gap = (0.1 * r * sign).view(-1, 2).sum(1)
            loss, slope = -torch.nn.functional.logsigmoid(gap), -0.1 * torch.sigmoid(-gap)
            weight = m
        else:
            weight = m / m.sum(1, keepdim=True).clamp(min=1)
            gap = (r / m.sum(1).clamp(min=1) * sign).view(-1, 2).sum(1) - 5.0
            loss, slope = gap ** 2, 2 * gap
        out = {"loss": loss, "rewards": 0.1 * r, "logps": logps}
        dlogps = (weight * (slope.repeat_interleave(2) * sign)[:, None] / c["pairs"]).view(-1)
    d = torch.empty(rows, V, device="cuda", dtype=torch.float64)
    for a in range(0, rows, block):
        p = torch.exp(s["logits"][a:a + block, :V].double() - lse[a:a + block, None])
        p[torch.arange(len(p)), s["targets"][a:a + block]] -= 1.0
        d[a:a + block] = -p * dlogps[a:a + block, None]
    return {**out, "dlogits": d}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    return (_exact_heads if op.startswith("heads") else _exact_dropout if op == "dropout" else _exact_loss)(s)
