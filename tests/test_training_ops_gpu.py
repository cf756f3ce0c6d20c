"""Kernels of the decoder-training operators against 64-bit formulas (see training_ops_oracle.py for the bounds)."""

import math

import numpy as np
import pytest
import torch

from meshtrain_b200 import ops
from tests import training_ops_oracle as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(autouse=True)
def _seed_and_status():
    torch.manual_seed(0)
    ops.set_backend("custom")
    yield
    torch.cuda.synchronize()
    assert ops.read_status(torch.cuda.current_device()) == 0, "a kernel reported a wait timeout"


def _rand(*shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, device=DEV) * scale).to(dtype)


def test_refusals():
    from tests.unit.test_training_ops import refusals

    refusals(DEV)
    g = torch.zeros(20, device=DEV)
    with pytest.raises(ValueError):  # a head dimension the kernel does not take
        ops.qk_norm_rope(torch.zeros(2, 40, device=DEV), g, g, 2, 1, 1, 20, 1e4)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(torch.zeros(2, 1024, device=DEV), *[torch.zeros(512, device=DEV)] * 2, 2, 1, 1, 512, 1e4)
    flat = torch.zeros(4 * 104 + 4, device=DEV)
    t, v = torch.zeros(4, dtype=torch.int64, device=DEV), torch.zeros(4, device=DEV)
    st = torch.zeros(4, 2, device=DEV)
    with pytest.raises(ValueError):  # rows the kernel cannot write in place: off a 16-byte boundary
        ops.token_logprobs_bwd(torch.zeros(4, 96, device=DEV), 96, t, st, v, out=flat[1:1 + 4 * 104].view(4, 104))
    with pytest.raises(ValueError):  # leading dimension 97
        ops.token_logprobs_bwd(torch.zeros(4, 96, device=DEV), 96, t, st, v, out=torch.zeros(4, 97, device=DEV))
    with pytest.raises(ValueError):
        ops.dropout(flat[:64], 0.1, 0, 0, out=flat[65:129])
    with pytest.raises(ValueError):  # more columns than 32-bit indexes take
        ops.token_logprobs(torch.zeros(1, 1, device=DEV).expand(1, (1 << 30) + 8), (1 << 30) + 1, t[:1])
    with pytest.raises(ValueError):  # another device
        ops.token_logprobs(torch.zeros(4, 96, device=DEV), 96, t.cpu())


# ------------------------------------------------------------------ head norms and rotation

HEADS = [  # rows, seq, heads, kv heads, head dim
    (1, 1, 1, 1, 16), (1, 1, 32, 8, 128), (64, 64, 32, 8, 128), (129, 43, 4, 2, 32), (77, 77, 9, 3, 80),
    (50, 25, 12, 4, 96), (33, 11, 5, 1, 256), (300, 100, 20, 20, 64), (17, 1000, 3, 0, 48), (19, 7, 0, 2, 112),
    (5000, 2500, 4, 1, 64), (40, 40, 40, 40, 16),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,seq,H,HK,hd", HEADS)
def test_qk_norm_rope(T, seq, H, HK, hd, dtype):
    qkv = _rand(T, (H + 2 * HK) * hd, dtype=dtype)
    qkv[0] = 0  # a head of zeros: eps alone under the root
    gq, gk = (1 + 0.2 * _rand(hd)).to(dtype), (1 + 0.2 * _rand(hd)).to(dtype)
    shape = (seq, H, HK, hd, 500000.0)
    y = ops.qk_norm_rope(qkv, gq, gk, *shape)
    oracle.close(y, *oracle.heads_forward(qkv, gq, gk, *shape, 1e-5), "y")
    dqk = _rand(T, (H + 2 * HK) * hd, dtype=dtype)
    want = oracle.heads_backward(dqk, qkv, gq, gk, *shape, 1e-5)
    runs = []
    for _ in range(2):
        dgq, dgk = torch.full((hd,), 0.5, device=DEV), torch.full((hd,), -0.25, device=DEV)
        dx = ops.qk_norm_rope_bwd(dqk, qkv, gq, gk, *shape, dgq, dgk)
        runs.append((dx, dgq, dgk))
    for a, b in zip(*runs):
        assert torch.equal(a, b)  # equal inputs, equal bits
    oracle.close(dx, *want[0], "dx")
    for got, base, (ref, slack) in ((dgq, 0.5, want[1]), (dgk, -0.25, want[2])):
        oracle.close(got, ref + base, slack + 2 * oracle.U * (ref.abs() + abs(base)), "gain")
    # in place over the gradient, with the value columns left as they were
    tail = dqk[:, (H + HK) * hd:].clone()
    dgq.fill_(0.5), dgk.fill_(-0.25)
    ops.qk_norm_rope_bwd(dqk, qkv, gq, gk, *shape, dgq, dgk, out=dqk)
    assert torch.equal(dqk[:, :(H + HK) * hd], dx) and torch.equal(dqk[:, (H + HK) * hd:], tail)
    assert torch.equal(dgq, runs[0][1]) and torch.equal(dgk, runs[0][2])


def test_qk_norm_rope_far_positions():
    """Position 10^6: an fp32 angle would be off by 0.06 rad."""
    seq, hd = 1_000_003, 64
    qkv = _rand(seq, hd + 16)
    g = torch.ones(hd, device=DEV)
    y = ops.qk_norm_rope(qkv, g, g, seq, 1, 0, hd, 10000.0)
    rows = torch.arange(seq - 64, seq)
    x = qkv[rows][:, :hd].cpu().double()
    u = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5)
    ang = torch.outer(rows.double(), torch.exp(torch.arange(32).double() * (-2 * math.log(10000.0) / hd)))
    a, b = u[:, :32], u[:, 32:]
    want = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], 1)
    oracle.close(y[rows], want, 32 * oracle.U * torch.cat([a.abs() + b.abs()] * 2, 1))


def test_qk_norm_rope_past_2_to_the_31_elements():
    T, H, HK, hd = 360_000, 32, 8, 128
    qkv = torch.ones(T, (H + 2 * HK) * hd, dtype=torch.bfloat16, device=DEV)
    qkv[-3:] = _rand(3, qkv.shape[1], dtype=torch.bfloat16)
    g = _rand(hd, dtype=torch.bfloat16)
    shape = (3, H, HK, hd, 10000.0)  # 360000 is a multiple of 3: the last rows have positions 0, 1, 2
    y = ops.qk_norm_rope(qkv, g, g, *shape)
    oracle.close(y[-3:], *oracle.heads_forward(qkv[-3:], g, g, *shape, 1e-5))
    del y
    dy = torch.zeros_like(qkv)
    dy[-3:] = _rand(3, qkv.shape[1], dtype=torch.bfloat16)
    tail = dy[-3:].clone()
    dg = torch.zeros(2, hd, device=DEV)
    ops.qk_norm_rope_bwd(dy, qkv, g, g, *shape, dg[0], dg[1], out=dy)
    want = oracle.heads_backward(tail, qkv[-3:], g, g, *shape, 1e-5)
    oracle.close(dy[-3:, :(H + HK) * hd], *want[0], "dx")
    oracle.close(dg[0], *want[1], "dq_gain")  # the other rows' gradients are zero
    oracle.close(dg[1], *want[2], "dk_gain")
    assert dy[:-3, :(H + HK) * hd].count_nonzero() == 0


def test_qk_norm_rope_one_gradient_for_both_gains():
    """A gain that query and key heads share has one gradient buffer; buffers may also overlap in part."""
    T, seq, H, HK, hd = 400, 50, 5, 2, 64
    x, dy, g = _rand(T, (H + HK) * hd), _rand(T, (H + HK) * hd), _rand(hd)
    shape = (seq, H, HK, hd, 10000.0)
    dq, dk = torch.zeros(2, hd, device=DEV)
    dx = ops.qk_norm_rope_bwd(dy, x, g, g, *shape, dq, dk)
    for shift in (0, 8, hd - 1, hd):
        both = torch.zeros(2 * hd, device=DEV)
        got = ops.qk_norm_rope_bwd(dy, x, g, g, *shape, both[:hd], both[shift:shift + hd])
        want = torch.zeros_like(both)
        want[:hd] += dq
        want[shift:shift + hd] += dk
        assert torch.equal(got, dx) and torch.equal(both, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_qk_norm_rope_layouts(dtype):
    """Rows on no 16-byte boundary, a wide row stride, a transposed layout and gains inside a larger buffer."""
    T, seq, H, HK, hd = 21, 7, 3, 1, 32
    cols = (H + HK) * hd
    base = _rand(T, cols, dtype=dtype)
    gains = _rand(2 * hd + 1, dtype=dtype)
    gq, gk = gains[1:hd + 1], gains[hd + 1:]
    shape = (seq, H, HK, hd, 10000.0)
    want = ops.qk_norm_rope(base, gq.clone(), gk.clone(), *shape)
    wide = torch.zeros(T, cols + 24, dtype=dtype, device=DEV)
    wide[:, :cols] = base
    odd = torch.zeros(T, cols + 3, dtype=dtype, device=DEV)
    odd[:, 3:] = base
    for x in (wide, odd[:, 3:], base.t().contiguous().t()):
        assert torch.equal(ops.qk_norm_rope(x, gq, gk, *shape), want)
    out = torch.full((T, cols + 8), 7.0, dtype=dtype, device=DEV)
    ops.qk_norm_rope(base, gq, gk, *shape, out=out)
    assert torch.equal(out[:, :cols], want) and out[:, cols:].eq(7).all()
    empty = ops.qk_norm_rope(base[:0], gq, gk, *shape)
    assert empty.shape == (0, cols)
    dg = torch.ones(2, hd, device=DEV)
    assert ops.qk_norm_rope_bwd(base[:0], base[:0], gq, gk, *shape, dg[0], dg[1]).shape == (0, cols)
    assert dg.eq(1).all()


# ------------------------------------------------------------------ dropout

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (64, 128), (1021, 1283), (0, 4), (3, 5, 11)])
def test_dropout(shape, dtype):
    x, res = _rand(*shape, dtype=dtype), _rand(*shape, dtype=dtype)
    for p, seed, offset in ((0.0, 0, 0), (0.1, 11, 12), (0.5, (1 << 64) - 1, (1 << 64) - 1), (0.9999, 1 << 40, 1 << 32)):
        y, slack, keep = oracle.dropout(x, p, seed, offset)
        got = ops.dropout(x, p, seed, offset)
        oracle.close(got, y, slack, "y")
        assert got[~keep.to(DEV)].eq(0).all()
        y, slack, _ = oracle.dropout(x, p, seed, offset, res)
        oracle.close(ops.dropout(x, p, seed, offset, residual=res), y, slack, "y + residual")
    want = ops.dropout(x, 0.3, 5, 6, residual=res)
    for target in ("x", "residual"):  # in place over either input
        a, b = x.clone(), res.clone()
        o = a if target == "x" else b
        assert ops.dropout(a, 0.3, 5, 6, residual=b, out=o) is o and torch.equal(o, want)
    with ops.use_backend("torch"):
        oracle.close(ops.dropout(x, 0.3, 5, 6), *oracle.dropout(x, 0.3, 5, 6)[:2], "torch backend")


def test_dropout_layouts_and_garbage():
    x = _rand(40, 24)
    want = ops.dropout(x, 0.4, 1, 2)
    buf = torch.zeros(40 * 24 + 1, device=DEV)
    buf[1:] = x.reshape(-1)
    assert torch.equal(ops.dropout(buf[1:].view(40, 24), 0.4, 1, 2), want)  # off a 16-byte boundary
    assert torch.equal(ops.dropout(x.t().contiguous().t(), 0.4, 1, 2), want)  # the mask follows the logical index
    bad = torch.full((4000,), math.nan, device=DEV)
    y = ops.dropout(bad, 0.5, 1, 2, residual=torch.ones(4000, device=DEV))
    keep = oracle.dropout(bad, 0.5, 1, 2)[2].to(DEV)
    assert y[~keep].eq(1).all() and y[keep].isnan().all()


def test_dropout_across_the_high_word_of_the_counter():
    """Groups 2^32 and on (elements 2^35 and on) count in the counter's second word."""
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 69 GB of device memory")
    n = (1 << 35) + 4099
    x = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    ops.dropout(x, 0.5, 3, 4, out=x)
    lo, low, half = (1 << 35) - 4096, np.uint64(0xFFFFFFFF), np.uint64(32)
    g = np.arange(lo // 8, (n + 7) // 8, dtype=np.uint64)
    assert g[0] >> half == 0 and g[-1] >> half == 1
    c, k = [g & low, g >> half, np.full_like(g, 4), np.zeros_like(g)], [3, 0]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> half) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    bits = np.stack([w.astype("<u4") for w in c], 1).view("<u2").reshape(-1)[:n - lo]
    assert torch.equal(x[lo:].cpu() != 0, torch.from_numpy(bits >= 32768))
    del x
    torch.cuda.empty_cache()


def test_dropout_more_than_2_to_the_32_elements():
    n = (1 << 32) + 4099
    x = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    y = ops.dropout(x, 0.5, 3, 4, out=x)
    lo = (1 << 32) - 4096  # compare the groups across the border: their counters' high word changes at 2^35
    g = torch.arange(lo // 8, (n + 7) // 8)
    import numpy as np

    c = [np.asarray(g & 0xFFFFFFFF, dtype=np.uint64), np.asarray(g >> 32, dtype=np.uint64),
         np.full(len(g), 4, np.uint64), np.zeros(len(g), np.uint64)]
    k = [3, 0]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & np.uint64(0xFFFFFFFF),
             (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & np.uint64(0xFFFFFFFF)]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    bits = np.stack([w.astype("<u4") for w in c], 1).view("<u2").reshape(-1)[:n - lo]
    assert torch.equal(y[lo:].cpu() != 0, torch.from_numpy(bits >= 32768))


def test_dropout_captured_graph_draws_a_new_mask_each_replay():
    x = _rand(512, 64, dtype=torch.bfloat16)
    step = torch.zeros(1, dtype=torch.int64, device=DEV)
    out = torch.empty_like(x)
    ops.dropout(x, 0.5, 9, step, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.dropout(x, 0.5, 9, step, out=out)
    for s in (0, 5, 1 << 33):
        step.fill_(s)
        graph.replay()
        assert torch.equal(out, ops.dropout(x, 0.5, 9, s))


# ------------------------------------------------------------------ losses over logits

# Few rows of every width: a warp, a block, a cluster of 2, 4 or 8 blocks per row, and past what a cluster holds;
# then many rows: 4 warps per row, and each block size of the stream kernels, several rows to a block.
LOGITS = [(1, 1), (2, 7), (5, 8), (33, 100), (64, 1024), (100, 3001), (37, 5003), (9, 16391), (16, 50257), (3, 128256),
          (2, 300007), (400, 1025), (1500, 4096), (3100, 4099), (2000, 12345), (1100, 30011), (700, 60001), (400, 131075)]


def _logits(T, V, dtype):
    width = (V + 7) // 8 * 8
    x = _rand(T, width, dtype=dtype, scale=3.0)
    x[:, V:] = math.nan  # padding columns are never looked at
    return x, torch.randint(0, V, (T,), device=DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V", LOGITS)
def test_token_logprobs(T, V, dtype):
    x, t = _logits(T, V, dtype)
    if T > 2:
        t[1], t[2] = -100, V
    lp, stats = ops.token_logprobs(x, V, t)
    want, wstats, _, _ = oracle.logprobs(x, V, t)
    oracle.close(lp, *want, "logp")
    oracle.close(stats, *wstats, "stats")
    up = _rand(T)
    if T > 3:
        up[3] = 0
    d = ops.token_logprobs_bwd(x, V, t, stats, up)
    assert d.shape == (T, V)
    oracle.close(d, *oracle.dlogits(x, V, t, up), "dlogits")
    pad = x[:, V:].clone()
    out = ops.token_logprobs_bwd(x, V, t, stats, up, out=x)
    assert torch.equal(out, d) and out.data_ptr() == x.data_ptr() and x[:, V:].isnan().all() and pad.isnan().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,copies", [(13, 1), (64, 1), (5003, 1), (50257, 1), (128256, 1), (2051, 40), (5003, 200),
                                      (29000, 80), (61003, 50), (120007, 40)])
def test_rows_of_infinities_and_nan(V, copies, dtype):
    """``copies`` of eight rows: the last eight, which blocks with several rows reach, are looked at."""
    x = _rand(8, (V + 7) // 8 * 8, dtype=dtype, scale=2.0)
    low = torch.finfo(dtype).min
    x[0] = -math.inf                 # nothing left
    x[1, 3:] = -math.inf             # a masked vocabulary
    x[2, 4] = math.nan
    x[3, V - 1] = math.inf
    x[4, 1:] = low                   # masked by the type's lowest value
    x[5] = low                       # every logit the lowest value: a uniform row
    x[6, :V - 1] = -math.inf         # one value left, the last
    t = torch.tensor([2, 1, 0, 0, 0, 5, V - 1, 7], device=DEV)
    many = lambda v: v.repeat(copies, *[1] * (v.dim() - 1))  # noqa: E731
    last = lambda v: v[-8:]  # noqa: E731
    xs, ts = many(x), many(t)
    lps, all_stats = ops.token_logprobs(xs, V, ts)
    lp, stats = last(lps), last(all_stats)
    assert torch.equal(lps.nan_to_num(7.0), many(lp).nan_to_num(7.0))
    (want, slack), (wstats, sslack), _, _ = oracle.logprobs(x, V, t)
    fine = [1, 4, 5, 6, 7]
    oracle.close(lp[fine], want[fine], slack[fine], "logp")
    oracle.close(stats[fine], wstats[fine], sslack[fine], "stats")
    assert lp[0] == -math.inf and stats[0].tolist() == [-math.inf, 0.0]
    assert lp[2].isnan() and stats[2, 1].isnan() and lp[3].isnan()
    up = torch.ones(8, device=DEV)
    d = last(ops.token_logprobs_bwd(xs, V, ts, all_stats, many(up)))
    assert d[0].eq(0).all() and d[1, 3:].eq(0).all() and d[2].isnan().all()
    oracle.close(d[fine], *[v[fine] for v in oracle.dlogits(x, V, t, up)], "dlogits")
    assert ops.token_logprobs_bwd(x, V, t, stats, torch.zeros(8, device=DEV)).eq(0).all()
    # the one-pass loss on the same rows
    z, one = torch.zeros(8, device=DEV), torch.ones(8, device=DEV)
    w = one.clone()
    w[[0, 2, 3]] = 0
    old = torch.where(w > 0, lp, math.nan)
    loss, lp2, d = map(last, ops.policy_loss_chunk(xs, V, ts, many(old), many(one), many(w)))
    assert loss[[0, 2, 3]].eq(0).all() and d[[0, 2, 3]].eq(0).all() and lp2[0] == -math.inf
    assert torch.allclose(loss[fine], -one[fine], atol=1e-5) and d[fine].isfinite().all()
    loss, _, d = ops.policy_loss_chunk(xs, V, ts, many(z), many(one), many(z))
    assert loss.eq(0).all() and d.eq(0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V", LOGITS + [(700, 333)])
def test_policy_loss_chunk(T, V, dtype):
    from tests.unit.test_training_ops import _policy_inputs

    x, t = _logits(T, V, dtype)
    old, ref, adv, w = _policy_inputs(x, V, t.cpu(), DEV)
    if T > 2:
        t[2] = -1
    kw = dict(clip_low=0.2, clip_high=0.3, kl_coef=0.05, grad_scale=0.5)
    got = ops.policy_loss_chunk(x, V, t, old, adv, w, ref_logps=ref, **kw)
    want = oracle.policy(x, V, t, old, adv, w, ref, 0.2, 0.3, 0.05, 0.5)
    for g, (r, s), n in zip(got, want, ("loss", "logp", "dlogits")):
        oracle.close(g, r, s, n)
    again = ops.policy_loss_chunk(x, V, t, old, adv, w, ref_logps=ref, out=x, **kw)
    for a, b in zip(got, again):
        assert torch.equal(a, b)
    assert again[2].data_ptr() == x.data_ptr() and x[:, V:].isnan().all()


@pytest.mark.parametrize("V", [9, 2051, 50257])
def test_policy_loss_at_probabilities_of_zero(V):
    """An old probability of 0 (or a ratio past the type's range) beside an advantage of 0, and a KL term of a
    token the policy gives probability 0: the formula's limits 0 and infinity, not NaN."""
    x = torch.zeros(4, V, device=DEV)
    x[2, 1] = -math.inf
    t = torch.ones(4, dtype=torch.int64, device=DEV)
    lp = -math.log(V)
    old = torch.tensor([-math.inf, -200.0, 0.0, lp], device=DEV)
    adv = torch.tensor([0.0, 0.0, 1.0, 1.0], device=DEV)
    loss, _, d = ops.policy_loss_chunk(x, V, t, old, adv)
    assert loss[:2].tolist() == [0.0, 0.0] and d[:2].eq(0).all()
    assert loss[2] == 0 and d[2].eq(0).all() and d[3].isfinite().all() and d[3, 1] < 0
    loss, lps, d = ops.policy_loss_chunk(x, V, t, old, adv, ref_logps=torch.full_like(old, lp), kl_coef=0.5)
    assert lps[2] == -math.inf and loss[2] == math.inf and loss[[0, 1, 3]].isfinite().all()


def test_policy_without_weights_or_reference():
    x, t = _logits(20, 999, torch.bfloat16)
    old, adv = -7 + _rand(20) * 0.1, _rand(20)
    got = ops.policy_loss_chunk(x, 999, t, old, adv)
    want = oracle.policy(x, 999, t, old, adv, None, None, 0.2, 0.2, 0.0, 1.0)
    for g, (r, s), n in zip(got, want, ("loss", "logp", "dlogits")):
        oracle.close(g, r, s, n)


@pytest.mark.parametrize("dtype", DTYPES)
def test_logits_layouts(dtype):
    """Unpadded odd rows, a shifted view, a row slice and broadcast per-row inputs."""
    T, V = 12, 517
    x = _rand(T, V, dtype=dtype)
    t = torch.randint(0, V, (T,), device=DEV)
    padded = torch.zeros(T, 528, dtype=dtype, device=DEV)
    padded[:, :V] = x
    lp, stats = ops.token_logprobs(padded, V, t)
    shifted = torch.zeros(T, V + 6, dtype=dtype, device=DEV)
    shifted[:, 3:3 + V] = x
    up = torch.full((1,), 0.25, device=DEV).expand(T)
    d = ops.token_logprobs_bwd(padded, V, t, stats, up)
    for y in (x, shifted[:, 3:3 + V], x.t().contiguous().t()):
        lp2, stats2 = ops.token_logprobs(y, V, t)
        assert torch.equal(lp, lp2) and torch.equal(stats, stats2)
        assert torch.equal(ops.token_logprobs_bwd(y, V, t, stats, up), d)
    stacked = torch.stack([t, t], 1)[:, 0]  # strided targets
    assert torch.equal(ops.token_logprobs(padded[::2], V, stacked[::2])[0], lp[::2])
    assert ops.token_logprobs(x[:0], V, t[:0])[0].shape == (0,)
    assert ops.token_logprobs_bwd(x[:0], V, t[:0], stats[:0], lp[:0]).shape == (0, V)


def test_logits_past_2_to_the_31_elements():
    T, V = 16500, 131072
    x = torch.zeros(T, V, dtype=torch.bfloat16, device=DEV)
    x[-3:] = _rand(3, V, dtype=torch.bfloat16)
    t = torch.randint(0, V, (T,), device=DEV)
    lp, stats = ops.token_logprobs(x, V, t)
    want, _, _, _ = oracle.logprobs(x[-3:], V, t[-3:])
    oracle.close(lp[-3:], *want)
    assert (lp[:-3] + math.log(V)).abs().max() < 1e-5
    want = oracle.policy(x[-3:], V, t[-3:], lp[-3:], torch.ones(3), None, None, 0.2, 0.2, 0.0, 1.0)
    tail = x[-3:].clone()
    ops.token_logprobs_bwd(x, V, t, stats, torch.ones(T, device=DEV), out=x)
    oracle.close(x[-3:], *oracle.dlogits(tail, V, t[-3:], torch.ones(3)))
    x[-3:] = tail
    _, _, d = ops.policy_loss_chunk(x, V, t, lp, torch.ones(T, device=DEV), out=x)
    oracle.close(d[-3:], *want[2])


@pytest.mark.parametrize("form,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.1), ("squared", 0.0)])
@pytest.mark.parametrize("P,S", [(1, 1), (2, 7), (3, 300), (5, 4097), (20, 17001), (1, 200_003), (200, 33), (0, 4), (2, 0)])
def test_preference_loss(P, S, form, smoothing):
    lp, ref = -5 * torch.rand(2 * P, S, device=DEV), -5 * torch.rand(2 * P, S, device=DEV)
    mask = torch.rand(2 * P, S, device=DEV) < 0.7
    if P > 1:
        mask[1] = False
    lp[~mask] = math.nan
    beta = 0.3 / max(1.0, S) ** 0.5
    runs = [ops.preference_loss(lp, ref, mask, beta, form=form, label_smoothing=smoothing, grad_scale=0.5)
            for _ in range(2)]
    want = oracle.preference(lp, ref, mask, beta, form, smoothing, 0.5)
    for g, again, r, n in zip(*runs, want, ("loss", "reward", "dlogps")):
        assert torch.equal(g, again)
        oracle.close(g, r, 1e-10 * (1 + r.abs()), n)


def test_preference_far_margins():
    """Margins far past where an exponential overflows stay finite and exact."""
    lp = torch.tensor([[2e4], [-2e4], [-2e4], [2e4]], device=DEV)
    loss, rewards, d = ops.preference_loss(lp, torch.zeros_like(lp), torch.ones_like(lp, dtype=torch.bool), 1.0)
    assert loss.tolist() == [0.0, 4e4] and d.reshape(-1).tolist() == [0.0, 0.0, -1.0, 1.0]


@pytest.mark.parametrize("S", [1, 5000])
def test_preference_of_an_impossible_answer(S):
    """A token of probability 0 makes the margin infinite: the loss of the side that has weight 0 is left out."""
    lp = torch.zeros(4, S, device=DEV)
    lp[:, -1] = torch.tensor([-1.0, -math.inf, -math.inf, -1.0], device=DEV)
    args = (torch.zeros_like(lp), torch.ones_like(lp, dtype=torch.bool), 0.5)
    loss, rewards, d = ops.preference_loss(lp, *args)
    assert loss.tolist() == [0.0, math.inf] and d[:, 0].tolist() == [0.0, 0.0, -0.5, 0.5]
    assert torch.equal(d, d[:, :1].expand(4, S)) and rewards.tolist() == [-0.5, -math.inf, -math.inf, -0.5]
    loss, _, d = ops.preference_loss(lp, *args, label_smoothing=1.0)
    assert loss.tolist() == [math.inf, 0.0] and d[:, 0].tolist() == [0.5, -0.5, 0.0, 0.0]
    assert ops.preference_loss(lp, *args, label_smoothing=0.25)[0].tolist() == [math.inf, math.inf]


# ------------------------------------------------------------------ together

def _preference_step(x, V, t, ref, mask, out):
    lp, stats = ops.token_logprobs(x, V, t)
    loss, rewards, dlp = ops.preference_loss(lp.view(ref.shape), ref, mask, 0.1, grad_scale=1.0 / (ref.shape[0] // 2))
    return loss, rewards, ops.token_logprobs_bwd(x, V, t, stats, dlp, out=out)


def test_preference_step_on_a_side_stream_and_captured():
    P, S, V = 2, 50, 3001
    x, t = _logits(2 * P * S, V, torch.bfloat16)
    ref, mask = -8 + _rand(2 * P, S), torch.rand(2 * P, S, device=DEV) < 0.8
    want = [v.clone() for v in _preference_step(x, V, t, ref, mask, None)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _preference_step(x, V, t, ref, mask, None)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):  # two graphs of the same call, replayed in turn on two streams
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = _preference_step(x, V, t, ref, mask, None)
        graphs.append((g, res))
    for _ in range(3):
        for (g, _), s in zip(graphs, (side, torch.cuda.current_stream())):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, res in graphs:
        for a, b in zip(res, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T,V", [(30, 50257), (300, 50257), (200, 500)])  # a cluster, a stream and a warp per row
def test_policy_loss_captured_and_on_two_streams(T, V):
    x, t = _logits(T, V, torch.bfloat16)
    old, adv = -9 + _rand(T), _rand(T)
    want = [v.clone() for v in ops.policy_loss_chunk(x, V, t, old, adv)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = ops.policy_loss_chunk(x, V, t, old, adv)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        for s in streams:  # two eager calls and a replay under way at once
            with torch.cuda.stream(s):
                outs.append(ops.policy_loss_chunk(x, V, t, old, adv))
        graph.replay()
    torch.cuda.synchronize()
    for got in outs + [res]:
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_qk_norm_rope_captured_twice():
    T, H, HK, hd = 300, 8, 2, 64
    x, dy = _rand(T, (H + 2 * HK) * hd, dtype=torch.bfloat16), _rand(T, (H + HK) * hd, dtype=torch.bfloat16)
    gq, gk = _rand(hd, dtype=torch.bfloat16), _rand(hd, dtype=torch.bfloat16)
    shape = (T, H, HK, hd, 10000.0)

    def step():
        dg = torch.zeros(2, hd, device=DEV)
        return ops.qk_norm_rope(x, gq, gk, *shape), ops.qk_norm_rope_bwd(dy, x, gq, gk, *shape, dg[0], dg[1]), dg

    want = [v.clone() for v in step()]
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step()
        graphs.append((g, res))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, res in graphs:
        for a, b in zip(res, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V", LOGITS)
def test_gradients_of_infinite_coefficients(T, V, dtype):
    """An upstream gradient past the type's range, and a KL term beside a target of probability 0: every entry is
    (onehot - softmax) times the infinity, the target's own too, wherever in its row it lies."""
    x, t = _logits(T, V, dtype)
    up = torch.full((T,), math.inf, device=DEV)
    up[1::2] = -math.inf
    up[::5] = 0.0
    ref = oracle.dlogits(x, V, t, up)[0]
    lp, stats = ops.token_logprobs(x, V, t)
    oracle.close(ops.token_logprobs_bwd(x, V, t, stats, up), ref, torch.zeros_like(ref), "dlogits")
    # A < 0 and an old probability of 0: rho and the coefficient are +inf
    zero = torch.zeros(T, device=DEV)
    _, _, d = ops.policy_loss_chunk(x, V, t, zero - math.inf, zero - 1, (up != 0).float())
    ref = oracle.dlogits(x, V, t, up.abs())[0]
    oracle.close(d, ref, torch.zeros_like(ref), "policy")
    # the KL term of a target of probability 0: -inf for it
    x[torch.arange(T, device=DEV), t] = -math.inf
    _, lp, d = ops.policy_loss_chunk(x, V, t, zero, zero, ref_logps=zero - 1, kl_coef=0.1)
    ref = oracle.dlogits(x, V, t, zero - math.inf)[0]
    oracle.close(d, ref, torch.zeros_like(ref), "KL term")
    if V > 1:
        assert lp.eq(-math.inf).all() and d[torch.arange(T, device=DEV), t].eq(-math.inf).all()
