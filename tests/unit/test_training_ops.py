"""Head norms with rotation, dropout and the preference and policy losses on CPU, and what they refuse."""

import math

import pytest
import torch

from meshtrain_b200 import ops
from meshtrain_b200.models.llama import LlamaBlock
from tests import training_ops_oracle as oracle


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)


def test_dropout_known_answers():
    """The known answer published with Philox4x32-10 for counter and key zero, and far counters and keys."""
    ones = (1 << 64) - 1
    bits = oracle.keep_bits(8, 0, 0)
    words = [int(bits[2 * i]) | int(bits[2 * i + 1]) << 16 for i in range(4)]
    assert words == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    for seed, offset in ((0, 0), (ones, ones), (1 << 40, (1 << 63) + 5), (7, 1 << 32)):
        keep = ops._keep_mask((3, 37), 30000, seed, offset, "cpu").numpy()
        assert (keep.reshape(-1) == (oracle.keep_bits(111, seed, offset) >= 30000)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,seq,H,HK,hd", [(1, 1, 1, 1, 16), (7, 3, 5, 1, 2), (33, 16, 4, 2, 80), (5, 8, 2, 0, 10)])
def test_qk_norm_rope(T, seq, H, HK, hd, dtype):
    qkv = torch.randn(T, (H + 2 * HK) * hd + 3).to(dtype)
    gq, gk = (1 + 0.2 * torch.randn(hd)).to(dtype), (1 + 0.2 * torch.randn(hd)).to(dtype)
    shape = (seq, H, HK, hd, 10000.0)
    y = ops.qk_norm_rope(qkv, gq, gk, *shape)
    oracle.close(y, *oracle.heads_forward(qkv, gq, gk, *shape, 1e-5), "y")
    dqk = torch.randn(T, (H + 2 * HK) * hd).to(dtype)
    tail = dqk[:, (H + HK) * hd:].clone()
    dgq, dgk = torch.full((hd,), 0.5), torch.full((hd,), -0.25)
    want = oracle.heads_backward(dqk, qkv, gq, gk, *shape, 1e-5)
    out = ops.qk_norm_rope_bwd(dqk, qkv, gq, gk, *shape, dgq, dgk, out=dqk)
    assert out.data_ptr() == dqk.data_ptr() and torch.equal(dqk[:, (H + HK) * hd:], tail)
    oracle.close(out, *want[0], "dx")
    for got, base, (ref, slack) in ((dgq, 0.5, want[1]), (dgk, -0.25, want[2])):
        oracle.close(got, ref + base, slack + 2 * oracle.U * (ref.abs() + abs(base)), "gain")


def test_qk_norm_rope_gradient_is_the_derivative():
    T, seq, H, HK, hd = 3, 2, 2, 1, 6
    x = torch.randn(T, (H + 2 * HK) * hd, dtype=torch.float64, requires_grad=True)
    gains = [torch.randn(hd, dtype=torch.float64, requires_grad=True) for _ in range(2)]

    class Op(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, gq, gk):
            ctx.save_for_backward(x, gq, gk)
            return ops.qk_norm_rope(x, gq, gk, seq, H, HK, hd, 100.0)

        @staticmethod
        def backward(ctx, dy):
            x, gq, gk = ctx.saved_tensors
            dg = torch.zeros(2, hd, dtype=torch.float64)
            dx = torch.zeros_like(x)
            ops.qk_norm_rope_bwd(dy, x, gq, gk, seq, H, HK, hd, 100.0, dg[0], dg[1], out=dx)
            return dx, dg[0], dg[1]

    assert torch.autograd.gradcheck(Op.apply, (x, *gains))


def test_qk_norm_rope_gains_of_64_bit_rows():
    """Gradients are held in fp32 whatever the model's type; beside 64-bit rows either type takes them."""
    T, shape = 5, (3, 2, 1, 6, 100.0)
    x, dy = (torch.randn(T, 18, dtype=torch.float64) for _ in range(2))
    gq, gk = (torch.randn(6, dtype=torch.float64) for _ in range(2))
    wide, narrow = (torch.zeros(2, 6, dtype=dt) for dt in (torch.float64, torch.float32))
    dx = [ops.qk_norm_rope_bwd(dy, x, gq, gk, *shape, g[0], g[1]) for g in (wide, narrow)]
    assert torch.equal(*dx)
    oracle.close(narrow, wide, torch.zeros_like(wide))

    block = LlamaBlock(32, 4, 2, 48, qk_norm=True).double()
    h = torch.randn(2, 4, 32, dtype=torch.float64, requires_grad=True)
    block(h).backward(torch.ones_like(h))
    assert all(p.grad.isfinite().all() and p.grad.any() for p in block.parameters()) and h.grad.dtype == h.dtype


def test_qk_norm_rope_one_gradient_for_both_gains():
    x, dy, g = torch.randn(5, 18), torch.randn(5, 18), torch.randn(6)
    apart, shared = torch.zeros(2, 6), torch.zeros(6)
    ops.qk_norm_rope_bwd(dy, x, g, g, 3, 2, 1, 6, 100.0, apart[0], apart[1])
    ops.qk_norm_rope_bwd(dy, x, g, g, 3, 2, 1, 6, 100.0, shared, shared)
    assert torch.equal(shared, apart.sum(0))


@pytest.mark.parametrize("shape", [(1,), (3, 5), (64, 33), (0, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_dropout(shape, dtype):
    x, res = torch.randn(shape).to(dtype), torch.randn(shape).to(dtype)
    for p in (0.0, 0.3, 0.9999):
        y, slack, keep = oracle.dropout(x, p, 11, 12)
        got = ops.dropout(x, p, 11, 12)
        oracle.close(got, y, slack, "y")
        assert torch.equal(got[~keep], torch.zeros_like(got[~keep]))
        y, slack, _ = oracle.dropout(x, p, 11, 12, res)
        oracle.close(ops.dropout(x, p, 11, 12, residual=res), y, slack, "y + residual")
    assert torch.equal(ops.dropout(x, 0.3, 11, torch.tensor(12)), ops.dropout(x, 0.3, 11, 12))
    x2 = x.clone()
    assert ops.dropout(x2, 0.3, 11, 12, out=x2) is x2 and torch.equal(x2, ops.dropout(x, 0.3, 11, 12))


def test_dropout_statistics_and_dropped_garbage():
    x = torch.ones(200_000)
    for p in (0.1, 0.5):
        kept = (ops.dropout(x, p, 1, 2) != 0).double().mean().item()
        assert abs(kept - (1 - p)) < 6 * math.sqrt(p * (1 - p) / x.numel())  # six standard deviations
    a, b = (ops.dropout(x, 0.5, 1, o) != 0 for o in (2, 3))
    assert abs((a == b).double().mean().item() - 0.5) < 6 * 0.5 / math.sqrt(x.numel())  # offsets are independent
    bad = torch.full((64,), float("nan"))
    y = ops.dropout(bad, 0.5, 1, 2)
    keep = oracle.dropout(bad, 0.5, 1, 2)[2]
    assert y[~keep].eq(0).all() and y[keep].isnan().all()


LOGITS = [(1, 1), (5, 7), (4, 64), (3, 1003)]


def _logits(T, V, dtype):
    x = (torch.randn(T, V + 5) * 3).to(dtype)
    t = torch.randint(0, V, (T,))
    return x, t


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,V", LOGITS)
def test_token_logprobs(T, V, dtype):
    x, t = _logits(T, V, dtype)
    t[-1] = -100
    lp, stats = ops.token_logprobs(x, V, t)
    want, wstats, _, _ = oracle.logprobs(x, V, t)
    oracle.close(lp, *want, "logp")
    oracle.close(stats, *wstats, "stats")
    up = torch.randn(T)
    up[0] = 0
    d = ops.token_logprobs_bwd(x, V, t, stats, up)
    oracle.close(d, *oracle.dlogits(x, V, t, up), "dlogits")
    x2 = x.clone()
    ops.token_logprobs_bwd(x2, V, t, stats, up, out=x2)
    assert torch.equal(x2[:, :V], d) and torch.equal(x2[:, V:], x[:, V:])


def test_token_logprobs_rows_of_infinities():
    V = 12
    x = torch.randn(6, V)
    x[0] = -math.inf
    x[5] = torch.finfo(torch.float32).min  # masked by the type's lowest value: a uniform row
    x[1, 3:] = -math.inf
    x[2, 4] = math.nan
    x[3, 5] = math.inf
    t = torch.tensor([2, 1, 0, 0, 7, 3])
    lp, stats = ops.token_logprobs(x, V, t)
    assert lp[0] == -math.inf and stats[0].tolist() == [-math.inf, 0.0]
    assert lp[2].isnan() and lp[3].isnan()
    fine = [1, 4, 5]
    oracle.close(lp[fine], *oracle.logprobs(x[fine], V, t[fine])[0])
    d = ops.token_logprobs_bwd(x, V, t, stats, torch.ones(6))
    oracle.close(d[fine], *oracle.dlogits(x[fine], V, t[fine], torch.ones(3)))
    assert d[0].eq(0).all() and d[1, 3:].eq(0).all() and d[2].isnan().all()
    assert ops.token_logprobs_bwd(x, V, t, stats, torch.zeros(6)).eq(0).all()


POLICY = dict(low=0.2, high=0.3, kl=0.05, scale=0.5)


def _policy_inputs(x, V, t, device="cpu"):
    T = t.shape[0]
    lp = oracle.logprobs(x, V, t)[0][0].float().cpu()
    r = torch.randn(T) * 0.2
    r[::3] = 0.0  # unchanged policy: both sides of the max equal
    old, ref, adv = lp - r, lp + torch.randn(T) * 0.1, torch.randn(T)
    w = torch.rand(T)
    w[1::4] = 0.0
    return [v.to(device) for v in (old, ref, adv, w)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,V", LOGITS + [(40, 33)])
def test_policy_loss_chunk(T, V, dtype):
    x, t = _logits(T, V, dtype)
    old, ref, adv, w = _policy_inputs(x, V, t)
    kw = dict(clip_low=0.2, clip_high=0.3, kl_coef=0.05, grad_scale=0.5)
    loss, lp, d = ops.policy_loss_chunk(x, V, t, old, adv, w, ref_logps=ref, **kw)
    want = oracle.policy(x, V, t, old, adv, w, ref, 0.2, 0.3, 0.05, 0.5)
    for got, (r, s), n in zip((loss, lp, d), want, ("loss", "logp", "dlogits")):
        oracle.close(got, r, s, n)
    kw["kl_coef"] = 0.0
    loss, lp, d = ops.policy_loss_chunk(x, V, t, old, adv, **kw)
    want = oracle.policy(x, V, t, old, adv, None, None, 0.2, 0.3, 0.0, 0.5)
    for got, (r, s), n in zip((loss, lp, d), want, ("loss", "logp", "dlogits")):
        oracle.close(got, r, s, n)


def test_policy_gradient_is_the_derivative():
    T, V = 4, 6
    x = torch.randn(T, V, dtype=torch.float64, requires_grad=True)
    t = torch.randint(0, V, (T,))
    lp = torch.log_softmax(x.detach(), -1).gather(1, t[:, None])[:, 0]
    old, ref = lp - torch.tensor([0.5, -0.5, 0.05, 0.4]), lp + 0.3 * torch.randn(T, dtype=torch.float64)
    adv, w = torch.tensor([1.0, -2.0, 0.5, -0.7], dtype=torch.float64), torch.rand(T, dtype=torch.float64)

    class Op(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            losses, _, d = ops.policy_loss_chunk(x, V, t, old, adv, w, ref_logps=ref, kl_coef=0.1)
            ctx.save_for_backward(d)
            return losses.sum()

        @staticmethod
        def backward(ctx, g):
            return ctx.saved_tensors[0] * g

    assert torch.autograd.gradcheck(Op.apply, (x,))


def test_policy_masked_rows_hold_garbage():
    x, t = _logits(4, 9, torch.float32)
    x[1], x[2, 3] = math.nan, math.inf
    t[3] = 9
    w = torch.tensor([1.0, 0.0, 0.0, 1.0])
    bad = torch.tensor([0.0, math.nan, math.inf, math.nan])
    loss, lp, d = ops.policy_loss_chunk(x, 9, t, bad, torch.tensor([1.0, math.nan, -math.inf, 1.0]), w,
                                        ref_logps=bad, kl_coef=0.1)
    assert loss[1:].eq(0).all() and d[1:].eq(0).all() and lp[3] == 0 and d[0].isfinite().all()


@pytest.mark.parametrize("form,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.1), ("squared", 0.0)])
@pytest.mark.parametrize("P,S", [(1, 1), (2, 7), (3, 300), (0, 4), (2, 0)])
def test_preference_loss(P, S, form, smoothing):
    lp, ref = -5 * torch.rand(2 * P, S), -5 * torch.rand(2 * P, S)
    mask = torch.rand(2 * P, S) < 0.7
    if P > 1:
        mask[1] = False  # an answer whose tokens are all masked
    lp[~mask] = math.nan
    got = ops.preference_loss(lp, ref, mask, 0.3, form=form, label_smoothing=smoothing, grad_scale=0.5)
    want = oracle.preference(lp, ref, mask, 0.3, form, smoothing, 0.5)
    for g, r, n in zip(got, want, ("loss", "reward", "dlogps")):
        oracle.close(g, r, 1e-12 * (1 + r.abs()), n)


@pytest.mark.parametrize("form,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.2), ("squared", 0.0)])
def test_preference_gradient_is_the_derivative(form, smoothing):
    lp = torch.randn(4, 5, dtype=torch.float64, requires_grad=True)
    ref, mask = torch.randn(4, 5, dtype=torch.float64), torch.rand(4, 5) < 0.6

    class Op(torch.autograd.Function):
        @staticmethod
        def forward(ctx, lp):
            losses, _, d = ops.preference_loss(lp, ref, mask, 0.7, form=form, label_smoothing=smoothing)
            ctx.save_for_backward(d)
            return losses.sum()

        @staticmethod
        def backward(ctx, g):
            return ctx.saved_tensors[0] * g

    assert torch.autograd.gradcheck(Op.apply, (lp,))


def test_policy_loss_at_probabilities_of_zero():
    """An old probability of 0 (or a ratio past the type's range) beside an advantage of 0, and a KL term of a
    token the policy gives probability 0: the formula's limits 0 and infinity, not NaN."""
    V = 9
    x = torch.zeros(4, V)
    x[2, 1] = -math.inf
    t = torch.ones(4, dtype=torch.int64)
    lp = -math.log(V)
    old = torch.tensor([-math.inf, -200.0, 0.0, lp])
    adv = torch.tensor([0.0, 0.0, 1.0, 1.0])
    loss, _, d = ops.policy_loss_chunk(x, V, t, old, adv)
    assert loss[:2].tolist() == [0.0, 0.0] and d[:2].eq(0).all()
    assert loss[2] == 0 and d[2].eq(0).all() and d[3].isfinite().all() and d[3, 1] < 0
    loss, lps, d = ops.policy_loss_chunk(x, V, t, old, adv, ref_logps=torch.full_like(old, lp), kl_coef=0.5)
    assert lps[2] == -math.inf and loss[2] == math.inf and loss[[0, 1, 3]].isfinite().all()


def test_gradients_of_infinite_coefficients():
    """The target's entry too is (onehot - softmax) times the infinity."""
    x, t = _logits(3, 7, torch.float32)
    up = torch.tensor([math.inf, -math.inf, 0.0])
    lp, stats = ops.token_logprobs(x, 7, t)
    ref = oracle.dlogits(x, 7, t, up)[0]
    oracle.close(ops.token_logprobs_bwd(x, 7, t, stats, up), ref, torch.zeros_like(ref))
    x[torch.arange(3), t] = -math.inf
    zero = torch.zeros(3)
    _, _, d = ops.policy_loss_chunk(x, 7, t, zero, zero, ref_logps=zero - 1, kl_coef=0.1)
    assert d[torch.arange(3), t].eq(-math.inf).all() and d.isinf().all()


def test_preference_of_an_impossible_answer():
    """A token of probability 0 makes the margin infinite: the loss of the side that has weight 0 is left out."""
    lp = torch.tensor([[-1.0], [-math.inf], [-math.inf], [-1.0]])
    args = (torch.zeros_like(lp), torch.ones_like(lp, dtype=torch.bool), 0.5)
    loss, rewards, d = ops.preference_loss(lp, *args)
    assert loss.tolist() == [0.0, math.inf] and d.reshape(-1).tolist() == [0.0, 0.0, -0.5, 0.5]
    assert rewards.tolist() == [-0.5, -math.inf, -math.inf, -0.5]
    loss, _, d = ops.preference_loss(lp, *args, label_smoothing=1.0)
    assert loss.tolist() == [math.inf, 0.0] and d.reshape(-1).tolist() == [0.5, -0.5, 0.0, 0.0]
    assert ops.preference_loss(lp, *args, label_smoothing=0.25)[0].tolist() == [math.inf, math.inf]


def test_preference_step_from_logits_is_the_derivative():
    """Log probabilities, loss and gradient of the logits together, against autograd of the formula in 64 bits."""
    P, S, V = 2, 6, 11
    x = torch.randn(2 * P * S, V, dtype=torch.float64)
    t = torch.randint(0, V, (2 * P * S,))
    t[5] = -100
    ref, mask = torch.randn(2 * P, S, dtype=torch.float64), torch.rand(2 * P, S) < 0.8
    lp, stats = ops.token_logprobs(x, V, t)
    _, _, dlp = ops.preference_loss(lp.view(2 * P, S), ref, mask, 0.2, grad_scale=1 / P)
    d = ops.token_logprobs_bwd(x, V, t, stats, dlp)
    xr = x.clone().requires_grad_()
    l2 = torch.log_softmax(xr, -1).gather(1, t.clamp(min=0)[:, None])[:, 0] * (t >= 0)
    r = ((l2.view(2 * P, S) - ref) * mask).sum(1)
    (-torch.nn.functional.logsigmoid(0.2 * (r[0::2] - r[1::2]))).mean().backward()
    assert torch.allclose(d, xr.grad, rtol=1e-10, atol=1e-14)


def _raises(fn, *args, **kw):
    with pytest.raises(ValueError):
        fn(*args, **kw)


def refusals(device):
    """Calls every backend refuses with a ValueError before any kernel runs."""
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device=device)  # noqa: E731
    x, g, dg = z(4, 96), z(32), z(32)
    good = (4, 1, 1, 32, 10000.0)
    _raises(ops.qk_norm_rope, z(4, 3, 32), g, g, *good)
    _raises(ops.qk_norm_rope, z(4, 63), g, g, *good)
    _raises(ops.qk_norm_rope, x, z(31), g, *good)
    _raises(ops.qk_norm_rope, x, g, z(32, dt=torch.bfloat16), *good)
    _raises(ops.qk_norm_rope, x, g, g, 0, 1, 1, 32, 10000.0)
    _raises(ops.qk_norm_rope, x, g, g, 4, 0, 0, 32, 10000.0)
    _raises(ops.qk_norm_rope, x, z(3), z(3), 4, 1, 1, 3, 10000.0)
    _raises(ops.qk_norm_rope, x, g, g, *good, out=z(4, 60))
    _raises(ops.qk_norm_rope, x, g, g, *good, out=z(4, 64, dt=torch.bfloat16))
    _raises(ops.qk_norm_rope, x, g, g, *good, out=z(64, 4).t())
    _raises(ops.qk_norm_rope_bwd, z(3, 64), x, g, g, *good, dg, dg)
    _raises(ops.qk_norm_rope_bwd, x, x, g, g, *good, z(31), dg)
    _raises(ops.qk_norm_rope_bwd, x, x, g, g, *good, z(64)[::2], dg)
    _raises(ops.qk_norm_rope_bwd, x, x, g, g, *good, z(32, dt=torch.bfloat16), dg)
    for p in (-0.1, 1.0, 0.999999, math.nan):
        _raises(ops.dropout, x, p, 0, 0)
    _raises(ops.dropout, x, 0.1, -1, 0)
    _raises(ops.dropout, x, 0.1, 0, 1 << 64)
    _raises(ops.dropout, x, 0.1, 0, z(1))
    _raises(ops.dropout, x, 0.1, 0, z(2, dt=torch.int64))
    _raises(ops.dropout, x, 0.1, 0, 0, residual=z(4, 95))
    _raises(ops.dropout, x, 0.1, 0, 0, residual=z(4, 96, dt=torch.bfloat16))
    _raises(ops.dropout, x, 0.1, 0, 0, out=z(96, 4).t())
    t, v = z(4, dt=torch.int64), z(4)
    _raises(ops.token_logprobs, x, 97, t)
    _raises(ops.token_logprobs, x, 0, t)
    _raises(ops.token_logprobs, x, 96, z(3, dt=torch.int64))
    _raises(ops.token_logprobs, x, 96, z(4, dt=torch.int32))
    _raises(ops.token_logprobs, x[0], 96, t)
    _raises(ops.token_logprobs_bwd, x, 96, t, z(4, 2), z(4, dt=torch.bfloat16))
    _raises(ops.token_logprobs_bwd, x, 96, t, z(9), v)
    _raises(ops.token_logprobs_bwd, x, 96, t, z(4, 2), v, out=z(4, 95))
    _raises(ops.token_logprobs_bwd, x, 96, t, z(4, 2), v, out=z(96, 4).t())
    _raises(ops.policy_loss_chunk, x, 96, t, v, z(5))
    _raises(ops.policy_loss_chunk, x, 96, t, v, v, clip_low=1.5)
    _raises(ops.policy_loss_chunk, x, 96, t, v, v, clip_high=-0.1)
    _raises(ops.policy_loss_chunk, x, 96, t, v, v, kl_coef=0.1)
    _raises(ops.policy_loss_chunk, x, 96, t, v, v, z(4, dt=torch.float16))
    lp, m = z(4, 5), z(4, 5, dt=torch.bool)
    _raises(ops.preference_loss, z(3, 5), z(3, 5), z(3, 5, dt=torch.bool))
    _raises(ops.preference_loss, lp, z(4, 6), m)
    _raises(ops.preference_loss, lp, lp, lp)
    _raises(ops.preference_loss, z(4, 5, dt=torch.bfloat16), lp, m)
    _raises(ops.preference_loss, lp, lp, m, beta=0.0)
    _raises(ops.preference_loss, lp, lp, m, form="hinge")
    _raises(ops.preference_loss, lp, lp, m, label_smoothing=1.5)
    _raises(ops.preference_loss, lp, lp, m, form="squared", label_smoothing=0.1)


def test_refusals():
    refusals("cpu")
