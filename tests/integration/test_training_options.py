"""Head norms, dropout and the preference and policy objectives in the models and the device engine, on CPU.

The references are the formulas under autograd, with the dropout masks taken from the generator."""

import math

import pytest
import torch
import torch.nn.functional as F

from meshtrain_b200 import ops
from meshtrain_b200.config import ConfigError, parse_config
from meshtrain_b200.models import build_model_spec
from meshtrain_b200.models.base import RNG_KEY
from meshtrain_b200.models.objectives import PolicyObjective, PreferenceObjective
from meshtrain_b200.parallel.spawn import spawn_ranks

GPT = {"type": "gpt", "layers": 2, "hidden_size": 32, "heads": 2, "vocab_size": 61, "seq_len": 12, "dtype": "float32"}
LLAMA = {"type": "llama", "layers": 2, "hidden_size": 32, "heads": 4, "n_kv_heads": 2, "ffn_hidden": 48,
         "vocab_size": 61, "seq_len": 12, "dtype": "float32"}
DROP = {"dropout": 0.25}
VARIANTS = [({**GPT, **DROP}, "gpt-dropout"), ({**LLAMA, "qk_norm": True}, "llama-qk-norm"),
            ({**LLAMA, "qk_norm": True, **DROP}, "llama-both")]
IDS = [name for _, name in VARIANTS]
CFGS = [cfg for cfg, _ in VARIANTS]


def _engine(cfg, M=1, seed=3, **kw):
    from meshtrain_b200.parallel.engine import PipelineEngine

    spec = build_model_spec(cfg, seed=seed)
    kw.setdefault("optimizer", "sgd")
    kw.setdefault("lr", 0.0)
    return spec, PipelineEngine(spec, layer_range=(0, spec.num_layers), stage=0, num_stages=1, device="cpu",
                                num_microbatches=M, **kw)


def _drop(x, p, rng, site):
    if not p:
        return x
    keep = ops._keep_mask(x.shape, round(p * 65536), rng[0], rng[1] + site, "cpu")
    return torch.where(keep, x / (1 - round(p * 65536) / 65536), 0.0)


def _rms(x, g):
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5) * g


def _rotate(x, theta):
    S, hd = x.shape[1], x.shape[-1]
    ang = torch.outer(torch.arange(S).double(), theta ** (torch.arange(hd // 2).double() * (-2.0 / hd)))
    cs, sn = ang.cos().float()[None, :, None], ang.sin().float()[None, :, None]
    a, b = x.chunk(2, -1)
    return torch.cat([a * cs - b * sn, b * cs + a * sn], -1)


def _formula(cfg, spec, params, tokens, step, mb, M):
    """Logits of the model written out, ``params`` as layer -> name -> tensor."""
    p, L, hd = cfg.get("dropout", 0.0), spec.num_layers, spec.d_model // spec.n_heads
    rng = lambda layer: (spec.seed, ((step * M + mb) * L + layer) * 4)  # noqa: E731
    B, S = tokens.shape
    w = params[0]
    x = w["tok.weight"][tokens]
    if spec.name == "gpt":
        x = x + w["pos.weight"][:S]
    x = _drop(x, p, rng(0), 2)
    for i in range(1, L - 1):
        w = params[i]
        if spec.name == "gpt":
            h = F.layer_norm(x, (spec.d_model,), w["ln1.weight"], w["ln1.bias"])
            q, k, v = (z.view(B, S, spec.n_heads, hd) for z in
                       F.linear(h, w["qkv.weight"], w["qkv.bias"]).split(spec.d_model, -1))
        else:
            h = _rms(x, w["attn_norm.weight"]) @ w["wqkv.weight"].t()
            q, k, v = (z.view(B, S, -1, hd) for z in
                       h.split([spec.n_heads * hd, spec.n_kv_heads * hd, spec.n_kv_heads * hd], -1))
            if cfg.get("qk_norm"):
                q, k = _rms(q, w["q_norm.weight"]), _rms(k, w["k_norm.weight"])
            q, k = _rotate(q, spec.rope_theta), _rotate(k, spec.rope_theta)
            k, v = (z.repeat_interleave(spec.n_heads // spec.n_kv_heads, 2) for z in (k, v))
        s = torch.einsum("bqhd,bkhd->bhqk", q, k) / math.sqrt(hd)
        a = torch.softmax(s.masked_fill(torch.ones(S, S, dtype=torch.bool).triu(1), -math.inf), -1)
        o = torch.einsum("bhqk,bkhd->bqhd", a, v).reshape(B, S, -1)
        if spec.name == "gpt":
            x = x + _drop(F.linear(o, w["proj.weight"], w["proj.bias"]), p, rng(i), 0)
            h = F.layer_norm(x, (spec.d_model,), w["ln2.weight"], w["ln2.bias"])
            h = F.gelu(F.linear(h, w["fc1.weight"], w["fc1.bias"]))
            x = x + _drop(F.linear(h, w["fc2.weight"], w["fc2.bias"]), p, rng(i), 1)
        else:
            x = x + _drop(o @ w["wo.weight"].t(), p, rng(i), 0)
            g, u = ops.split_gate_up(_rms(x, w["mlp_norm.weight"]) @ w["w_gate_up.weight"].t())
            x = x + _drop((F.silu(g) * u) @ w["w_down.weight"].t(), p, rng(i), 1)
    w = params[L - 1]
    if spec.name == "gpt":
        return F.linear(F.layer_norm(x, (spec.d_model,), w["ln.weight"], w["ln.bias"]), w["out.weight"], w["out.bias"])
    return _rms(x, w["ln.weight"]) @ w["out.weight"].t()


def _reference(cfg, spec, eng, loss_of, step, x, M):
    """Loss and gradients of the mean of ``loss_of(logits, microbatch)`` under autograd."""
    params = [{n: q.detach().clone().requires_grad_() for n, q in layer.named_parameters()} for layer in eng.layers]
    n = x.shape[0] // M
    loss = sum(loss_of(_formula(cfg, spec, params, x[m * n:(m + 1) * n], step, m, M), m) for m in range(M)) / M
    loss.backward()
    return float(loss.detach()), {f"model.layers.{i}.{n}": q.grad for i, layer in enumerate(params)
                                  for n, q in layer.items()}


def _same(got, ref, tol=1e-4):
    for k, r in ref.items():
        err = (got[k] - r).abs().max().item()
        assert err <= tol * (r.abs().max().item() + 1e-6), (k, err)


@pytest.mark.parametrize("cfg", CFGS, ids=IDS)
def test_engine_matches_the_formula(cfg):
    M, step = 2, 5
    spec, eng = _engine(cfg, M)
    x, y = spec.make_batch(0, 4)
    st = eng.train_step(step, x, y)
    ce = lambda lg, m: F.cross_entropy(lg.reshape(-1, lg.shape[-1]), y[2 * m:2 * m + 2].reshape(-1))  # noqa: E731
    loss, ref = _reference(cfg, spec, eng, ce, step, x, M)
    assert float(st.loss) / M == pytest.approx(loss, rel=1e-5)
    _same(eng.named_gradients_cpu(), ref)


@pytest.mark.parametrize("cfg", [CFGS[0], CFGS[2]], ids=["gpt", "llama"])
def test_dropout_differs_by_step_and_microbatch_and_repeats(cfg):
    spec, eng = _engine(cfg, 2)
    x, y = spec.make_batch(0, 2)
    x, y = torch.cat([x[:1], x[:1]]), torch.cat([y[:1], y[:1]])  # two equal microbatches
    losses = [float(eng.train_step(s, x, y).loss) for s in (0, 0, 1)]
    assert losses[0] == losses[1] != losses[2]
    _, one = _engine(cfg, 1)
    assert abs(float(one.train_step(0, x[:1], y[:1]).loss) - losses[0] / 2) > 1e-6


@pytest.mark.parametrize("cfg", CFGS, ids=IDS)
def test_recompute_and_half_blocks_see_the_same_masks(cfg):
    spec, eng = _engine(cfg, 2)
    x, y = spec.make_batch(0, 4)
    loss = float(eng.train_step(3, x, y).loss)
    ref = eng.named_gradients_cpu()
    _, again = _engine(cfg, 2, recompute=set(range(1, spec.num_layers - 1)))
    assert float(again.train_step(3, x, y).loss) == loss
    for k, g in again.named_gradients_cpu().items():
        assert torch.equal(g, ref[k]), k
    half, split = _engine({**cfg, "split_blocks": True}, 2)
    assert half.num_layers == spec.num_layers + spec.n_blocks
    assert float(split.train_step(3, x, y).loss) == loss
    for k, g in split.named_gradients_cpu().items():
        assert torch.equal(g, ref[k]), k


def _rank_train(cfg, objective=False):
    from meshtrain_b200.api import PipelineTrainer

    torch.set_num_threads(1)
    tr = PipelineTrainer(cfg, num_microbatches=4, optimizer="adam", lr=1e-3, device="cpu", microbatch_size=2, seed=3,
                         objective=PreferenceObjective(beta=0.5) if objective else None)
    losses = []
    try:
        x, y = tr.spec.make_batch(0, 8)
        extras = None
        if objective:
            ref = tr.logprobs(x, y)
            assert (ref is None) == (not tr.is_last)
            if tr.is_last:
                assert ref.shape == y.shape and (ref < 0).all()
                extras = {"ref_logps": ref, "mask": torch.arange(y.shape[1]).expand(y.shape) > 3}
        for step in range(3):
            losses.append(tr.loss_value(tr.step(step, x, y, timed=False, extras=extras)))
        params = tr.engine.named_parameters_cpu()
    finally:
        tr.close()
    return losses, params


@pytest.mark.parametrize("cfg,objective", [(CFGS[0], False), (CFGS[2], False), (CFGS[2], True)],
                         ids=["gpt", "llama", "llama-preference"])
def test_two_stages_match_one(cfg, objective):
    one_losses, one = _rank_train(cfg, objective)
    res = spawn_ranks(_rank_train, 2, cfg, objective, timeout_s=240)
    losses = [r[0] for r in res if r[0][0] is not None][0]
    assert losses == pytest.approx(one_losses, rel=1e-6)
    for _, params in res:
        for k, v in params.items():
            assert torch.allclose(v, one[k], rtol=1e-5, atol=1e-7), k


def test_evaluation_does_not_drop():
    spec = build_model_spec(CFGS[2], seed=1)
    layer = spec.build_layer(1)
    x = torch.randn(2, 12, 32)
    layer.eval()
    assert torch.equal(layer.fwd(x, {}), layer.fwd(x, {}))
    layer.train()
    a, b = {}, {}
    assert not torch.equal(layer.fwd(x, a), layer.fwd(x, b)) and a[RNG_KEY] != b[RNG_KEY]
    assert torch.equal(layer.fwd(x, {RNG_KEY: (1, 8)}), layer.fwd(x, {RNG_KEY: (1, 8)}))
    half = build_model_spec({**CFGS[0], "split_blocks": True}).build_layer(1).eval()
    assert torch.equal(half(x), half(x))


@pytest.mark.parametrize("cfg", CFGS, ids=IDS)
def test_layers_under_autograd_drop_alike_both_ways(cfg):
    """The host runtime's path: a layer called as a module draws its numbers once for both directions."""
    spec = build_model_spec(cfg, seed=1)
    layer = spec.build_layer(1)
    x = torch.randn(2, 12, 32, requires_grad=True)
    torch.manual_seed(5)
    y = layer(x)
    dy = torch.randn_like(y)
    y.backward(dy)
    torch.manual_seed(5)
    saved: dict = {}
    grads = {n: torch.zeros_like(q) for n, q in layer.named_parameters()}
    with torch.no_grad():
        y2 = layer.fwd(x.detach(), saved)
        dx = layer.bwd(dy, saved, grads)
    assert torch.equal(y, y2) and torch.equal(x.grad, dx)


@pytest.mark.parametrize("index", [0, 1])
@pytest.mark.parametrize("train", [True, False])
def test_backward_follows_its_forward_after_a_change_of_mode(index, train):
    """The gradient is that of the pass that ran: a layer put into the other mode before its backward runs
    changes nothing."""
    spec = build_model_spec(CFGS[0], seed=1)
    layer = spec.build_layer(index).train(train)
    x = torch.randint(0, 61, (2, 12)) if index == 0 else torch.randn(2, 12, 32)
    dy = torch.randn(2, 12, 32)
    out = []
    for change in (False, True):
        saved = {RNG_KEY: (7, 16)}
        grads = {n: torch.zeros_like(q) for n, q in layer.named_parameters()}
        with torch.no_grad():
            layer.train(train).fwd(x, saved)
            dx = layer.train(train != change).bwd(dy, saved, grads)
        out.append([*grads.values()] + ([] if dx is None else [dx]))
    assert all(torch.equal(a, b) for a, b in zip(*out))


def _pair_inputs(spec, B=4):
    x, y = spec.make_batch(0, B)
    y = y.clone()
    y[:, :2] = -100  # the prompt has no targets
    mask = torch.rand(y.shape) < 0.8
    mask[3] = False  # an answer with no token left
    return x, y, mask


@pytest.mark.parametrize("form,smoothing", [("sigmoid", 0.1), ("squared", 0.0)])
@pytest.mark.parametrize("cfg", [GPT, CFGS[2]], ids=["gpt", "llama"])
def test_preference_objective_matches_the_formula(cfg, form, smoothing):
    torch.manual_seed(0)
    M, beta = 2, 0.4
    spec, eng = _engine(cfg, M, objective=PreferenceObjective(beta, form, smoothing))
    x, y, mask = _pair_inputs(spec)
    ref = -4 + torch.randn(y.shape)
    st = eng.train_step(1, x, y, extras={"ref_logps": ref, "mask": mask})

    def loss_of(lg, m):
        part = slice(2 * m, 2 * m + 2)
        lp = torch.log_softmax(lg, -1).gather(-1, y[part].clamp(min=0)[..., None])[..., 0] * (y[part] >= 0)
        r, n = ((lp - ref[part]) * mask[part]).sum(1), mask[part].sum(1).clamp(min=1)
        if form == "squared":
            return (r[0] / n[0] - r[1] / n[1] - 0.5 / beta).square()
        h = beta * (r[0] - r[1])
        return -(1 - smoothing) * F.logsigmoid(h) - smoothing * F.logsigmoid(-h)

    loss, want = _reference(cfg, spec, eng, loss_of, 1, x, M)
    assert float(st.loss) / M == pytest.approx(loss, rel=1e-4)
    _same(eng.named_gradients_cpu(), want, 5e-4)


@pytest.mark.parametrize("with_ref", [True, False])
def test_policy_objective_matches_the_formula(with_ref):
    torch.manual_seed(0)
    M, cfg, kl = 2, CFGS[2], 0.1 if with_ref else 0.0
    spec, eng = _engine(cfg, M, objective=PolicyObjective(0.2, 0.3, kl))
    x, y, mask = _pair_inputs(spec)
    mask[3, 5] = True
    old = eng.logprobs(x, y) + 0.3 * torch.randn(y.shape)
    adv, ref = torch.randn(y.shape), old + 0.1 * torch.randn(y.shape)
    st = eng.train_step(1, x, y, extras={"old_logps": old, "advantages": adv, "mask": mask,
                                         "ref_logps": ref if with_ref else None})

    def loss_of(lg, m):
        part = slice(2 * m, 2 * m + 2)
        has = y[part] >= 0
        lp = torch.log_softmax(lg, -1).gather(-1, y[part].clamp(min=0)[..., None])[..., 0]
        ratio, A, d = torch.exp(lp - old[part]), adv[part], ref[part] - lp
        loss = torch.maximum(-A * ratio, -A * ratio.clamp(0.8, 1.3)) + kl * (torch.exp(d) - d - 1)
        return (loss * mask[part] * has).sum() / mask[part].sum()

    loss, want = _reference(cfg, spec, eng, loss_of, 1, x, M)
    assert float(st.loss) / M == pytest.approx(loss, rel=1e-4, abs=1e-6)
    _same(eng.named_gradients_cpu(), want, 5e-4)


def test_losses_in_chunks_match_one_chunk():
    torch.manual_seed(0)
    head = build_model_spec(GPT, seed=2).build_layer(3)
    x = torch.randn(4, 12, 32)
    y = torch.randint(0, 61, (4, 12))
    y[0, :5] = -100
    f32 = lambda: torch.randn(4, 12) - 4  # noqa: E731
    mask = torch.rand(4, 12) < 0.7
    calls = {"fwd_preference_loss": dict(ref_logps=f32(), mask=mask),
             "fwd_policy_loss": dict(old_logps=f32(), advantages=f32(), mask=mask, ref_logps=f32(), kl_coef=0.1)}
    for name, kw in calls.items():
        runs = []
        for chunk in (48, 7):
            saved, loss = {}, torch.zeros(())
            grads = {n: torch.zeros_like(q) for n, q in head.named_parameters()}
            with torch.no_grad():
                getattr(head, name)(x, y, saved, grads, loss, 0.5, chunk_tokens=chunk, **kw)
            runs.append((loss, saved["dx"], grads))
        (l0, d0, g0), (l1, d1, g1) = runs
        assert torch.allclose(l0, l1, rtol=1e-6) and torch.allclose(d0, d1, rtol=1e-4, atol=1e-7)
        for n in g0:
            assert torch.allclose(g0[n], g1[n], rtol=1e-4, atol=1e-6), (name, n)
    with torch.no_grad():
        assert torch.allclose(head.logprobs(x, y, 48), head.logprobs(x, y, 7), rtol=1e-6)
        want = torch.log_softmax(head(x), -1).gather(-1, y.clamp(min=0)[..., None])[..., 0] * (y >= 0)
    assert torch.allclose(head.logprobs(x, y), want, atol=1e-5)


@pytest.mark.parametrize("name", ["fwd_preference_loss", "fwd_policy_loss"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_losses_of_a_64_bit_head(name, dtype):
    """fp32 per-token tensors (what ``logprobs`` and an engine's step bring) or 64-bit ones, which an fp32 head
    refuses."""
    torch.manual_seed(0)
    head = build_model_spec(GPT, seed=2).build_layer(3).double()
    x, y = torch.randn(4, 12, 32, dtype=torch.float64), torch.randint(0, 61, (4, 12))
    lp = head.logprobs(x, y).detach()
    adv = torch.randn(4, 12)
    kw = dict(ref_logps=lp) if name == "fwd_preference_loss" else dict(old_logps=lp, advantages=adv)
    kw = {k: v.to(dtype) for k, v in kw.items()} | {"mask": torch.rand(4, 12) < 0.7}

    def run(head, x):
        grads, loss, saved = {n: torch.zeros(q.shape) for n, q in head.named_parameters()}, torch.zeros(()), {}
        with torch.no_grad():
            getattr(head, name)(x, y, saved, grads, loss, 1.0, **kw)
        return loss, saved["dx"], grads

    loss, dx, grads = run(head, x)
    assert dx.dtype == torch.float64
    single = head.float()
    if dtype == torch.float64:
        with pytest.raises(ValueError):
            run(single, x.float())
        return
    loss32, dx32, grads32 = run(single, x.float())
    assert torch.allclose(loss, loss32, rtol=1e-5, atol=1e-6)
    _same({"dx": dx.float(), **grads}, {"dx": dx32, **grads32}, 1e-4)


@pytest.mark.parametrize("name", ["fwd_loss", "fwd_preference_loss", "fwd_policy_loss"])
def test_chunked_losses_wait_for_deferred_weight_gradients(name, monkeypatch):
    """The chunks share one logits buffer: with weight gradients run as late as a side stream may run them,
    each still has to see its own chunk's rows."""
    torch.manual_seed(0)
    head = build_model_spec(GPT, seed=2).build_layer(3)
    x, y = torch.randn(4, 12, 32), torch.randint(0, 61, (4, 12))
    f32 = lambda: torch.randn(4, 12) - 4  # noqa: E731
    mask = torch.rand(4, 12) < 0.7
    kw = {"fwd_loss": {}, "fwd_preference_loss": dict(ref_logps=f32(), mask=mask),
          "fwd_policy_loss": dict(old_logps=f32(), advantages=f32(), mask=mask)}[name]

    def run():
        grads = {n: torch.zeros_like(q) for n, q in head.named_parameters()}
        with torch.no_grad():
            getattr(head, name)(x, y, {}, grads, torch.zeros(()), 0.5, chunk_tokens=7, **kw)
        return grads

    want = run()
    real, late = ops.linear_wgrad_, []

    def drain(device=None):
        while late:
            real(*late.pop(0))

    monkeypatch.setattr(ops, "linear_wgrad_", lambda *args: late.append(args))
    monkeypatch.setattr(ops, "wait_wgrad", drain, raising=False)
    got = run()
    drain()
    for n, r in want.items():
        assert torch.equal(got[n], r), n


@pytest.mark.parametrize("chunk", [48, 7])
def test_preference_loss_holds_one_buffer_of_logits(chunk, monkeypatch):
    """What the memory estimate counts: both passes over the logits go through the same buffer."""
    head = build_model_spec(GPT, seed=2).build_layer(3)
    made = []
    real = head._logits_buffer
    monkeypatch.setattr(head, "_logits_buffer", lambda *a: made.append(1) or real(*a))
    grads = {n: torch.zeros_like(q) for n, q in head.named_parameters()}
    with torch.no_grad():
        head.fwd_preference_loss(torch.randn(4, 12, 32), torch.randint(0, 61, (4, 12)), {}, grads, torch.zeros(()), 1.0,
                                 ref_logps=-torch.rand(4, 12), mask=torch.ones(4, 12, dtype=torch.bool),
                                 chunk_tokens=chunk)
    assert len(made) == 1


def test_objective_refusals():
    spec, eng = _engine(GPT, 1, objective=PreferenceObjective())
    x, y = spec.make_batch(0, 4)
    ref, mask = torch.zeros(4, 12), torch.ones(4, 12, dtype=torch.bool)
    for extras in (None, {"ref_logps": ref}, {"ref_logps": ref, "mask": mask, "other": ref},
                   {"ref_logps": ref.double(), "mask": mask}, {"ref_logps": ref[:2], "mask": mask}):
        with pytest.raises(ValueError):
            eng.train_step(0, x, y, extras=extras)
    _, plain = _engine(GPT, 1)
    with pytest.raises(ValueError):
        plain.train_step(0, x, y, extras={"mask": mask})
    _, odd = _engine(GPT, 1, objective=PreferenceObjective())
    with pytest.raises(ValueError):
        odd.train_step(0, x[:3], y[:3], extras={"ref_logps": ref[:3], "mask": mask[:3]})
    with pytest.raises(ValueError):
        _engine({"type": "mlp", "dtype": "float32"}, 1, objective=PreferenceObjective())


def test_logprobs_of_a_middle_stage_needs_its_batch():
    from meshtrain_b200.parallel.engine import PipelineEngine

    spec = build_model_spec(GPT, seed=3)
    middle = PipelineEngine(spec, layer_range=(1, 2), stage=1, num_stages=3, device="cpu", num_microbatches=2,
                            links=object())
    with pytest.raises(ValueError, match="microbatch_size"):
        middle.logprobs()


@pytest.mark.parametrize("rows", [2, 5])
def test_a_batch_that_the_microbatches_do_not_divide_is_refused_alike(rows):
    for objective in (None, PreferenceObjective()):
        spec, eng = _engine(GPT, 4, objective=objective)
        x, y = spec.make_batch(0, rows)
        extras = objective and {"ref_logps": torch.zeros(rows, 12), "mask": torch.ones(rows, 12, dtype=torch.bool)}
        with pytest.raises(ValueError, match="divisible by the number of microbatches"):
            eng.train_step(0, x, y, extras=extras)


def test_config_keys():
    model = {k: v for k, v in LLAMA.items()}
    cfg = parse_config({"model": {**model, "qk_norm": True, "dropout": 0.1}})
    spec = cfg.build_model_spec()
    assert spec.qk_norm and spec.dropout == 0.1 and spec.build_layer(1).q_norm.weight.shape == (8,)
    plain = parse_config({"model": model}).build_model_spec()
    assert not plain.qk_norm and plain.dropout == 0.0 and not hasattr(plain.build_layer(1), "q_norm")
    assert "dropout" not in parse_config({"model": model}).model_spec_dict()
    for bad in ({**GPT, "qk_norm": True}, {**GPT, "dropout": 1.0}, {**GPT, "dropout": -0.1},
                {**GPT, "dropout": 0.9999999}, {"type": "mlp", "dropout": 0.1}):
        with pytest.raises(ConfigError):
            parse_config({"model": bad})


@pytest.mark.parametrize("cfg", CFGS, ids=IDS)
def test_meta_profile_is_that_of_the_model_without_dropout(cfg):
    from meshtrain_b200.planner.graph import profile_model

    with_drop, without = (profile_model(build_model_spec({**cfg, "dropout": p}), 2) for p in (0.2, 0.0))
    assert with_drop == without


def test_random_numbers_come_from_the_cpu_generator_whatever_the_default_device():
    layer = build_model_spec(CFGS[0]).build_layer(1)
    torch.manual_seed(3)
    want = layer._rng({}, 1)
    torch.manual_seed(3)
    with torch.device("meta"):
        assert layer._rng({}, 1) == want


def test_planner_counts_the_normalised_heads():
    from meshtrain_b200.planner.graph import analytic_profile

    a, b = (analytic_profile(build_model_spec({**LLAMA, "qk_norm": on}), 2)[1] for on in (False, True))
    assert b.saved_bytes - a.saved_bytes == 2 * 12 * 6 * 8 * 4 and b.params - a.params == 16
