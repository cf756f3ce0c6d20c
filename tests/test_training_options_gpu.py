"""Head norms, dropout and the preference and policy objectives on the kernels, in the block and the engine."""

import pytest
import torch
import torch.nn.functional as F

from meshtrain_b200 import ops
from meshtrain_b200.models import build_model_spec
from meshtrain_b200.models.base import RNG_KEY
from meshtrain_b200.models.objectives import PolicyObjective, PreferenceObjective

pytestmark = pytest.mark.gpu

GPT = {"type": "gpt", "layers": 2, "hidden_size": 512, "heads": 8, "vocab_size": 2051, "seq_len": 256,
       "dtype": "bfloat16", "dropout": 0.2}
LLAMA = {"type": "llama", "layers": 2, "hidden_size": 512, "heads": 4, "n_kv_heads": 2, "ffn_hidden": 1024,
         "vocab_size": 20011, "seq_len": 256, "dtype": "bfloat16", "dropout": 0.1, "qk_norm": True}


@pytest.fixture(autouse=True)
def _custom_kernels():
    torch.manual_seed(0)
    ops.set_backend("custom")
    yield
    ops.set_backend("custom")
    torch.cuda.synchronize()
    assert ops.read_status(torch.cuda.current_device()) == 0


def _rel_l2(out, ref):
    out, ref = out.float(), ref.float()
    return ((out - ref).norm() / (ref.norm() + 1e-12)).item()


def _rms(x, w):
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5) * w


@pytest.mark.parametrize("hidden,H,HK", [(1024, 8, 2), (512, 8, 8)])  # head dimension 128 and 64
def test_llama_block_with_head_norms_and_dropout(hidden, H, HK):
    from meshtrain_b200.models.llama import LlamaBlock

    B, S, ffn, theta, p, rng = 2, 640, 1536, 500000.0, 0.15, (77, 1 << 35)
    hd = hidden // H
    block = LlamaBlock(hidden, H, HK, ffn, rope_theta=theta, qk_norm=True, dropout=p)
    for n in ("q_norm", "k_norm"):
        getattr(block, n).weight.data.add_(0.2 * torch.randn(hd))
    block = block.cuda().to(torch.bfloat16)
    x, dy = (torch.randn(B, S, hidden, device="cuda").to(torch.bfloat16) for _ in range(2))
    saved = {RNG_KEY: rng}
    y = block.fwd(x, saved)
    grads = {n: torch.zeros(q.shape, device="cuda") for n, q in block.named_parameters()}
    dx = block.bwd(dy, saved, grads)

    w = {n: q.detach().float().requires_grad_() for n, q in block.named_parameters()}
    xf = x.float().requires_grad_()
    drop = lambda t, site: torch.where(  # noqa: E731
        ops._keep_mask(t.shape, round(p * 65536), rng[0], rng[1] + site, "cuda"), t / (1 - round(p * 65536) / 65536), 0.0)
    q, k, v = (_rms(xf, w["attn_norm.weight"]) @ w["wqkv.weight"].t()).view(B, S, -1, hd).split([H, HK, HK], 2)
    ang = torch.outer(torch.arange(S, device="cuda").double(),
                      theta ** (torch.arange(hd // 2, device="cuda").double() * (-2.0 / hd)))
    cs, sn = ang.cos().float()[None, :, None], ang.sin().float()[None, :, None]

    def rotate(t):
        a, b = t.chunk(2, -1)
        return torch.cat([a * cs - b * sn, b * cs + a * sn], -1)

    q, k = rotate(_rms(q, w["q_norm.weight"])), rotate(_rms(k, w["k_norm.weight"]))
    k, v = (t.repeat_interleave(H // HK, 2) for t in (k, v))
    s = torch.einsum("bqhd,bkhd->bhqk", q, k) / hd ** 0.5
    s = s.masked_fill(torch.ones(S, S, dtype=torch.bool, device="cuda").triu(1), float("-inf"))
    o = torch.einsum("bhqk,bkhd->bqhd", torch.softmax(s, -1), v).reshape(B, S, -1)
    x1 = xf + drop(o @ w["wo.weight"].t(), 0)
    g, u = ops.split_gate_up(_rms(x1, w["mlp_norm.weight"]) @ w["w_gate_up.weight"].t())
    ref = x1 + drop((F.silu(g) * u) @ w["w_down.weight"].t(), 1)
    ref.backward(dy.float())
    # bf16 activations between the GEMMs, as in the block without these options
    assert _rel_l2(y, ref) < 2e-2
    assert _rel_l2(dx, xf.grad) < 3e-2
    for name, grad in grads.items():
        assert _rel_l2(grad, w[name].grad) < 3e-2, name


def _step(cfg, objective=None, recompute=None, backend="custom", deferred=True, chunk_tokens=None, repeats=1):
    from meshtrain_b200.parallel.engine import PipelineEngine

    ops.set_backend(backend)
    spec = build_model_spec(cfg, seed=7)
    eng = PipelineEngine(spec, layer_range=(0, spec.num_layers), stage=0, num_stages=1, device="cuda:0",
                         num_microbatches=2, optimizer="sgd", lr=0.0, init_on_device=True, objective=objective,
                         recompute=set(range(1, spec.num_layers - 1)) if recompute else None,
                         deferred_wgrad=deferred)
    if chunk_tokens:
        eng.layers[-1]._chunk_tokens = lambda T: chunk_tokens
    x, y = spec.make_batch(0, 8)
    y = y.clone()
    extras = None
    if objective is not None:
        y[:, :9] = -100
        g = torch.Generator().manual_seed(1)
        noise = lambda: 0.2 * torch.randn(y.shape, generator=g)  # noqa: E731
        lp = eng.logprobs(x, y).cpu()
        mask = torch.rand(y.shape, generator=g) < 0.8
        extras = {"ref_logps": lp + noise(), "mask": mask}
        if isinstance(objective, PolicyObjective):
            extras |= {"old_logps": lp + noise(), "advantages": 5 * noise()}
    before = ops.launches()
    for _ in range(repeats):  # lr 0: each repeats the last
        st = eng.train_step(4, x.pin_memory(), y.pin_memory(), extras=extras)
    torch.cuda.synchronize()
    return float(st.loss) / 2, eng.named_gradients_cpu(), ops.launches() - before


@pytest.mark.parametrize("objective", [None, PreferenceObjective(0.3), PolicyObjective(kl_coef=0.1)],
                         ids=["cross-entropy", "preference", "policy"])
@pytest.mark.parametrize("cfg", [GPT, LLAMA], ids=["gpt", "llama"])
def test_engine_on_the_kernels_matches_torch(cfg, objective):
    loss, grads, launched = _step(cfg, objective)
    want, ref, none = _step(cfg, objective, backend="torch")
    assert launched > 0 and none == 0
    assert loss == pytest.approx(want, rel=2e-2, abs=2e-3)
    # Both run in bf16, each with its own rounding: 5e-2.  The clip's gradient jumps besides.  A log ratio is a
    # difference of two passes' log probabilities; bf16 logits of 2 to 4 are off by 2^-7 / sqrt(3) = 4.5e-3
    # (root mean square), so the two runs' log ratios differ by sqrt(4) * 4.5e-3 = 9e-3, 7e-3 in the mean.
    # Log ratios have a deviation of 0.2, so a density of 1.1 to 1.4 per unit at the borders, and a border
    # matters for one sign of the advantage: 7e-3 * (1.1 + 1.4) / 2 = 0.9% of the tokens keep their gradient
    # in one run and lose it in the other, sqrt(0.009) = 0.095 of the gradient's norm.
    bound = 5e-2 + (0.095 if isinstance(objective, PolicyObjective) else 0.0)
    for k, r in ref.items():
        assert _rel_l2(grads[k], r) < bound, k


def test_logprobs_under_a_failure_watch():
    """With peers to watch, the pass waits for its end on the host, by polling."""
    from meshtrain_b200.parallel.engine import PipelineEngine

    spec = build_model_spec(LLAMA, seed=7)
    eng = PipelineEngine(spec, layer_range=(0, spec.num_layers), stage=0, num_stages=1, device="cuda:0",
                         num_microbatches=2, init_on_device=True)
    x, y = spec.make_batch(0, 4)
    want = eng.logprobs(x, y)
    eng.failure_check = lambda: None
    got = eng.logprobs(x, y)
    assert torch.cuda.current_stream().query() and torch.equal(got, want)


def test_recompute_repeats_the_masks():
    loss, grads, _ = _step(LLAMA)
    again, other, _ = _step(LLAMA, recompute=True)
    assert again == pytest.approx(loss, rel=1e-3)
    for k, r in grads.items():
        assert _rel_l2(other[k], r) < 2e-2, k


@pytest.mark.parametrize("objective", [None, PreferenceObjective(0.3), PolicyObjective(kl_coef=0.1)],
                         ids=["cross-entropy", "preference", "policy"])
@pytest.mark.parametrize("cfg", [GPT, LLAMA], ids=["gpt", "llama"])
def test_chunks_of_logits_with_deferred_weight_gradients(cfg, objective):
    """Eight chunks per microbatch share a logits buffer that weight gradients on the side stream read."""
    chunked = dict(chunk_tokens=128, repeats=4)
    _, want, _ = _step(cfg, objective, deferred=False, **chunked)
    _, one, _ = _step(cfg, objective, deferred=False)
    _, got, _ = _step(cfg, objective, **chunked)
    # The head's: the same GEMMs in the same order; fp32 sums whose order is free (split products, column sums)
    # differ by a few of their 2^-24 half steps: 1e-5.  Below it, attention's backward sums in any order ahead of
    # bf16 roundings of 2^-8 each: 2e-2, as for a recomputed forward.  One chunk and eight: GEMMs of other shapes,
    # whose bf16 logits may round differently, which the clip's border sees as above.
    clip = 0.095 if isinstance(objective, PolicyObjective) else 0.0
    for k, r in want.items():
        assert _rel_l2(got[k], r) < (1e-5 if k.startswith("model.layers.3.") else 2e-2), k
        assert _rel_l2(one[k], r) < 2e-2 + clip, k
