"""Functional op layer over the hand-written sm_100a kernels.

Every hot op of the models is one function here with an explicit forward and
backward (no autograd inside).  Dispatch rule, per call:

* CUDA tensor, bf16, backend ``"custom"`` (default) -> the kernel in the
  in-tree extension ``meshtrain_b200.ops._C``.  If the extension is missing on
  a CUDA machine the call raises; there is no silent library fallback.
* anything else (CPU tensors, fp32, or backend ``"torch"``) -> a plain PyTorch
  restatement of the same math.  That path is the numerics oracle for the
  kernels, the fp32 parity path, and what runs on CPU-only hosts.

``qk_norm_rope``, ``dropout``, ``token_logprobs``, ``policy_loss_chunk`` and their
backwards have kernels for bf16, fp16 and fp32 alike.

The reference runs all of these as stock PyTorch ops (reference
models/tiny_transformer.py:19-59, runtime/stage.py:28-36); here they are the
replacement kernels' entry points.
"""

from __future__ import annotations

import math
import os
import threading
from contextlib import contextmanager

import torch
import torch.nn.functional as F

_EXT = None
_EXT_ERR: str | None = None
_BACKEND = os.environ.get("MESHTRAIN_KERNELS", "custom")

EPI_BF16, EPI_GELU, EPI_RESID, EPI_DGELU, EPI_F32, EPI_SWIGLU = range(6)


# Kernel launches issued through this module since import (each binding call
# launches one kernel; the attention bindings report their own count).
LAUNCHES = 0
_MULTI_LAUNCH = {"attention_fwd": 1, "attention_bwd": 3, "qk_norm_rope_bwd": 2}
_NO_LAUNCH = {"read_status"}


class _CountingExtension:
    """Proxy over the compiled module that counts kernel launches."""

    def __init__(self, ext):
        self._ext = ext

    def __getattr__(self, name):
        fn = getattr(self._ext, name)
        if name in _NO_LAUNCH or not callable(fn):
            return fn
        n = _MULTI_LAUNCH.get(name, 1)

        def call(*args, **kwargs):
            global LAUNCHES
            LAUNCHES += n
            return fn(*args, **kwargs)

        object.__setattr__(self, name, call)
        return call


def launches() -> int:
    return LAUNCHES


def _load():
    global _EXT, _EXT_ERR
    if _EXT is not None or _EXT_ERR is not None:
        return _EXT
    try:
        import importlib

        # MT_OPS_DEBUG=1: the debug-checks build (setup.py with MT_DEBUG_CHECKS=1)
        name = "meshtrain_b200.ops._C_debug" if os.environ.get("MT_OPS_DEBUG") == "1" else "meshtrain_b200.ops._C"
        _EXT = _CountingExtension(importlib.import_module(name))
    except Exception as exc:  # pragma: no cover - depends on the build
        _EXT_ERR = f"{type(exc).__name__}: {exc}"
    return _EXT


def extension():
    """The compiled kernel module; raises if it is not built."""
    ext = _load()
    if ext is None:
        raise RuntimeError(
            "meshtrain_b200 CUDA extension is not built (python setup.py build_ext --inplace): " + str(_EXT_ERR))
    return ext


def extension_available() -> bool:
    return _load() is not None


def backend() -> str:
    return _BACKEND


def set_backend(name: str) -> None:
    """``custom`` (hand-written kernels on CUDA) or ``torch`` (PyTorch ops everywhere)."""
    global _BACKEND
    if name not in ("custom", "torch"):
        raise ValueError(f"unknown kernel backend {name!r}")
    _BACKEND = name


@contextmanager
def use_backend(name: str):
    prev = _BACKEND
    set_backend(name)
    try:
        yield
    finally:
        set_backend(prev)


def _custom(*tensors: torch.Tensor) -> bool:
    """True when this call must go to the CUDA kernels."""
    t = tensors[0]
    if not (t.is_cuda and _BACKEND == "custom"):
        return False
    if any(x is not None and x.dtype not in (torch.bfloat16, torch.int64, torch.float32) for x in tensors):
        return False
    if t.dtype != torch.bfloat16:
        return False
    extension()  # raise loudly if the kernels are missing on a CUDA host
    return True


_KERNEL_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _custom_float(t: torch.Tensor) -> bool:
    """``_custom`` for the operators whose kernels also take fp16 and fp32 (then ``_EXT`` is loaded).
    Their bindings check the arguments themselves: a small call is bound by its launch."""
    if not (t.is_cuda and _BACKEND == "custom" and t.dtype in _KERNEL_DTYPES):
        return False
    if _EXT is None:
        extension()
    return True


def _acc(t: torch.Tensor) -> torch.dtype:
    """Type the plain restatements compute in."""
    return torch.float64 if t.dtype == torch.float64 else torch.float32


def _require(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _vector(t: torch.Tensor, n: int, like: torch.Tensor, dtype: torch.dtype, name: str) -> torch.Tensor:
    """``t`` as a contiguous vector of ``n`` values of ``dtype`` on ``like``'s device."""
    _require(t.numel() == n and t.dtype == dtype and t.device == like.device,
             f"{name} must have {n} values of {dtype} on {like.device}, got {tuple(t.shape)} of {t.dtype} on {t.device}")
    return t.reshape(-1).contiguous()


def _mat(x: torch.Tensor) -> torch.Tensor:
    """2-D row-major view suitable for TMA: unit column stride, row stride a
    multiple of 8 elements (16 bytes), 16-byte aligned base.  Rows whose width
    is not a multiple of 8 are copied into a padded buffer (the padding is
    never read: tensor maps carry the logical width)."""
    x2 = x.reshape(-1, x.shape[-1])
    if x2.stride(-1) == 1 and x2.stride(0) % 8 == 0 and x2.stride(0) >= x2.shape[1] and x2.data_ptr() % 16 == 0:
        return x2
    rows, cols = x2.shape
    ld = (cols + 7) // 8 * 8
    buf = torch.empty(rows, ld, dtype=x2.dtype, device=x2.device)
    buf[:, :cols] = x2
    return buf[:, :cols]


# ----------------------------------------------------------------------------- linear

def linear(x: torch.Tensor, w: torch.Tensor, b: torch.Tensor | None = None, *, gelu: bool = False,
           residual: torch.Tensor | None = None):
    """y = x W^T + b [+ residual]; with ``gelu`` returns (gelu(h), h)."""
    if _custom(x, w):
        ext = extension()
        x2, w2 = _mat(x), _mat(w)
        M, N = x2.shape[0], w2.shape[0]
        out = torch.empty(M, N, device=x.device, dtype=torch.bfloat16)
        if gelu:
            h = torch.empty_like(out)
            ext.gemm(x2, False, w2, False, out, EPI_GELU, b, None, h, 0.0)
            return out.view(*x.shape[:-1], N), h.view(*x.shape[:-1], N)
        if residual is not None:
            ext.gemm(x2, False, w2, False, out, EPI_RESID, b, _mat(residual), None, 0.0)
        else:
            ext.gemm(x2, False, w2, False, out, EPI_BF16, b, None, None, 0.0)
        return out.view(*x.shape[:-1], N)
    y = F.linear(x, w, b)
    if gelu:
        return F.gelu(y), y
    if residual is not None:
        y = y + residual
    return y


def linear_dgrad(dy: torch.Tensor, w: torch.Tensor, *, gelu_pre: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """dx = dy W  (times gelu'(gelu_pre) when given: the GELU backward fused in).

    ``out`` (a contiguous [M, N] bf16 tensor, e.g. a row block of a larger
    buffer) receives the result directly instead of a new tensor.
    """
    if _custom(dy, w):
        ext = extension()
        dy2, w2 = _mat(dy), _mat(w)
        M, N = dy2.shape[0], w2.shape[1]
        if out is None:
            out = torch.empty(M, N, device=dy.device, dtype=torch.bfloat16)
        elif tuple(out.shape) != (M, N) or out.dtype != torch.bfloat16 or not out.is_contiguous():
            raise ValueError("linear_dgrad: out must be a contiguous bf16 [M, N] tensor")
        if gelu_pre is not None:
            ext.gemm(dy2, False, w2, True, out, EPI_DGELU, None, _mat(gelu_pre), None, 0.0)
        else:
            ext.gemm(dy2, False, w2, True, out, EPI_BF16, None, None, None, 0.0)
        return out.view(*dy.shape[:-1], N)
    dx = dy @ w
    if gelu_pre is not None:
        dx = dx * gelu_grad(gelu_pre)
    if out is not None:
        out.copy_(dx)
        return out
    return dx


# Deferred weight gradients: inside ``deferred_wgrad()`` the weight-gradient GEMMs
# and bias column sums go to one side stream per device, so they fill the SMs that
# the critical-path kernels (input-gradient GEMMs, attention) leave idle in their
# last waves.  They only accumulate into gradient buffers that nothing reads until
# the block ends, and the block's exit makes the current stream wait for them.
_WGRAD = threading.local()
_WGRAD_STREAMS: dict[int, torch.cuda.Stream] = {}


def _wgrad_stream(device: torch.device) -> torch.cuda.Stream:
    idx = device.index if device.index is not None else torch.cuda.current_device()
    st = _WGRAD_STREAMS.get(idx)
    if st is None:
        st = _WGRAD_STREAMS[idx] = torch.cuda.Stream(device=idx)
    return st


@contextmanager
def deferred_wgrad(enabled: bool = True, timer=None):
    """Run ``linear_wgrad_`` calls of the block on a side stream; join on exit.

    ``timer.side_work(stream)``, when given, is called before each side-stream
    GEMM is enqueued, so the caller can bracket that work with CUDA events and
    count it as busy time of the device.
    """
    outer = getattr(_WGRAD, "used", None)
    if not enabled or outer is not None or not torch.cuda.is_available():
        yield
        return
    _WGRAD.used = set()
    _WGRAD.timer = timer
    try:
        yield
    finally:
        used, _WGRAD.used, _WGRAD.timer = _WGRAD.used, None, None
        for idx in used:
            torch.cuda.current_stream(idx).wait_stream(_WGRAD_STREAMS[idx])


def wait_wgrad(device: torch.device) -> None:
    """The current stream waits for the weight gradients deferred so far on ``device``: called before
    memory that ``linear_wgrad_`` was given is written again (nothing to wait for outside ``deferred_wgrad``)."""
    if device.index in (getattr(_WGRAD, "used", None) or ()):
        torch.cuda.current_stream(device).wait_stream(_WGRAD_STREAMS[device.index])


def linear_wgrad_(dy: torch.Tensor, x: torch.Tensor, w_grad: torch.Tensor, b_grad: torch.Tensor | None = None) -> None:
    """w_grad += dy^T x (fp32 accumulate); b_grad += sum_t dy.

    Inside ``deferred_wgrad`` dy and x may still be read after the call: freeing them is safe, writing
    them again needs ``wait_wgrad`` first."""
    if _custom(dy, x) and w_grad.dtype == torch.float32:
        ext = extension()
        dy2, x2 = _mat(dy), _mat(x)
        used = getattr(_WGRAD, "used", None)
        if used is not None:
            side = _wgrad_stream(dy.device)
            side.wait_stream(torch.cuda.current_stream(dy.device))  # dy, x and the gradient buffers are ready
            timer = getattr(_WGRAD, "timer", None)
            if timer is not None:
                timer.side_work(side)
            with torch.cuda.stream(side):
                ext.gemm(dy2, True, x2, True, w_grad, EPI_F32, None, None, None, 1.0)
                if b_grad is not None:
                    ext.colsum_(dy2, b_grad)
            dy2.record_stream(side)  # the allocator keeps them until the side stream has read them
            x2.record_stream(side)
            used.add(side.device.index)
            return
        ext.gemm(dy2, True, x2, True, w_grad, EPI_F32, None, None, None, 1.0)
        if b_grad is not None:
            ext.colsum_(dy2, b_grad)
        return
    dy2, x2 = dy.reshape(-1, dy.shape[-1]), x.reshape(-1, x.shape[-1])
    if dy2.dtype == torch.bfloat16 and dy2.is_cuda:
        w_grad += (dy2.t() @ x2).to(w_grad.dtype)
    else:
        w_grad += (dy2.t().to(w_grad.dtype) @ x2.to(w_grad.dtype))
    if b_grad is not None:
        b_grad += dy2.to(b_grad.dtype).sum(0)


def gelu_grad(h: torch.Tensor) -> torch.Tensor:
    hf = h.float()
    cdf = 0.5 * (1.0 + torch.erf(hf / math.sqrt(2.0)))
    pdf = torch.exp(-0.5 * hf * hf) / math.sqrt(2.0 * math.pi)
    return (cdf + hf * pdf).to(h.dtype)


# SwiGLU: the fused gate/up weight stores rows in blocks of 32 = [16 gate | 16 up].

def interleave_gate_up(w_gate: torch.Tensor, w_up: torch.Tensor) -> torch.Tensor:
    F_, d = w_gate.shape
    g = w_gate.reshape(F_ // 16, 16, d)
    u = w_up.reshape(F_ // 16, 16, d)
    return torch.cat([g, u], dim=1).reshape(2 * F_, d)


def split_gate_up(raw: torch.Tensor):
    *lead, n2 = raw.shape
    r = raw.reshape(*lead, n2 // 32, 32)
    return r[..., :16].reshape(*lead, n2 // 2), r[..., 16:].reshape(*lead, n2 // 2)


def merge_gate_up(g: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
    *lead, f = g.shape
    return torch.cat([g.reshape(*lead, f // 16, 16), u.reshape(*lead, f // 16, 16)], dim=-1).reshape(*lead, 2 * f)


def swiglu_linear(x: torch.Tensor, w_gu: torch.Tensor):
    """(silu(x Wg^T) * (x Wu^T), raw) with the interleaved fused weight."""
    if _custom(x, w_gu):
        ext = extension()
        x2, w2 = _mat(x), _mat(w_gu)
        M, N2 = x2.shape[0], w2.shape[0]
        out = torch.empty(M, N2 // 2, device=x.device, dtype=torch.bfloat16)
        raw = torch.empty(M, N2, device=x.device, dtype=torch.bfloat16)
        ext.gemm(x2, False, w2, False, out, EPI_SWIGLU, None, None, raw, 0.0)
        return out.view(*x.shape[:-1], N2 // 2), raw.view(*x.shape[:-1], N2)
    raw = F.linear(x, w_gu)
    g, u = split_gate_up(raw)
    return F.silu(g) * u, raw


def swiglu_bwd(dout: torch.Tensor, raw: torch.Tensor) -> torch.Tensor:
    if _custom(dout, raw):
        return extension().swiglu_bwd(dout.contiguous(), raw.contiguous())
    g, u = split_gate_up(raw.float())
    sg = torch.sigmoid(g)
    d = dout.float()
    dg = d * u * (sg * (1 + g * (1 - sg)))
    du = d * g * sg
    return merge_gate_up(dg, du).to(raw.dtype)


# ----------------------------------------------------------------------------- norms

def layernorm(x: torch.Tensor, g: torch.Tensor, b: torch.Tensor, eps: float = 1e-5):
    """(y, mean, rstd) with fp32 statistics."""
    if _custom(x, g, b):
        y, mean, rstd = extension().layernorm_fwd(x.contiguous(), g, b, eps)
        return y, mean, rstd
    xf = x.float()
    mean = xf.mean(-1)
    var = xf.var(-1, unbiased=False)
    rstd = torch.rsqrt(var + eps)
    y = F.layer_norm(x, (x.shape[-1],), g, b, eps)
    return y, mean.reshape(-1), rstd.reshape(-1)


def layernorm_bwd(dy, x, g, mean, rstd, dres, dg_acc, db_acc):
    if _custom(dy, x, g) and dg_acc.dtype == torch.float32:
        return extension().layernorm_bwd(dy.contiguous(), x.contiguous(), g, mean, rstd,
                                         None if dres is None else dres.contiguous(), dg_acc, db_acc)
    d = x.shape[-1]
    xf = x.reshape(-1, d).float()
    dyf = dy.reshape(-1, d).float()
    xh = (xf - mean[:, None]) * rstd[:, None]
    wdy = dyf * g.float()
    m1 = wdy.mean(-1, keepdim=True)
    m2 = (wdy * xh).mean(-1, keepdim=True)
    dx = rstd[:, None] * (wdy - m1 - xh * m2)
    dg_acc += (dyf * xh).sum(0).to(dg_acc.dtype)
    db_acc += dyf.sum(0).to(db_acc.dtype)
    if dres is not None:
        dx = dx + dres.reshape(-1, d).float()
    return dx.to(x.dtype).reshape(x.shape)


def rmsnorm(x: torch.Tensor, g: torch.Tensor, eps: float = 1e-5):
    if _custom(x, g):
        y, rstd = extension().rmsnorm_fwd(x.contiguous(), g, eps)
        return y, rstd
    xf = x.float()
    rstd = torch.rsqrt(xf.pow(2).mean(-1) + eps)
    y = (xf * rstd[..., None] * g.float()).to(x.dtype)
    return y, rstd.reshape(-1)


def rmsnorm_bwd(dy, x, g, rstd, dres, dg_acc):
    if _custom(dy, x, g) and dg_acc.dtype == torch.float32:
        return extension().rmsnorm_bwd(dy.contiguous(), x.contiguous(), g, rstd,
                                       None if dres is None else dres.contiguous(), dg_acc)
    d = x.shape[-1]
    xf = x.reshape(-1, d).float()
    dyf = dy.reshape(-1, d).float()
    xh = xf * rstd[:, None]
    wdy = dyf * g.float()
    m2 = (wdy * xh).mean(-1, keepdim=True)
    dx = rstd[:, None] * (wdy - xh * m2)
    dg_acc += (dyf * xh).sum(0).to(dg_acc.dtype)
    if dres is not None:
        dx = dx + dres.reshape(-1, d).float()
    return dx.to(x.dtype).reshape(x.shape)


# ----------------------------------------------------------------------------- embedding

def embedding(ids: torch.Tensor, tok: torch.Tensor, pos: torch.Tensor | None, seq_len: int) -> torch.Tensor:
    """tok[ids] (+ pos[t % seq_len]); returns [T, d]."""
    flat = ids.reshape(-1)
    if _custom(tok) and flat.is_cuda:
        return extension().embedding_fwd(flat, tok, pos, seq_len)
    out = F.embedding(flat, tok)
    if pos is not None:
        T = flat.shape[0]
        out = out + pos[torch.arange(T, device=flat.device) % seq_len]
    return out


def embedding_bwd_(ids, dy, tok_grad, pos_grad, seq_len: int) -> None:
    flat = ids.reshape(-1)
    dy2 = dy.reshape(-1, dy.shape[-1])
    if _custom(dy2) and tok_grad.dtype == torch.float32:
        extension().embedding_bwd(flat, dy2.contiguous(), tok_grad, pos_grad, seq_len)
        return
    tok_grad.index_add_(0, flat, dy2.to(tok_grad.dtype))
    if pos_grad is not None:
        T = flat.shape[0]
        pos_grad.index_add_(0, torch.arange(T, device=flat.device) % seq_len, dy2.to(pos_grad.dtype))


# ----------------------------------------------------------------------------- rope

def rope_(qk: torch.Tensor, seq_len: int, heads: int, head_dim: int, theta: float, inverse: bool = False) -> None:
    """Rotate-half RoPE in place on the first ``heads`` heads of each row of qk [T, >=heads*hd]."""
    if _custom(qk):
        extension().rope_(qk, seq_len, heads, head_dim, theta, inverse)
        return
    T = qk.shape[0]
    half = head_dim // 2
    pos = (torch.arange(T, device=qk.device) % seq_len).float()
    inv = theta ** (-2.0 * torch.arange(half, device=qk.device).float() / head_dim)
    ang = pos[:, None] * inv[None]
    cs, sn = torch.cos(ang), torch.sin(ang)
    if inverse:
        sn = -sn
    v = qk[:, : heads * head_dim].reshape(T, heads, head_dim).float()
    x1, x2 = v[..., :half], v[..., half:]
    o1 = x1 * cs[:, None] - x2 * sn[:, None]
    o2 = x2 * cs[:, None] + x1 * sn[:, None]
    qk[:, : heads * head_dim] = torch.cat([o1, o2], -1).reshape(T, heads * head_dim).to(qk.dtype)


def _check_heads(name, qkv, q_gain, k_gain, seq_len, heads, kv_heads, head_dim, theta, eps) -> int:
    _require(qkv.dim() == 2 and heads >= 0 and kv_heads >= 0 and heads + kv_heads >= 1 and head_dim >= 2
             and head_dim % 2 == 0 and qkv.shape[1] >= (heads + kv_heads) * head_dim,
             f"{name}: qkv must be [rows, >= (heads + kv_heads) * head_dim] with an even head_dim")
    _require(seq_len >= 1 and theta > 0 and eps >= 0, f"{name}: needs seq_len >= 1, theta > 0 and eps >= 0")
    for g, what in ((q_gain, "q_gain"), (k_gain, "k_gain")):
        _require(tuple(g.shape) == (head_dim,) and g.dtype == qkv.dtype and g.device == qkv.device,
                 f"{name}: {what} must be [head_dim] of qkv's dtype and device")
    return (heads + kv_heads) * head_dim


def _out_rows(name, out, like, rows, cols):
    """``out`` checked as a row-major [rows, >= cols] matrix, or a new one as the kernels lay it out."""
    if out is None:
        ld = (cols + 7) // 8 * 8
        return torch.empty(rows, ld, dtype=like.dtype, device=like.device)[:, :cols]
    _require(out.dim() == 2 and out.shape[0] == rows and out.shape[1] >= cols and out.stride(1) == 1
             and (rows < 2 or out.stride(0) >= cols) and out.dtype == like.dtype and out.device == like.device,
             f"{name}: out must be [rows, >= {cols}] row-major of the input's dtype and device")
    return out[:, :cols]


def _gain_rows(q_gain, k_gain, heads, kv_heads, dt):
    return torch.cat([q_gain.to(dt).expand(heads, -1), k_gain.to(dt).expand(kv_heads, -1)])


def _rope_angles(rows, seq_len, head_dim, theta, dt, device):
    """(cos, sin) [rows, 1, head_dim / 2]; the angles in fp64 (an fp32 angle is off by 4e-3 at position 1e5)."""
    half = head_dim // 2
    inv = theta ** (torch.arange(half, device=device, dtype=torch.float64) * (-2.0 / head_dim))
    ang = (torch.arange(rows, device=device) % seq_len).double()[:, None] * inv
    return ang.cos().to(dt)[:, None], ang.sin().to(dt)[:, None]


def qk_norm_rope(qkv, q_gain, k_gain, seq_len: int, heads: int, kv_heads: int, head_dim: int, theta: float,
                 eps: float = 1e-5, out: torch.Tensor | None = None) -> torch.Tensor:
    """RMS norm of every query and key head of each row of ``qkv``, then rotate-half RoPE, in one pass.

    ``qkv`` [T, >= (heads + kv_heads) * head_dim] holds the query heads, then the key heads (columns
    behind them are not read); row t has position t % seq_len.  Each head is scaled by
    ``(mean(x^2) + eps)^-1/2`` times ``q_gain`` / ``k_gain`` [head_dim] and rotated as ``rope_`` does.
    The kernels take head dimensions that are multiples of 16 up to 256 and refuse others.
    Returns [T, (heads + kv_heads) * head_dim], in ``out`` when given, which must not overlap ``qkv``:
    that is what the backward needs.  On CUDA an ``out`` has its rows on 16-byte boundaries, with a leading
    dimension that is a multiple of 8 (so in the losses below); inputs of any layout are taken, copied first
    where their rows are not so.
    """
    if _custom_float(qkv):
        return _EXT.qk_norm_rope_fwd(qkv, q_gain, k_gain, seq_len, heads, kv_heads, head_dim, theta, eps, out)
    cols = _check_heads("qk_norm_rope", qkv, q_gain, k_gain, seq_len, heads, kv_heads, head_dim, theta, eps)
    T = qkv.shape[0]
    res = _out_rows("qk_norm_rope", out, qkv, T, cols)
    dt, half = _acc(qkv), head_dim // 2
    x = qkv[:, :cols].to(dt).reshape(T, -1, head_dim)
    u = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * _gain_rows(q_gain, k_gain, heads, kv_heads, dt)
    cs, sn = _rope_angles(T, seq_len, head_dim, theta, dt, qkv.device)
    a, b = u[..., :half], u[..., half:]
    res.copy_(torch.cat([a * cs - b * sn, b * cs + a * sn], -1).reshape(T, cols))
    return res


def qk_norm_rope_bwd(dqk, qkv, q_gain, k_gain, seq_len: int, heads: int, kv_heads: int, head_dim: int, theta: float,
                     dq_gain: torch.Tensor, dk_gain: torch.Tensor, eps: float = 1e-5,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient of ``qk_norm_rope``: returns that of ``qkv``'s query and key columns, and adds the gains'
    to ``dq_gain`` / ``dk_gain`` (fp32 [head_dim]; beside fp64 rows, which have no kernel, fp64 too), which may be one tensor.

    ``dqk`` [T, >= (heads + kv_heads) * head_dim] is the gradient of the result.  ``out`` may be ``dqk``
    itself (columns behind the heads stay as they are) or memory that does not overlap the inputs.
    Equal inputs give equal bits.
    """
    if _custom_float(qkv):
        return _EXT.qk_norm_rope_bwd(dqk, qkv, q_gain, k_gain, seq_len, heads, kv_heads, head_dim, theta, dq_gain,
                                     dk_gain, eps, out)
    cols = _check_heads("qk_norm_rope_bwd", qkv, q_gain, k_gain, seq_len, heads, kv_heads, head_dim, theta, eps)
    T = qkv.shape[0]
    _require(dqk.dim() == 2 and dqk.shape[0] == T and dqk.shape[1] >= cols and dqk.dtype == qkv.dtype
             and dqk.device == qkv.device, f"qk_norm_rope_bwd: dqk must be [rows, >= {cols}] of qkv's dtype and device")
    for g, what in ((dq_gain, "dq_gain"), (dk_gain, "dk_gain")):
        _require(tuple(g.shape) == (head_dim,) and g.dtype in (torch.float32, _acc(qkv)) and g.device == qkv.device
                 and g.is_contiguous(), f"qk_norm_rope_bwd: {what} must be contiguous torch.float32 [head_dim]")
    res = _out_rows("qk_norm_rope_bwd", out, qkv, T, cols)
    dt, half = _acc(qkv), head_dim // 2
    x = qkv[:, :cols].to(dt).reshape(T, -1, head_dim)
    dy = dqk[:, :cols].to(dt).reshape(T, -1, head_dim)
    cs, sn = _rope_angles(T, seq_len, head_dim, theta, dt, qkv.device)
    a, b = dy[..., :half], dy[..., half:]
    du = torch.cat([a * cs + b * sn, b * cs - a * sn], -1)
    r = torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    dgain = (du * x * r).sum(0)
    dq_gain += dgain[:heads].sum(0)
    dk_gain += dgain[heads:].sum(0)
    w = du * _gain_rows(q_gain, k_gain, heads, kv_heads, dt)
    dx = r * (w - x * r * (w * x * r).mean(-1, keepdim=True))
    res.copy_(dx.reshape(T, cols))
    return res


# ----------------------------------------------------------------------------- dropout

_U32 = 0xFFFFFFFF


def _signed64(v: int) -> int:
    return v - (1 << 64) if v >= 1 << 63 else v


def _mul32(a: torch.Tensor, m: int):
    """(high, low) 32-bit words of a * m for 32-bit values held in int64."""
    return (a * (m >> 16) + ((a * (m & 0xFFFF)) >> 16)) >> 16, (a * m) & _U32


def _keep_mask(shape, cut: int, seed: int, offset, device) -> torch.Tensor:
    """The elements ``dropout`` keeps: 16 bits each of Philox4x32-10 (Salmon, Moraes, Dror, Shaw,
    "Parallel random numbers: as easy as 1, 2, 3", 2011) at counter (element // 8, offset), key ``seed``."""
    n = math.prod(shape)
    g = torch.arange((n + 7) // 8, device=device)
    off = torch.as_tensor(_signed64(offset) if isinstance(offset, int) else offset, dtype=torch.int64, device=device)
    zero = torch.zeros_like(g)
    c = [g & _U32, g >> 32, zero + (off & _U32), zero + ((off >> 32) & _U32)]
    k0, k1 = seed & _U32, seed >> 32
    for _ in range(10):
        (h0, l0), (h1, l1) = _mul32(c[0], 0xD2511F53), _mul32(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & _U32, (k1 + 0xBB67AE85) & _U32
    words = torch.stack(c, -1)
    bits = torch.stack([words & 0xFFFF, words >> 16], -1).reshape(-1)[:n]
    return (bits >= cut).reshape(shape)


def dropout(x: torch.Tensor, p: float, seed: int, offset, residual: torch.Tensor | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """``residual + keep * x / (1 - p)``, the mask ``keep`` a function of (seed, offset, element index).

    No mask is stored: the same call on the gradient of the result is the backward with respect to
    ``x`` (the residual's gradient is the result's), and a recomputed forward repeats the mask.  ``p``
    is taken to the nearest 1/65536, and the scale is the inverse of that exact keep probability.
    ``seed`` and ``offset`` are 64-bit: one seed per run, another offset for every use of it.  ``offset``
    may be a one-element int64 tensor on x's device, read when the kernel runs, so that a captured graph
    draws another mask at each replay.  ``out`` may be ``x`` or ``residual``; it is contiguous, and on
    CUDA starts on a 16-byte boundary.  Dropped elements add exactly 0, whatever ``x`` holds there.
    """
    cut = round(p * 65536) if 0.0 <= p < 1.0 else 65536
    _require(cut < 65536, f"dropout: p must be in [0, 1) and round below 1, got {p}")
    on_device = isinstance(offset, torch.Tensor)
    _require(0 <= seed < 1 << 64 and (on_device or 0 <= offset < 1 << 64),
             "dropout: seed and offset must be 64-bit unsigned integers")
    if _custom_float(x):
        return _EXT.dropout(x, cut, _signed64(seed), 0 if on_device else _signed64(offset),
                            offset if on_device else None, residual, out)
    _require(not on_device or (offset.numel() == 1 and offset.dtype == torch.int64 and offset.device == x.device),
             "dropout: an offset tensor must be one int64 on x's device")
    for t, what in ((residual, "residual"), (out, "out")):
        _require(t is None or (t.shape == x.shape and t.dtype == x.dtype and t.device == x.device),
                 f"dropout: {what} must have x's shape, dtype and device")
    _require(out is None or out.is_contiguous(), "dropout: out must be contiguous")
    dt = _acc(x)
    keep = _keep_mask(x.shape, cut, seed, offset.reshape(()) if on_device else offset, x.device)
    y = torch.where(keep, x.to(dt) * (65536 / (65536 - cut)), 0.0)
    if residual is not None:
        y = residual.to(dt) + y
    return y.to(x.dtype) if out is None else out.copy_(y)


# ----------------------------------------------------------------------------- attention

def attention(q, k, v, *, causal: bool = True, scale: float | None = None):
    """Flash attention over [B, S, H, hd] views (GQA when k/v have fewer heads).

    Returns (o [B,S,Hq,hd] contiguous, lse [B,Hq,S] fp32).
    """
    from meshtrain_b200.ops import attention_impl

    return attention_impl.forward(q, k, v, causal=causal, scale=scale)


def attention_bwd(dout, q, k, v, o, lse, *, causal: bool = True, scale: float | None = None, out=None):
    """Returns (dq, dk, dv) with the shapes of q, k, v (written into ``out`` views when given)."""
    from meshtrain_b200.ops import attention_impl

    return attention_impl.backward(dout, q, k, v, o, lse, causal=causal, scale=scale, out=out)


# ----------------------------------------------------------------------------- loss

def cross_entropy_chunk_(logits: torch.Tensor, vocab: int, targets: torch.Tensor, loss_sum: torch.Tensor,
                         loss_scale: float, grad_scale: float) -> None:
    """In place: logits[:, :vocab] -> (softmax - onehot) * grad_scale; loss_sum += sum ce * loss_scale."""
    if _custom(logits) and targets.is_cuda:
        extension().cross_entropy_(logits, vocab, targets.reshape(-1), loss_sum, loss_scale, grad_scale)
        return
    lg = logits[:, :vocab].float()
    tg = targets.reshape(-1)
    lse = torch.logsumexp(lg, -1)
    valid = (tg >= 0) & (tg < vocab)
    tgc = tg.clamp(0, vocab - 1)
    ce = (lse - lg.gather(1, tgc[:, None])[:, 0]) * valid
    loss_sum += ce.sum() * loss_scale
    grad = torch.softmax(lg, -1)
    grad[torch.arange(lg.shape[0], device=lg.device), tgc] -= 1.0
    grad *= (grad_scale * valid.float())[:, None]
    logits[:, :vocab] = grad.to(logits.dtype)


def _check_logits(name, logits, vocab, targets):
    _require(logits.dim() == 2 and 1 <= vocab <= logits.shape[1] and logits.is_floating_point(),
             f"{name}: logits must be [rows, >= vocab]")
    return _vector(targets, logits.shape[0], logits, torch.int64, f"{name}: targets")


def _plain_logprobs(logits, vocab, tg):
    dt = _acc(logits)
    lg = logits[:, :vocab].to(dt)
    m = lg.nan_to_num(-math.inf, math.inf, -math.inf).amax(-1)
    s = torch.exp(lg - torch.where(m == -math.inf, 0.0, m)[:, None]).sum(-1)
    valid = (tg >= 0) & (tg < vocab)
    lp = (lg.gather(1, tg.clamp(0, vocab - 1)[:, None])[:, 0] - m) - s.log()
    lp = torch.where((m == -math.inf) & (s == 0), -math.inf, lp)
    return torch.where(valid, lp, 0.0), torch.stack([m, s], -1)


def _plain_dlogits(logits, vocab, tg, stats, dlogps, res):
    lg = logits[:, :vocab].to(_acc(logits))
    m, s = stats.view(-1, 2).unbind(-1)
    at = tg.clamp(0, vocab - 1)[:, None]
    up = torch.where((tg == at[:, 0]) & ~((m == -math.inf) & (s == 0)), dlogps, 0.0)
    d = -torch.exp(lg - torch.where(m == -math.inf, 0.0, m)[:, None]) / s[:, None]
    d.scatter_add_(1, at, torch.ones_like(up)[:, None])
    res.copy_(torch.where((up == 0)[:, None], 0.0, d * up[:, None]))
    return res


def token_logprobs(logits: torch.Tensor, vocab: int, targets: torch.Tensor):
    """(logps [T], stats [T, 2]), fp32: the log probability of each row's target, and the row's maximum m
    and sum of exp(x - m), which the backward takes (log-sum-exp = m + log of the sum).

    ``logits`` [T, >= vocab] as the LM head's GEMM leaves them.  A target outside [0, vocab) marks a row
    without a token: logp 0.  A row whose logits are all -inf has m = logp = -inf and the sum 0.
    """
    if _custom_float(logits):
        return _EXT.token_logprobs(logits, vocab, targets)
    tg = _check_logits("token_logprobs", logits, vocab, targets)
    return _plain_logprobs(logits, vocab, tg)


def token_logprobs_bwd(logits: torch.Tensor, vocab: int, targets: torch.Tensor, stats: torch.Tensor,
                       dlogps: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient of the logits from that of ``token_logprobs``'s logps: (onehot - softmax) * dlogps.
    ``stats`` is what ``token_logprobs`` returned for these logits.

    Rows without a token, rows whose ``dlogps`` is 0 and rows of nothing but -inf get zeros whatever they
    hold.  ``out`` may be ``logits`` (overwritten; on CUDA only rows as ``qk_norm_rope`` writes them);
    otherwise a new matrix, whose rows are padded to a multiple of 8 columns as the LM head's GEMMs take
    them.  Returns its first ``vocab`` columns.
    """
    if _custom_float(logits):
        return _EXT.token_logprobs_bwd(logits, vocab, targets, stats, dlogps, out)
    tg = _check_logits("token_logprobs_bwd", logits, vocab, targets)
    T, dt = logits.shape[0], _acc(logits)
    stats = _vector(stats, 2 * T, logits, dt, "token_logprobs_bwd: stats")
    dlogps = _vector(dlogps, T, logits, dt, "token_logprobs_bwd: dlogps")
    res = _out_rows("token_logprobs_bwd", out, logits, T, vocab)
    return _plain_dlogits(logits, vocab, tg, stats, dlogps, res)


def policy_loss_chunk(logits: torch.Tensor, vocab: int, targets: torch.Tensor, old_logps: torch.Tensor,
                      advantages: torch.Tensor, weights: torch.Tensor | None = None, *,
                      ref_logps: torch.Tensor | None = None, clip_low: float = 0.2, clip_high: float = 0.2,
                      kl_coef: float = 0.0, grad_scale: float = 1.0, out: torch.Tensor | None = None):
    """Clipped policy loss of sampled tokens with a KL term, forward and backward in one pass over the logits.

    Per row, with logp the log probability of its target and rho = exp(logp - old_logps):

        loss = weights * (max(-A rho, -A clip(rho, 1 - clip_low, 1 + clip_high))
                          + kl_coef * (exp(d) - d - 1)),    A = advantages, d = ref_logps - logp

    ``weights`` carry the mask and the normalisation (mask / tokens for a mean over tokens; None: 1).
    A row of weight 0 or whose target is outside [0, vocab) has loss 0 and gradient 0 whatever it holds.
    Where both sides of the max are equal the gradient is the unclipped side's.  Returns (losses [T],
    logps [T], dlogits), the last the gradient of ``grad_scale * sum(losses)``; ``out`` as in
    ``token_logprobs_bwd``.  All per-row tensors are fp32 [T].
    """
    if _custom_float(logits):
        return _EXT.policy_loss(logits, vocab, targets, old_logps, advantages, weights, ref_logps, clip_low, clip_high,
                                kl_coef, grad_scale, out)
    name = "policy_loss_chunk"
    tg = _check_logits(name, logits, vocab, targets)
    T, dt = logits.shape[0], _acc(logits)
    old, adv, w, ref = (None if t is None else _vector(t, T, logits, dt, f"{name}: {n}") for t, n in (
        (old_logps, "old_logps"), (advantages, "advantages"), (weights, "weights"), (ref_logps, "ref_logps")))
    _require(0.0 <= clip_low <= 1.0 and clip_high >= 0.0, f"{name}: needs 0 <= clip_low <= 1 and clip_high >= 0")
    _require(kl_coef == 0.0 or ref is not None, f"{name}: a KL term needs ref_logps")
    if kl_coef == 0.0:
        ref = None
    res = _out_rows(name, out, logits, T, vocab)
    lp, stats = _plain_logprobs(logits, vocab, tg)
    valid = (tg >= 0) & (tg < vocab)
    lpd = lp.double()
    ratio = torch.exp(lpd - old)
    ratio = torch.where((adv == 0) & (ratio == math.inf), 0.0, ratio)  # A rho = 0, however large rho is
    free, bound = -adv * ratio, -adv * ratio.clamp(1.0 - clip_low, 1.0 + clip_high)
    loss = torch.maximum(free, bound)
    d = torch.where((free >= bound) | free.isnan(), free, 0.0)
    if ref is not None:
        back = ref - lpd
        loss = loss + kl_coef * torch.where(back == math.inf, math.inf, torch.expm1(back) - back)
        d = d - kl_coef * torch.expm1(back)
    if w is not None:
        valid = valid & (w != 0)
        loss, d = loss * w, d * w
    loss = torch.where(valid, loss, 0.0).to(dt)
    dlogps = torch.where(valid, d * grad_scale, 0.0).to(dt)
    return loss, lp, _plain_dlogits(logits, vocab, tg, stats, dlogps, res)


def preference_loss(logps: torch.Tensor, ref_logps: torch.Tensor, mask: torch.Tensor, beta: float = 0.1, *,
                    form: str = "sigmoid", label_smoothing: float = 0.0, grad_scale: float = 1.0):
    """Preference loss of pairs of answers from the log ratios of their tokens, and its gradient.

    ``logps`` and ``ref_logps`` [2 P, S] fp32 are the tokens' log probabilities under the trained and the
    reference model; rows 2i and 2i + 1 are pair i's preferred and rejected answer; ``mask`` [2 P, S]
    bool marks the tokens that count.  With r the masked sum of logps - ref_logps of a row and n its count:

        sigmoid:  h = beta (r_0 - r_1),  loss = -(1 - s) log sigma(h) - s log sigma(-h),  s = label_smoothing
        squared:  loss = (r_0 / n_0 - r_1 / n_1 - 1 / (2 beta))^2

    An empty row has r = 0 and no gradient.  Returns (losses [P], rewards [2 P] = beta r, dlogps [2 P, S],
    the gradient of ``grad_scale * sum(losses)``).  Masked tokens are not looked at.
    """
    _require(form in ("sigmoid", "squared"), f"preference_loss: unknown form {form!r} (sigmoid, squared)")
    if _custom_float(logps):
        return _EXT.preference_loss(logps, ref_logps, mask, beta, label_smoothing, form == "squared", grad_scale)
    dt = _acc(logps)
    _require(logps.dim() == 2 and logps.shape[0] % 2 == 0 and logps.dtype == dt,
             "preference_loss: logps must be fp32 [2 pairs, S]")
    _require(beta > 0 and 0.0 <= label_smoothing <= 1.0, "preference_loss: needs beta > 0 and 0 <= label_smoothing <= 1")
    _require(form == "sigmoid" or label_smoothing == 0.0, "preference_loss: label_smoothing is the sigmoid form's")
    for t, n, want in ((ref_logps, "ref_logps", dt), (mask, "mask", torch.bool)):
        _require(t.shape == logps.shape and t.dtype == want and t.device == logps.device,
                 f"preference_loss: {n} must be {want} with logps's shape and device")
    r = torch.where(mask, logps.double() - ref_logps, 0.0).sum(-1)
    r0, r1 = r[0::2], r[1::2]
    if form == "sigmoid":
        h = beta * (r0 - r1)
        # a side of weight 0 is left out: it may be infinite
        losses = sum((-w * F.logsigmoid(g) for w, g in ((1 - label_smoothing, h), (label_smoothing, -h)) if w),
                     torch.zeros_like(h))
        up = beta * (label_smoothing - torch.sigmoid(-h))
        up = torch.stack([up, -up], -1).reshape(-1)
    else:
        n = mask.sum(-1).clamp(min=1)
        gap = r0 / n[0::2] - r1 / n[1::2] - 0.5 / beta
        losses = gap.square()
        up = torch.stack([2 * gap, -2 * gap], -1).reshape(-1) / n
    dlogps = torch.where(mask, (up * grad_scale)[:, None], 0.0).to(dt)
    return losses.to(dt), (beta * r).to(dt), dlogps


# ----------------------------------------------------------------------------- optimizer

def adam_(p, g, m, v, p_lowp, *, lr, beta1, beta2, eps, weight_decay, decoupled, step, grad_scale=1.0):
    """Fused Adam/AdamW on flat fp32 buffers (torch.optim semantics); optional bf16 copy-out."""
    bc1 = 1.0 - beta1 ** step
    bc2 = 1.0 - beta2 ** step
    if p.is_cuda and _BACKEND == "custom":
        extension().adam_(p, g, m, v, p_lowp, lr, beta1, beta2, eps, weight_decay, decoupled, bc1, bc2, grad_scale)
        return
    gg = g * grad_scale if grad_scale != 1.0 else g
    if decoupled:
        p.mul_(1 - lr * weight_decay)
    elif weight_decay:
        gg = gg + weight_decay * p
    m.mul_(beta1).add_(gg, alpha=1 - beta1)
    v.mul_(beta2).addcmul_(gg, gg, value=1 - beta2)
    denom = (v.sqrt() / math.sqrt(bc2)).add_(eps)
    p.addcdiv_(m, denom, value=-lr / bc1)
    if p_lowp is not None:
        p_lowp.copy_(p)


def read_status(device: int = 0) -> int:
    """Non-zero if a kernel on ``device`` gave up a bounded wait since the last call."""
    return int(extension().read_status(device))


def read_checks() -> int:
    """Failed-check codes (``kErrCheck*``) of the debug-checks build since the last call on the
    current device; always 0 with the release build."""
    return int(extension().read_checks())


def debug_checks_built() -> bool:
    return bool(extension().debug_checks_built())
