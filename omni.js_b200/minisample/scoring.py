"""Scoring a [B, V] block of logits on the GPU: log-probabilities of given ids
with the entropy and the top alternatives of each row, their gradient, and
distillation from a teacher's top values (ms_logprobs, ms_logprobs_backward,
ms_distill in include/minisample.h, which says what each output is for every
kind of row).  Sampler's methods of the same names call these functions.

The reference returns ids only (src/generation.js:71-81): no counterpart.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _native as N
from .sampler import _written

_DTYPES = {torch.float32: N.MS_F32, torch.bfloat16: N.MS_BF16, torch.float16: N.MS_F16}
_KINDS = {"logits": N.MS_TEACHER_LOGITS, "logprobs": N.MS_TEACHER_LOGPROBS}


class LogProbs(NamedTuple):
    """Outputs of Sampler.logprobs; those not asked for are None."""

    logprobs: Optional[torch.Tensor]      # fp32, the tokens' shape
    entropy: Optional[torch.Tensor]       # fp32 [B]
    top_ids: Optional[torch.Tensor]       # int32 [B, top_n]
    top_logprobs: Optional[torch.Tensor]  # fp32 [B, top_n]
    row_max: Optional[torch.Tensor]       # fp64 [B], for logprobs_backward
    row_sum: Optional[torch.Tensor]       # fp64 [B]


# ---------------------------------------------------------------- argument checks
def _block(s, x, what="logits"):
    """(dtype, B, V, row stride) of a [B, V] block on the sampler's device."""
    dtype = _DTYPES.get(x.dtype) if isinstance(x, torch.Tensor) and x.is_cuda else None
    if dtype is None or x.dim() != 2:
        raise ValueError(f"{what} must be a [B, V] float32, bfloat16 or float16 CUDA tensor")
    B, V = x.shape
    ld, col = x.stride()
    if col != 1 and V > 1:
        raise ValueError(f"{what} must have unit column stride")
    if B <= 1:
        ld = V
    elif ld < V:
        raise ValueError(f"{what} must have a row stride of at least V (an expanded block has its rows on one another)")
    if x.get_device() != s.device_index:
        raise ValueError(f"{what} is on cuda:{x.get_device()}, the sampler on cuda:{s.device_index}")
    return dtype, B, V, ld


def _no_tangent(x):
    """Refuses a dual tensor: the calls have no forward-mode derivatives, and read
    the primal by its address."""
    if isinstance(x, torch.Tensor) and forward_ad.unpack_dual(x).tangent is not None:
        raise ValueError("logits have a tangent: the scoring calls have no forward-mode derivatives")


def _rows(t, name, x, dtype, shape):
    """Checks a small per-row argument: type, shape, device; contiguous."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.get_device() != x.get_device():
        raise ValueError(f"{name} must be a {dtype} tensor on {x.device}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _tokens(tokens, x):
    """(contiguous tokens or None, their number a row)."""
    if tokens is None:
        return None, 0
    if not isinstance(tokens, torch.Tensor) or tokens.dim() not in (1, 2) or tokens.shape[0] != x.shape[0]:
        raise ValueError("tokens must be a [B] or [B, n] int32 tensor")
    n = 1 if tokens.dim() == 1 else tokens.shape[1]
    if n == 0:
        raise ValueError("tokens must have at least one id a row (None for no tokens)")
    return _rows(tokens, "tokens", x, torch.int32, tokens.shape), n


def _grad_out(s, x, out):
    if out is None:
        return torch.empty_like(x, memory_format=torch.contiguous_format)
    _block(s, out, "out")
    if out.dtype != x.dtype or out.shape != x.shape:
        raise ValueError("out must have the logits' shape and type")
    return out


def _p(t):
    return None if t is None else t.data_ptr()


def _on(s, stream, tensors, call):
    """`call` on `stream`: what it allocates belongs to that stream, and what it
    reads is not reused by another one before it is done."""
    if stream.device.index != s.device_index:
        raise ValueError(f"stream is on {stream.device}, the sampler on cuda:{s.device_index}")
    with torch.cuda.stream(stream):
        r = call()
    for t in tensors:
        if t is not None:
            t.record_stream(stream)
    return r


# the current stream's handle without the Stream object around it, where torch has that
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _current(s):
    # handle 0 is the legacy default stream, which the C ABI knows as 1
    return _raw_stream(s.device_index) or 1


# ---------------------------------------------------------------- log-probabilities
def _logprobs(s, x, tokens, temperature, top_n, entropy, stats):
    dtype, B, V, ld = _block(s, x)
    tok, n = _tokens(tokens, x)
    if not 0 <= top_n <= N.MS_SCORE_MAX:
        raise ValueError(f"top_n must be in [0, {N.MS_SCORE_MAX}]")
    dev = x.device
    lp = torch.empty(tokens.shape, dtype=torch.float32, device=dev) if n else None
    ent = torch.empty(B, dtype=torch.float32, device=dev) if entropy else None
    ids = torch.empty((B, top_n), dtype=torch.int32, device=dev) if top_n else None
    top = torch.empty((B, top_n), dtype=torch.float32, device=dev) if top_n else None
    mx = torch.empty(B, dtype=torch.float64, device=dev) if stats else None
    sm = torch.empty(B, dtype=torch.float64, device=dev) if stats else None
    out = N.MsScores(_p(lp), _p(ent), _p(ids), _p(top), _p(mx), _p(sm))
    s._check(s._L.ms_logprobs(s._ctx, x.data_ptr(), dtype, B, V, ld, float(temperature), _p(tok), n, top_n,
                              ctypes.byref(out), _current(s)))
    return LogProbs(lp, ent, ids, top, mx, sm)


class _LogProbsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, s, tokens, temperature, top_n, entropy, stats):
        o = _logprobs(s, x, tokens, temperature, top_n, entropy, True)
        ctx.save_for_backward(x, tokens, o.row_max, o.row_sum, o.entropy)
        ctx.s, ctx.temperature = s, temperature
        ctx.set_materialize_grads(False)
        if not stats:  # the backward pass's, not the caller's
            o = o._replace(row_max=None, row_sum=None)
        ctx.mark_non_differentiable(*(t for t in (o.top_ids, o.top_logprobs, o.row_max, o.row_sum) if t is not None))
        return tuple(o)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_lp, g_ent, *_):
        x, tokens, mx, sm, ent = ctx.saved_tensors
        if g_lp is None and g_ent is None:
            return (None,) * 7
        dx = logprobs_backward(ctx.s, x, tokens, mx, sm, g_lp, g_ent, ent if g_ent is not None else None,
                               temperature=ctx.temperature)
        return (dx,) + (None,) * 6


def logprobs(s, logits, tokens=None, *, temperature=1.0, top_n=0, entropy=False, stats=False, stream=None):
    if stream is not None:
        return _on(s, stream, (logits, tokens),
                   lambda: logprobs(s, logits, tokens, temperature=temperature, top_n=top_n, entropy=entropy,
                                    stats=stats))
    _no_tangent(logits)
    if (isinstance(logits, torch.Tensor) and logits.requires_grad and torch.is_grad_enabled()
            and (tokens is not None or entropy)):  # the outputs that carry gradients
        return LogProbs(*_LogProbsFn.apply(logits, s, tokens, temperature, top_n, entropy, stats))
    return _logprobs(s, logits, tokens, temperature, top_n, entropy, stats)


def logprobs_backward(s, logits, tokens, row_max, row_sum, g_logprobs=None, g_entropy=None, entropy=None, *,
                      temperature=1.0, out=None, stream=None):
    if stream is not None:
        return _on(s, stream, (logits, tokens, row_max, row_sum, g_logprobs, g_entropy, entropy, out),
                   lambda: logprobs_backward(s, logits, tokens, row_max, row_sum, g_logprobs, g_entropy, entropy,
                                             temperature=temperature, out=out))
    _no_tangent(logits)
    dtype, B, V, ld = _block(s, logits)
    tok, n = _tokens(tokens, logits)
    row_max = _rows(row_max, "row_max", logits, torch.float64, (B,))
    row_sum = _rows(row_sum, "row_sum", logits, torch.float64, (B,))
    if g_logprobs is not None:
        if n == 0:
            raise ValueError("g_logprobs needs tokens")
        g_logprobs = _rows(g_logprobs, "g_logprobs", logits, torch.float32, tokens.shape)
    if g_entropy is not None:
        g_entropy = _rows(g_entropy, "g_entropy", logits, torch.float32, (B,))
        entropy = _rows(entropy, "entropy", logits, torch.float32, (B,))
    dx = _grad_out(s, logits, out)
    s._check(s._L.ms_logprobs_backward(s._ctx, logits.data_ptr(), dtype, B, V, ld, float(temperature), _p(tok),
                                       n, row_max.data_ptr(), row_sum.data_ptr(), _p(entropy), _p(g_logprobs),
                                       _p(g_entropy), dx.data_ptr(), dx.stride(0), _current(s)))
    if out is not None:
        _written(out)
    return dx


# ---------------------------------------------------------------- distillation
def _distill(s, x, ids, values, weight, temperature, kind, want_loss, dx):
    dtype, B, V, ld = _block(s, x)
    if kind not in _KINDS:
        raise ValueError("kind must be 'logits' or 'logprobs'")
    if not isinstance(ids, torch.Tensor) or ids.dim() != 2:
        raise ValueError("teacher_ids must be a [B, K] int32 tensor")
    K = ids.shape[1]
    ids = _rows(ids, "teacher_ids", x, torch.int32, (B, K))
    values = _rows(values, "teacher_values", x, torch.float32, (B, K))
    if weight is not None:
        weight = _rows(weight, "weight", x, torch.float32, (B,))
    loss = torch.empty(B, dtype=torch.float32, device=x.device) if want_loss else None
    s._check(s._L.ms_distill(s._ctx, x.data_ptr(), dtype, B, V, ld, float(temperature), ids.data_ptr(),
                             values.data_ptr(), K,
                             _KINDS[kind], _p(weight), _p(loss), _p(dx), dx.stride(0) if dx is not None else 0,
                             _current(s)))
    return loss


class _DistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, s, ids, values, temperature, kind):
        loss = _distill(s, x, ids, values, None, temperature, kind, True, None)
        ctx.save_for_backward(x, ids, values)
        ctx.s, ctx.temperature, ctx.kind = s, temperature, kind
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x, ids, values = ctx.saved_tensors
        dx = _grad_out(ctx.s, x, None)
        _distill(ctx.s, x, ids, values, g, ctx.temperature, ctx.kind, False, dx)
        return (dx,) + (None,) * 5


def distill_loss(s, logits, teacher_ids, teacher_values, *, temperature=1.0, kind="logprobs", stream=None):
    if stream is not None:
        return _on(s, stream, (logits, teacher_ids, teacher_values),
                   lambda: distill_loss(s, logits, teacher_ids, teacher_values, temperature=temperature, kind=kind))
    _no_tangent(logits)
    if isinstance(logits, torch.Tensor) and logits.requires_grad and torch.is_grad_enabled():
        return _DistillFn.apply(logits, s, teacher_ids, teacher_values, temperature, kind)
    return _distill(s, logits, teacher_ids, teacher_values, None, temperature, kind, True, None)


def distill_grad(s, logits, teacher_ids, teacher_values, weight=None, *, temperature=1.0, kind="logprobs", out=None,
                 stream=None):
    if stream is not None:
        return _on(s, stream, (logits, teacher_ids, teacher_values, weight, out),
                   lambda: distill_grad(s, logits, teacher_ids, teacher_values, weight, temperature=temperature,
                                        kind=kind, out=out))
    _no_tangent(logits)
    _block(s, logits)
    dx = _grad_out(s, logits, out)
    loss = _distill(s, logits, teacher_ids, teacher_values, weight, temperature, kind, True, dx)
    if out is not None:
        _written(out)
    return loss, dx
