"""Gated delta rule: the recurrence of a matrix-valued state.

For each head, with a state S of ``(dv, dk)`` and ``a[t] = exp(log_decay[t])``,

    S[t]   = a[t] S[t-1] + beta[t] (v[t] - a[t] S[t-1] k[t]) k[t]^T
    out[t] = scale S[t] q[t]

where the scan of ops.py has one number per channel.  The reference has no such operator.

* ``gated_delta``          -- differentiable, once (training)
* ``gated_delta_forward``  -- no autograd (a prompt: state in, state out)
* ``gated_delta_step``     -- token by token, the state updated in place (serving)

``q``, ``k``: (batch, seqlen, key_heads, dk); ``v``, ``out``: (batch, seqlen, heads, dv); ``log_decay``,
``beta``: (batch, seqlen, heads); contiguous CUDA tensors of one dtype, float32 / float16 / bfloat16.
``heads`` is a multiple of ``key_heads``: value head h uses key head ``h // (heads // key_heads)``.  States
are float32 (batch, heads, dv, dk).  dk: a multiple of 8 up to 128; dv: a multiple of 8; any seqlen >= 1.
q, k, v, states and ``out`` start on 16 bytes (in a step only q, k and the state); ``log_decay`` and ``beta``
may be slices that start anywhere, which a call over a sequence copies.

``log_decay`` is usually <= 0 and may be -inf: the state before that token counts no more, which is how a
sequence packed behind another begins (the gradient with respect to that ``log_decay`` is 0).

An infinity or a NaN spoils nothing before its token: in q it spoils that token's output, in v its column of
the outputs from there on, in k, log_decay or beta its head from there on, a reset or not.  So what pads a
batch behind a sequence does not reach its outputs; for its final state and its gradients it has to be
finite (beta 0 writes nothing).

Sums, states and the decay's running sums are held in 32 bits or more.  The products run on 16-bit tensor
cores with operands cut into exact parts: to 2^-16 relative where everything that comes out has 16 bits, to
2^-24 where a float32 tensor does (float32 data, or a state that is taken, returned or differentiated).
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib
from .checkpoint8 import dequantize8, quantize8
from .ops import (_EXT, DTYPE_CODES, NVTX, _aligned, _check_input, _fn, _launch, _once, _wanted,
                  nvtx_range)

__all__ = ["gated_delta", "gated_delta_forward", "gated_delta_step"]


def validate_delta(q, k, v, log_decay, beta, state=None, out=None) -> None:
    """Raise RuntimeError unless the tensors form a valid call."""
    for t, name in ((q, "q"), (k, "k"), (v, "v"), (log_decay, "log_decay"), (beta, "beta")):
        _check_input(t, name)
    validate_delta_layout(q, k, v, log_decay, beta, state, out)


def validate_delta_layout(q, k, v, log_decay, beta, state=None, out=None) -> None:
    """Device-independent checks (shapes, dtypes, devices); CPU-testable."""
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        if t.dim() != 4:
            raise RuntimeError(f"{name} must be 4-D (batch, seqlen, heads, channels), got {tuple(t.shape)}")
    b, l, h, dv = v.shape
    hk, dk = q.shape[2], q.shape[3]
    if q.shape != k.shape:
        raise RuntimeError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must have the same shape")
    if tuple(q.shape[:2]) != (b, l):
        raise RuntimeError(f"q {tuple(q.shape)} and v {tuple(v.shape)} must agree in batch and seqlen")
    if hk < 1 or h < 1 or h % hk:
        raise RuntimeError(f"heads of v ({h}) must be a positive multiple of the heads of q and k ({hk})")
    if l < 1:
        raise RuntimeError(f"seqlen must be >= 1 (got {l})")
    if dk % 8 or not 8 <= dk <= 128:
        raise RuntimeError(f"dk must be a multiple of 8 in [8, 128] (got {dk})")
    if dv % 8 or not 8 <= dv <= 65536:
        raise RuntimeError(f"dv must be a multiple of 8 in [8, 65536] (got {dv})")
    for t, name in ((log_decay, "log_decay"), (beta, "beta")):
        if tuple(t.shape) != (b, l, h):
            raise RuntimeError(f"{name} must have shape {(b, l, h)} (batch, seqlen, heads), got {tuple(t.shape)}")
    for t, name in ((q, "q"), (k, "k"), (log_decay, "log_decay"), (beta, "beta")):
        if t.dtype != v.dtype:
            raise RuntimeError(f"{name} dtype {t.dtype} must equal v dtype {v.dtype}")
        if t.device != v.device:
            raise RuntimeError(f"{name} and v must be on the same device")
    if state is not None:
        if not isinstance(state, torch.Tensor):
            raise RuntimeError("the state must be a torch.Tensor")
        if tuple(state.shape) != (b, h, dv, dk):
            raise RuntimeError(f"the state must have shape {(b, h, dv, dk)} (batch, heads, dv, dk), "
                               f"got {tuple(state.shape)}")
        if state.device != v.device:
            raise RuntimeError("the state must be on the device of v")
    if out is not None:
        if out.shape != v.shape or out.dtype != v.dtype or out.device != v.device:
            raise RuntimeError("out must match v in shape, dtype and device")
        if not out.is_contiguous():
            raise RuntimeError("out must be contiguous")


def _check_written(t: Optional[torch.Tensor], name: str) -> None:
    if t is not None and t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient, which writing it here would lose: detach it")


def _written(*tensors) -> None:
    # a backward pass that has saved one of these must notice
    for t in tensors:
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _sizes(q, v):
    b, l, h, dv = v.shape
    return b, l, q.shape[2], h, q.shape[3], dv


def _state_in(state: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if state is None else state.to(torch.float32).contiguous()


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _scale(scale: Optional[float], q: torch.Tensor) -> float:
    if scale is not None:
        return float(scale)
    return q.shape[-1] ** -0.5 if isinstance(q, torch.Tensor) and q.dim() and q.shape[-1] else 1.0


def _delta_workspace(q, v, wide: bool, backward: bool) -> torch.Tensor:
    # from torch's allocator at every call: it follows streams and graph
    # captures, so no two calls that may overlap share one
    nbytes = _fn("fpscan_delta_workspace_bytes")(*_sizes(q, v), DTYPE_CODES[v.dtype], 1 if wide else 0,
                                                 1 if backward else 0)
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=v.device)


def _tensors(*ts) -> bool:
    # what the compiled binding takes; anything else gets its error from validate_delta
    return _EXT is not None and all(t is None or isinstance(t, torch.Tensor) for t in ts)


def _run_forward(q, k, v, log_decay, beta, state, scale, return_state, out=None):
    if _tensors(q, k, v, log_decay, beta, state, out):
        return _EXT.delta_forward(q, k, v, log_decay, beta, _state_in(state), scale, return_state, out)
    _lib.load()
    validate_delta(q, k, v, log_decay, beta, state, out)
    _check_written(out, "out")
    state, log_decay, beta = _state_in(state), _aligned(log_decay), _aligned(beta)
    wide = state is not None or return_state
    given = out
    if out is None:
        out = torch.empty_like(v)
    b, l, hk, h, dk, dv = _sizes(q, v)
    final = torch.empty(b, h, dv, dk, dtype=torch.float32, device=v.device) if return_state else None
    ws = _delta_workspace(q, v, wide, False)
    _launch(v.get_device(), "fpscan_delta_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(),
            log_decay.data_ptr(), beta.data_ptr(), _ptr(state), out.data_ptr(), _ptr(final),
            b, l, hk, h, dk, dv, scale, DTYPE_CODES[v.dtype], 1 if wide else 0, ws.data_ptr(), ws.numel())
    _written(given)
    return out, final


def gated_delta_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                        beta: torch.Tensor, initial_state: Optional[torch.Tensor] = None,
                        scale: Optional[float] = None, return_state: bool = False,
                        out: Optional[torch.Tensor] = None
                        ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """The gated delta rule over a sequence (no autograd): ``out``, or ``(out, final_state)`` with
    ``return_state``.  ``scale`` defaults to ``dk ** -0.5``; ``initial_state`` to zero."""
    out, final = _run_forward(q, k, v, log_decay, beta, initial_state, _scale(scale, q), bool(return_state), out)
    return (out, final) if return_state else out


def gated_delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                     beta: torch.Tensor, state: torch.Tensor, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gated delta rule for the next token, or the next few (seqlen of the inputs), of each sequence:
    returns the outputs and updates ``state`` in place (float32, contiguous).  No autograd: in grad mode a state
    that requires a gradient, as the last one of ``gated_delta`` does, is refused (detach it)."""
    if not (isinstance(state, torch.Tensor) and state.is_cuda and state.dtype == torch.float32
            and state.is_contiguous()):
        raise RuntimeError("state must be a contiguous float32 CUDA tensor")
    if _tensors(q, k, v, log_decay, beta, out):
        return _EXT.delta_step(q, k, v, log_decay, beta, state, _scale(scale, q), out)
    validate_delta(q, k, v, log_decay, beta, state, out)
    _check_written(state, "state")
    _check_written(out, "out")
    given = out
    if out is None:
        out = torch.empty_like(v)
    _launch(v.get_device(), "fpscan_delta_step", q.data_ptr(), k.data_ptr(), v.data_ptr(),
            log_decay.data_ptr(), beta.data_ptr(), state.data_ptr(), out.data_ptr(), state.data_ptr(),
            *_sizes(q, v), _scale(scale, q), DTYPE_CODES[v.dtype])
    _written(state, given)
    return out


def gated_delta_backward(q, k, v, log_decay, beta, grad_out, initial_state=None, grad_final=None,
                         scale: Optional[float] = None, need_initial: bool = False):
    """Gradients of ``gated_delta_forward``: (dq, dk, dv, dlog_decay, dbeta, dinitial); ``grad_final`` is
    the gradient of the final state, ``dinitial`` is None unless ``need_initial``."""
    if _tensors(q, k, v, log_decay, beta, grad_out, initial_state, grad_final):
        return _EXT.delta_backward(q, k, v, log_decay, beta, grad_out, _state_in(initial_state),
                                   _state_in(grad_final), _scale(scale, q), need_initial)
    validate_delta(q, k, v, log_decay, beta, initial_state, grad_out)
    _check_input(grad_out, "grad_out")
    if grad_final is not None:
        validate_delta_layout(q, k, v, log_decay, beta, grad_final)
    state, grad_final = _state_in(initial_state), _state_in(grad_final)
    grad_final = None if grad_final is None else _aligned(grad_final)
    log_decay, beta, grad_out = _aligned(log_decay), _aligned(beta), _aligned(grad_out)
    b, l, hk, h, dk, dv = _sizes(q, v)
    wide = state is not None or grad_final is not None or need_initial
    grads = [torch.empty_like(t) for t in (q, k, v, log_decay, beta)]
    dinitial = torch.empty(b, h, dv, dk, dtype=torch.float32, device=v.device) if need_initial else None
    ws = _delta_workspace(q, v, wide, True)
    _launch(v.get_device(), "fpscan_delta_bwd", q.data_ptr(), k.data_ptr(), v.data_ptr(),
            log_decay.data_ptr(), beta.data_ptr(), _ptr(state), grad_out.data_ptr(), _ptr(grad_final),
            *(t.data_ptr() for t in grads), _ptr(dinitial), b, l, hk, h, dk, dv, _scale(scale, q),
            DTYPE_CODES[v.dtype], 1 if wide else 0, ws.data_ptr(), ws.numel())
    return (*grads, dinitial)


class GatedDelta(torch.autograd.Function):
    """Differentiable gated delta rule (the compiled binding has the same one).  Saves its inputs (q, k and v
    in 8 bits with ``checkpoint8``) and recomputes the chunks' states in the backward pass."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay, beta, state, scale, return_state, checkpoint8):
        with nvtx_range("fpscan.delta.forward"):
            out, final = _run_forward(q, k, v, log_decay, beta, state, scale, return_state)
        ctx.state_dtype = None if state is None else state.dtype
        state = _state_in(state)
        kept = [t for x in (q, k, v) for t in quantize8(x)] if checkpoint8 else [q, k, v]
        ctx.save_for_backward(*kept, log_decay, beta, state)
        ctx.scale, ctx.checkpoint8, ctx.dtype = scale, checkpoint8, v.dtype
        ctx.set_materialize_grads(False)
        return (out, final) if return_state else out

    @staticmethod
    def backward(ctx, grad_out, grad_final=None):
        *kept, log_decay, beta, state = ctx.saved_tensors
        if grad_out is None and grad_final is None:
            return (None,) * 9
        with nvtx_range("fpscan.delta.backward"):
            q, k, v = ([dequantize8(kept[i], kept[i + 1], ctx.dtype) for i in (0, 2, 4)]
                       if ctx.checkpoint8 else kept)
            grad_out = torch.zeros_like(v) if grad_out is None else grad_out.contiguous()
            *grads, dstate = gated_delta_backward(q, k, v, log_decay, beta, grad_out, state, grad_final,
                                                  ctx.scale, need_initial=ctx.needs_input_grad[5])
        if dstate is not None:
            dstate = dstate.to(ctx.state_dtype)
        return (*_once((*grads, dstate), "gated_delta"), None, None, None)


def gated_delta(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                beta: torch.Tensor, initial_state: Optional[torch.Tensor] = None,
                scale: Optional[float] = None, return_state: bool = False, checkpoint8: bool = False
                ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Differentiable gated delta rule over a sequence: ``out``, or ``(out, final_state)`` with
    ``return_state``; differentiable in all five inputs, the initial and the final state.
    ``checkpoint8=True`` keeps q, k and v for the backward pass, where one can follow, in 8 bits
    (``quantize8``): gradients are those of the rule at the values that these stand for."""
    scale, return_state, checkpoint8 = _scale(scale, q), bool(return_state), bool(checkpoint8)
    if not NVTX and _tensors(q, k, v, log_decay, beta, initial_state):
        out, final = _EXT.gated_delta(q, k, v, log_decay, beta, initial_state, scale, return_state, checkpoint8)
        return (out, final) if return_state else out
    checkpoint8 = checkpoint8 and _wanted(q, k, v, log_decay, beta, initial_state)
    return GatedDelta.apply(q, k, v, log_decay, beta, initial_state, scale, return_state, checkpoint8)
