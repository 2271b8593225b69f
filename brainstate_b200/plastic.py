"""Plastic synapses: weight matrices that learn while they are used.

The gated delta rule keeps a synaptic matrix ``S`` of shape ``(dk, dv)`` per batch row and value
head.  Every token (time step) first lets the matrix decay, then corrects its answer to the key
towards the value (an error-correcting Hebbian update), then answers the query::

    u_t = beta_t (v_t - e^{g_t} S_{t-1}^T k_t)
    S_t = e^{g_t} S_{t-1} + k_t u_t^T
    o_t = scale S_t^T q_t

``delta_rule`` runs whole sequences (chunked over 64 tokens on the tensor cores, differentiable),
``delta_rule_step`` one token with the state updated in place.  States are float32; sums and
everything the state depends on are held to 32-bit accuracy also for 16-bit inputs.  Keys should
have a norm of at most about 1 and ``beta`` lie in [0, 1] (the rule diverges where
``beta |k|^2 > 2``); ``g`` is at most 0, and ``-inf`` drops the state.  Kernels:
``csrc/plastic*.cu``.
"""
from __future__ import annotations

import struct
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import call_on, lib
from .event import _require_cuda

__all__ = ['delta_rule', 'delta_rule_step']

_TYPES = {torch.float32: _lib.T_F32, torch.bfloat16: _lib.T_BF16, torch.float16: _lib.T_F16}
_DESC = struct.Struct('=2q5if7Q15q')       # bsx_delta_t

# Sequences of at most this many tokens go token by token (one launch, the state read and written
# once, 1.3 us a token) instead of by chunks, whose cost does not depend on the tokens in them.  Measured
# with 16 heads of 128 x 128 in bfloat16: 1 row, 8 tokens 12.7 us against 14.0 us, 16 tokens 23.2 us
# against 14.0 us; 64 rows, 8 tokens 95 us against 157 us, 16 tokens 171 us against 158 us.
RECURRENT_TOKENS = 8


def _dense_rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 else t.contiguous()      # contiguous() leaves a dimension of one entry as it is


def _dense_like(t: torch.Tensor) -> torch.Tensor:
    """A new dense tensor of this shape and type.  From a dense tensor in two thirds of the host's time for a shape."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _describe(q, k, v, g, beta, initial, lengths, scale) -> bytes:
    B, T, Hk, dk = q.shape
    _, _, Hv, dv = v.shape
    (qb, qt, qh, _), (kb, kt, kh, _), (vb, vt, vh, _) = q.stride(), k.stride(), v.stride()
    return _DESC.pack(B, T, Hk, Hv, dk, dv, _TYPES[q.dtype], scale, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(),
                      beta.data_ptr(), 0 if initial is None else initial.data_ptr(),
                      0 if lengths is None else lengths.data_ptr(), qb, qt, qh, kb, kt, kh, vb, vt, vh,
                      *g.stride(), *beta.stride())


def _forward(q, k, v, g, beta, initial, lengths, scale):
    B, T, _, dk = q.shape
    _, _, Hv, dv = v.shape
    o = _dense_like(v)
    state = g.new_empty((B, Hv, dk, dv)) if initial is None else _dense_like(initial)
    d = _describe(q, k, v, g, beta, initial, lengths, scale)
    if T <= RECURRENT_TOKENS:
        call_on(v.get_device(), lib().bsx_delta_recurrent, d, o.data_ptr(), state.data_ptr())
    else:
        n = lib().bsx_delta_workspace_bytes(d)
        ws = g.new_empty(n // 4)
        call_on(v.get_device(), lib().bsx_delta_forward, d, o.data_ptr(), state.data_ptr(), ws.data_ptr(), n)
    return o, state


class _DeltaRule(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, v, g, beta, initial, lengths, scale):
        ctx.scale = scale
        ctx.save_for_backward(q, k, v, g, beta, initial, lengths)
        ctx.set_materialize_grads(False)
        return _forward(q, k, v, g, beta, initial, lengths, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, do, dstate):
        if do is None and dstate is None:
            return (None,) * 8
        q, k, v, g, beta, initial, lengths = ctx.saved_tensors
        # dense whatever the strides of the inputs
        dq, dk, dv, dg, dbeta = _dense_like(q), _dense_like(k), _dense_like(v), _dense_like(g), _dense_like(beta)
        do = v.new_zeros(v.shape) if do is None else do.contiguous()
        dstate = None if dstate is None else dstate.contiguous()
        dinitial = _dense_like(initial) if ctx.needs_input_grad[5] else None
        d = _describe(q, k, v, g, beta, initial, lengths, ctx.scale)
        n = lib().bsx_delta_backward_workspace_bytes(d)
        ws = g.new_empty(n // 4)
        call_on(v.get_device(), lib().bsx_delta_backward, d, do.data_ptr(), None if dstate is None else dstate.data_ptr(),
                dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dg.data_ptr(), dbeta.data_ptr(),
                None if dinitial is None else dinitial.data_ptr(), ws.data_ptr(), n)
        return dq, dk, dv, dg, dbeta, dinitial, None, None


def _fits(q, k, v, g, beta, state, lead: int) -> bool:
    """Whether the kernels take the arguments; ``lead`` is the number of dimensions before the heads."""
    try:
        qs, vs, gs, dev = q.shape, v.shape, g.shape, q.get_device()
        return (dev >= 0 and k.get_device() == dev and v.get_device() == dev and g.get_device() == dev
                and beta.get_device() == dev and q.dtype in _TYPES and k.dtype == q.dtype and v.dtype == q.dtype
                and g.dtype.is_floating_point and beta.dtype.is_floating_point and len(qs) == lead + 2
                and k.shape == qs and len(vs) == lead + 2 and vs[:lead] == qs[:lead] and gs == vs[:-1] and beta.shape == gs
                and qs[lead] > 0 and vs[lead] > 0 and vs[lead] % qs[lead] == 0 and 1 <= qs[-1] <= 128
                and 1 <= vs[-1] <= 4096
                and (state is None or (state.dtype == torch.float32 and state.get_device() == dev
                                       and state.shape == (qs[0], vs[lead], qs[-1], vs[-1]))))
    except AttributeError:
        return False


def _check(q, k, v, g, beta, state, lead: int):
    if not _fits(q, k, v, g, beta, state, lead):
        _refuse(q, k, v, g, beta, state, lead)


def _refuse(q, k, v, g, beta, state, lead: int):
    """Says what does not fit."""
    for name, t, dims in (('q', q, lead + 2), ('k', k, lead + 2), ('v', v, lead + 2), ('g', g, lead + 1),
                          ('beta', beta, lead + 1)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f'{name} must be a tensor')
        _require_cuda(t, name)
        if t.dim() != dims:
            raise ValueError(f'{name} has {t.dim()} dimensions, expected {dims}')
        if t.device != q.device:
            raise ValueError(f'{name} is on {t.device}, q on {q.device}')
    if q.dtype not in _TYPES:
        raise TypeError(f'q, k and v must be float32, bfloat16 or float16, got {q.dtype}')
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f'q, k and v must have one type, got {q.dtype}, {k.dtype} and {v.dtype}')
    for name, t in (('g', g), ('beta', beta)):
        if not t.dtype.is_floating_point:
            raise TypeError(f'{name} must be floating point, got {t.dtype}')
    if k.shape != q.shape:
        raise ValueError(f'q {tuple(q.shape)} and k {tuple(k.shape)} differ in shape')
    if v.shape[:lead] != q.shape[:lead]:
        raise ValueError(f'v {tuple(v.shape)} does not go with q {tuple(q.shape)}')
    if g.shape != v.shape[:-1] or beta.shape != v.shape[:-1]:
        raise ValueError(f'g {tuple(g.shape)} and beta {tuple(beta.shape)} must have the shape {tuple(v.shape[:-1])}')
    hk, dk = q.shape[-2:]
    hv, dv = v.shape[-2:]
    if hk < 1 or hv < 1 or hv % hk != 0:
        raise ValueError(f'{hv} value heads cannot share {hk} key heads evenly')
    if not 1 <= dk <= 128:
        raise ValueError(f'key size {dk} is outside 1 to 128')
    if not 1 <= dv <= 4096:
        raise ValueError(f'value size {dv} is outside 1 to 4096')
    if state is not None:
        if not isinstance(state, torch.Tensor):
            raise TypeError('state must be a tensor')
        _require_cuda(state, 'state')
        if state.dtype != torch.float32:
            raise TypeError(f'the state must be float32, got {state.dtype}')
        if tuple(state.shape) != (q.shape[0], hv, dk, dv):
            raise ValueError(f'the state has shape {tuple(state.shape)}, expected {(q.shape[0], hv, dk, dv)}')
        if state.device != q.device:
            raise ValueError(f'the state is on {state.device}, q on {q.device}')


def delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor, *,
               scale: Optional[float] = None, initial_state: Optional[torch.Tensor] = None,
               lengths: Optional[torch.Tensor] = None):
    """Sequences through plastic synapses.  Returns ``(o, state)``; differentiable (reverse mode, once).

    Parameters
    ----------
    q, k : ``(batch, tokens, k_heads, dk)``, float32, bfloat16 or float16, ``dk <= 128``.
    v : ``(batch, tokens, v_heads, dv)`` of the same type.  ``v_heads`` is a multiple of ``k_heads``;
        value head ``h`` uses key head ``h // (v_heads // k_heads)``.
    g, beta : ``(batch, tokens, v_heads)``: logarithm of the decay (``<= 0``) and learning rate.  Cast to float32.
    scale : factor of the outputs, ``dk ** -0.5`` by default.
    initial_state : ``(batch, v_heads, dk, dv)`` float32; zero by default.
    lengths : ``(batch,)`` integers on the device (not read by the host; clipped to ``[0, tokens]``).
        Tokens of a row from its length on are not read — they may hold anything — and their
        outputs and gradients are zero.

    ``o`` is ``(batch, tokens, v_heads, dv)`` of the inputs' type, ``state`` the float32 state after each
    row's last token.  Any strides are taken; a last dimension that is not dense is copied.  Results
    are the same on every call.
    """
    _check(q, k, v, g, beta, initial_state, 2)
    if lengths is not None:
        _require_cuda(lengths, 'lengths')
        if lengths.dtype not in (torch.int32, torch.int64):
            raise TypeError(f'lengths must be int32 or int64, got {lengths.dtype}')
        if tuple(lengths.shape) != (q.shape[0],):
            raise ValueError(f'lengths has shape {tuple(lengths.shape)}, expected {(q.shape[0],)}')
        if lengths.device != q.device:
            raise ValueError(f'lengths is on {lengths.device}, q on {q.device}')
        if lengths.dtype != torch.int32:
            lengths = lengths.clamp(0, q.shape[1]).to(torch.int32)
        lengths = lengths.contiguous()
    if g.dtype != torch.float32:
        g = g.to(torch.float32)
    if beta.dtype != torch.float32:
        beta = beta.to(torch.float32)
    if initial_state is not None:
        initial_state = initial_state.contiguous()
    args = (_dense_rows(q), _dense_rows(k), _dense_rows(v), g, beta, initial_state, lengths,
            q.shape[-1] ** -0.5 if scale is None else float(scale))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad
                                    or beta.requires_grad or (initial_state is not None and initial_state.requires_grad)):
        return _DeltaRule.apply(*args)
    return _forward(*args)


def delta_rule_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                    state: torch.Tensor, *, scale: Optional[float] = None) -> torch.Tensor:
    """One token for every row: ``q, k (batch, k_heads, dk)``, ``v (batch, v_heads, dv)``, ``g, beta (batch,
    v_heads)``.  ``state`` (dense float32) is updated in place; returns ``o (batch, v_heads, dv)``.

    Not differentiable, since the old state is gone: raises where a gradient would be recorded (use
    ``delta_rule`` with one token there).
    """
    if state is None:
        raise TypeError('state must be a tensor')
    _check(q, k, v, g, beta, state, 1)
    if not state.is_contiguous():
        raise ValueError('the state must be contiguous: it is updated in place')
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad
                                    or beta.requires_grad or state.requires_grad):
        raise RuntimeError('delta_rule_step updates the state in place and records no gradient: '
                           'use delta_rule, or call it under torch.no_grad()')
    (qb, qh, qc), (kb, kh, kc), (vb, vh, vc) = q.stride(), k.stride(), v.stride()
    if qc != 1 or kc != 1 or vc != 1:
        q, k, v = _dense_rows(q), _dense_rows(k), _dense_rows(v)
        (qb, qh, _), (kb, kh, _), (vb, vh, _) = q.stride(), k.stride(), v.stride()
    if g.dtype != torch.float32:
        g = g.to(torch.float32)
    if beta.dtype != torch.float32:
        beta = beta.to(torch.float32)
    (B, Hk, dk), (_, Hv, dv) = q.shape, v.shape
    o = _dense_like(v)
    (gb, gh), (bb, bh) = g.stride(), beta.stride()
    at = state.data_ptr()
    d = _DESC.pack(B, 1, Hk, Hv, dk, dv, _TYPES[q.dtype], dk ** -0.5 if scale is None else scale, q.data_ptr(), k.data_ptr(),
                   v.data_ptr(), g.data_ptr(), beta.data_ptr(), at, 0, qb, 0, qh, kb, 0, kh, vb, 0, vh, gb, 0, gh, bb, 0, bh)
    call_on(v.get_device(), lib().bsx_delta_recurrent, d, o.data_ptr(), at)
    if not state.is_inference():       # such tensors have no version: nothing was recorded with them
        torch.autograd.graph.increment_version(state)
    return o
