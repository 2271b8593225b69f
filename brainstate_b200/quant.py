"""Dense products in 8-bit integers: the serving form of a trained dense layer.

``Int8Dense`` holds a weight matrix as 8-bit integers with one scale per output channel, laid out once.
``x @ w`` quantises the rows of ``x`` on the way (one scale per row) and multiplies in integers;
``EventArray(spk) @ w`` takes spikes as 0 and 1, without any rounding of the input.  The definition,
kept to the bit: ``scale = float32(max|.| / 127)``, ``q = round(value / scale)`` (ties to even, exact
quotient), ``out = (sum qx qw) * scale_x * scale_w``.  Kernels: ``csrc/int8_*.cu``.

There is no gradient: train in float (``EventLinear``), then quantise.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._lib import check, lib, ptr
from .event import EventArray, _require_cuda

__all__ = ['Int8Dense', 'Int8Rows', 'quantize_rows', 'int8_matmul']

_TYPES = {torch.float32: _lib.T_F32, torch.bfloat16: _lib.T_BF16, torch.float16: _lib.T_F16}
_EVENTS = {torch.bool: _lib.T_EVENT8, torch.uint8: _lib.T_EVENT8, torch.float32: _lib.T_EVENT32}


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _rows(x, n: Optional[int]):
    """``(x as rows of dense entries, format, leading shape)``; ``n``: the row length wanted."""
    event = isinstance(x, EventArray)
    t = x.value if event else x
    if not isinstance(t, torch.Tensor):
        raise TypeError(f'expected a tensor or an EventArray, got {type(t).__name__}')
    _require_cuda(t, 'input')
    kinds = _EVENTS if event else _TYPES
    if t.dtype not in kinds:
        raise TypeError('spikes must be bool, uint8 or float32' if event else
                        'rows must be float32, bfloat16 or float16 (wrap spikes in EventArray)' + f', got {t.dtype}')
    if t.dim() < 1 or (n is not None and t.shape[-1] != n):
        raise ValueError(f'input has shape {tuple(t.shape)}, expected rows of {n}')
    if torch.is_grad_enabled() and t.requires_grad:
        raise RuntimeError('the 8-bit product has no gradient: call it under torch.no_grad(), or train with EventLinear')
    lead, n = tuple(t.shape[:-1]), t.shape[-1]
    if n == 0:
        raise ValueError('rows without entries cannot be quantised')
    x2 = t.reshape(-1, n) if t.numel() else t.new_empty((0 if 0 in lead else 1, n))
    if n > 1 and x2.stride(-1) != 1:
        x2 = x2.contiguous()
    return x2, kinds[t.dtype], lead


class Int8Rows:
    """Rows in 8 bits: ``q`` ``(rows, padded)`` int8 (zero beyond ``n``), ``scale`` ``(rows,)`` float32, ``lead`` the leading
    shape and ``dtype`` the type that products of them have by default.  Made by :func:`quantize_rows`; worth it where
    several matrices take the same input."""

    __slots__ = ('q', 'scale', 'n', 'lead', 'dtype')

    def __init__(self, q, scale, n, lead, dtype):
        self.q, self.scale, self.n, self.lead, self.dtype = q, scale, n, lead, dtype

    @property
    def shape(self):
        return self.lead + (self.n,)

    def dequantize(self) -> torch.Tensor:
        """The float32 values that the integers stand for."""
        return (self.q[:, :self.n].to(torch.float32) * self.scale.unsqueeze(-1)).reshape(self.shape)

    def __matmul__(self, w):
        return int8_matmul(self, w) if isinstance(w, Int8Dense) else NotImplemented


def quantize_rows(x) -> Int8Rows:
    """Rows of a float tensor (``EventArray``: spikes) in 8 bits with one scale each."""
    x2, fmt, lead = _rows(x, None)
    m, n = x2.shape
    q = torch.empty((m, lib().bsx_int8_row_bytes(n)), dtype=torch.int8, device=x2.device)
    scale = torch.empty(m, dtype=torch.float32, device=x2.device)
    with torch.cuda.device(x2.device):
        check(lib().bsx_int8_quantize_rows(ptr(x2), fmt, x2.stride(0), m, n, ptr(q), ptr(scale), _stream(x2)))
    return Int8Rows(q, scale, n, lead, torch.float32 if isinstance(x, EventArray) else x2.dtype)


class Int8Dense:
    """A dense ``(n_pre, n_post)`` weight matrix in 8 bits.

    ``weight``: float32, bfloat16 or float16 on the GPU.  ``q`` is ``(n_post, padded n_pre)`` int8 — a row
    per output channel, zero beyond ``n_pre`` — and ``scale`` ``(n_post,)`` float32.
    """

    def __init__(self, weight: torch.Tensor):
        _require_cuda(weight, 'weight')
        if weight.dim() != 2:
            raise ValueError(f'weight must be (n_pre, n_post), got {tuple(weight.shape)}')
        if weight.dtype not in _TYPES:
            raise TypeError(f'weight must be float32, bfloat16 or float16, got {weight.dtype}')
        if weight.shape[0] == 0:
            raise ValueError('a matrix without inputs cannot be quantised')
        w = weight.detach().contiguous()
        self.shape = (int(w.shape[0]), int(w.shape[1]))
        with torch.cuda.device(w.device):
            self.q = torch.empty((self.shape[1], lib().bsx_int8_row_bytes(self.shape[0])), dtype=torch.int8, device=w.device)
            self.scale = torch.empty(self.shape[1], dtype=torch.float32, device=w.device)
            check(lib().bsx_int8_quantize_weights(ptr(w), _TYPES[w.dtype], *self.shape, ptr(self.q), ptr(self.scale),
                                                  _stream(w)))

    def dequantize(self) -> torch.Tensor:
        """The float32 weights that the integers stand for."""
        return (self.q[:, :self.shape[0]].to(torch.float32) * self.scale.unsqueeze(-1)).t().contiguous()

    def __rmatmul__(self, x):
        if isinstance(x, (torch.Tensor, EventArray)):
            return int8_matmul(x, self)
        return NotImplemented


def int8_matmul(x, w: Int8Dense, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``x @ w``: ``x`` a float tensor, ``EventArray`` or :class:`Int8Rows` with rows of ``n_pre`` entries; leading
    dimensions are kept.  ``out_dtype`` (float32, bfloat16, float16) defaults to the type of ``x``, float32 for spikes.
    Bit-identical on every call."""
    if not isinstance(w, Int8Dense):
        raise TypeError(f'expected an Int8Dense, got {type(w).__name__}')
    n_pre, n_post = w.shape
    rows = isinstance(x, Int8Rows)
    if rows:
        if x.n != n_pre:
            raise ValueError(f'input has rows of {x.n}, expected {n_pre}')
        data, lead, kind = x.q, x.lead, x.dtype
    else:
        data, fmt, lead = _rows(x, n_pre)
        kind = torch.float32 if fmt >= _lib.T_EVENT8 else data.dtype
    kind = kind if out_dtype is None else out_dtype
    if kind not in _TYPES:
        raise TypeError(f'out_dtype must be float32, bfloat16 or float16, got {kind}')
    if data.device != w.q.device:
        raise ValueError(f'input is on {data.device}, the weights on {w.q.device}')
    m = data.shape[0]
    out = torch.empty((m, n_post), dtype=kind, device=data.device)
    with torch.cuda.device(data.device):
        if rows:
            n = lib().bsx_int8_matmul_workspace_bytes(m, n_pre, n_post)
            ws = torch.empty(n, dtype=torch.uint8, device=data.device) if n else None
            check(lib().bsx_int8_matmul(ptr(data), ptr(x.scale), ptr(w.q), ptr(w.scale), m, n_pre, n_post, ptr(out),
                                        _TYPES[kind], ptr(ws), n, _stream(data)))
        else:
            n = lib().bsx_int8_dense_workspace_bytes(m, n_pre, n_post)
            ws = torch.empty(n, dtype=torch.uint8, device=data.device)
            check(lib().bsx_int8_dense(ptr(data), fmt, data.stride(0), ptr(w.q), ptr(w.scale), m, n_pre, n_post, ptr(out),
                                       _TYPES[kind], ptr(ws), n, _stream(data)))
    return out.reshape(lead + (n_post,))
