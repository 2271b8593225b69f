"""Dense products in 8-bit integers: the serving form of a trained dense layer.

``Int8Dense`` holds a weight matrix as 8-bit integers with one scale per output channel, laid out once.
``x @ w`` quantises the rows of ``x`` on the way (one scale per row) and multiplies in integers;
``EventArray(spk) @ w`` takes spikes as 0 and 1, without any rounding of the input.  The definition,
kept to the bit: ``scale = float32(max|.| / 127)``, ``q = round(value / scale)`` (ties to even, exact
quotient), ``out = (sum qx qw) * scale_x * scale_w``.  Kernels: ``csrc/int8_*.cu``.

There is no gradient: train in float (``EventLinear``), then quantise.
"""
from __future__ import annotations

from functools import lru_cache
from typing import Optional

import torch

from . import _lib
from ._lib import call_on, lib
from .event import EventArray, _require_cuda

__all__ = ['Int8Dense', 'Int8Rows', 'quantize_rows', 'int8_matmul']

_TYPES = {torch.float32: _lib.T_F32, torch.bfloat16: _lib.T_BF16, torch.float16: _lib.T_F16}
_MATMULS = (torch.Tensor.__matmul__, torch.Tensor.matmul, torch.matmul)
_EVENTS = {torch.bool: _lib.T_EVENT8, torch.uint8: _lib.T_EVENT8, torch.float32: _lib.T_EVENT32}


@lru_cache(maxsize=4096)
def _workspace_bytes(given: bool, m: int, n_pre: int, n_post: int) -> int:
    """Workspace of a product over ``given`` 8-bit rows, or of one that quantises them."""
    return (lib().bsx_int8_matmul_workspace_bytes if given else lib().bsx_int8_dense_workspace_bytes)(m, n_pre, n_post)


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
    if len(lead) != 1:
        t = t.reshape(-1, n) if t.numel() else t.new_empty((0, n))
    if n > 1 and t.stride(-1) != 1:
        t = t.contiguous()
    return t, kinds[t.dtype], lead


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
    call_on(x2.get_device(), lib().bsx_int8_quantize_rows, x2.data_ptr(), fmt, x2.stride(0), m, n, q.data_ptr(),
            scale.data_ptr())
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
        self.q = torch.empty((self.shape[1], lib().bsx_int8_row_bytes(self.shape[0])), dtype=torch.int8, device=w.device)
        self.scale = torch.empty(self.shape[1], dtype=torch.float32, device=w.device)
        call_on(w.get_device(), lib().bsx_int8_quantize_weights, w.data_ptr(), _TYPES[w.dtype], *self.shape,
                self.q.data_ptr(), self.scale.data_ptr())

    def dequantize(self) -> torch.Tensor:
        """The float32 weights that the integers stand for."""
        return (self.q[:, :self.shape[0]].to(torch.float32) * self.scale.unsqueeze(-1)).t().contiguous()

    def __rmatmul__(self, x):
        if isinstance(x, (torch.Tensor, EventArray)):
            return int8_matmul(x, self)
        return NotImplemented

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        # ``tensor @ w`` comes here first; sent on, it would reach __rmatmul__ only after an error was raised and dropped
        if func in _MATMULS and not kwargs and len(args) == 2 and isinstance(args[1], cls):
            return int8_matmul(*args)
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
    if out_dtype is not None:
        kind = out_dtype
        if kind not in _TYPES:
            raise TypeError(f'out_dtype must be float32, bfloat16 or float16, got {kind}')
    m, dev = data.shape[0], data.get_device()
    if dev != w.q.get_device():
        raise ValueError(f'input is on {data.device}, the weights on {w.q.device}')
    out = data.new_empty(lead + (n_post,)) if kind is data.dtype else data.new_empty(lead + (n_post,), dtype=kind)
    if rows:
        n = _workspace_bytes(True, m, n_pre, n_post)
        ws = data.new_empty(n) if n else None
        call_on(dev, lib().bsx_int8_matmul, data.data_ptr(), x.scale.data_ptr(), w.q.data_ptr(), w.scale.data_ptr(), m, n_pre,
                n_post, out.data_ptr(), _TYPES[kind], None if ws is None else ws.data_ptr(), n)
    else:
        n = _workspace_bytes(False, m, n_pre, n_post)
        ws = w.q.new_empty(n) if n else None
        call_on(dev, lib().bsx_int8_dense, data.data_ptr(), fmt, data.stride(0), w.q.data_ptr(), w.scale.data_ptr(), m, n_pre,
                n_post, out.data_ptr(), _TYPES[kind], None if ws is None else ws.data_ptr(), n)
    return out
