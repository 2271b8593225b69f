"""A layer of plastic synapses: its weight matrix is state and learns by the gated delta rule.

``DeltaSynapse`` holds one float32 matrix per batch row and value head and follows the calling
convention of the other stateful layers: ``init_state(batch_size)``, then one time step per
``update`` — or a whole sequence per ``run``.  See :mod:`brainstate_b200.plastic` for the rule.
"""
from __future__ import annotations

from typing import Optional

import torch

from ..plastic import delta_rule, delta_rule_step
from ._event_fixedprob import _device
from ._module import Module, Size
from ._state import State

__all__ = ['DeltaSynapse']


class DeltaSynapse(Module):
    """``in_size`` and ``out_size`` are the key and value sizes of one head (the last dimension counts),
    ``v_heads`` defaults to ``k_heads``."""

    __module__ = 'brainstate_b200.nn'

    def __init__(self, in_size: Size, out_size: Size, k_heads: int = 1, v_heads: Optional[int] = None,
                 scale: Optional[float] = None, name: Optional[str] = None, device=None):
        super().__init__(name=name)
        self.in_size = in_size
        self.out_size = out_size
        self.k_heads = int(k_heads)
        self.v_heads = self.k_heads if v_heads is None else int(v_heads)
        if self.k_heads < 1 or self.v_heads < 1 or self.v_heads % self.k_heads != 0:
            raise ValueError(f'{self.v_heads} value heads cannot share {self.k_heads} key heads evenly')
        self.scale = self.in_size[-1] ** -0.5 if scale is None else float(scale)
        self.device = _device(device)
        self.state = State(None)

    def init_state(self, batch_size: int):
        """Sets every matrix to zero."""
        self.state.value = torch.zeros((batch_size, self.v_heads, self.in_size[-1], self.out_size[-1]),
                                       dtype=torch.float32, device=self.device)

    reset_state = init_state

    def _ready(self):
        if self.state.value is None:
            raise RuntimeError('call init_state(batch_size) first')
        return self.state.value

    def update(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor,
               beta: torch.Tensor) -> torch.Tensor:
        """One time step: ``q, k (batch, k_heads, in)``, ``v (batch, v_heads, out)``, ``g, beta (batch, v_heads)``.
        The matrices are updated in place; where a gradient is recorded they are replaced instead, so
        that it reaches back through the steps."""
        state = self._ready()
        if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, g, beta, state)):
            o, new = delta_rule(*(t.unsqueeze(1) for t in (q, k, v, g, beta)), scale=self.scale, initial_state=state)
            self.state.value = new
            return o.squeeze(1)
        return delta_rule_step(q, k, v, g, beta, state, scale=self.scale)

    def run(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
            lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
        """A sequence, ``(batch, tokens, ...)``, continued from the state and leaving the state behind it."""
        o, self.state.value = delta_rule(q, k, v, g, beta, scale=self.scale, initial_state=self._ready(),
                                         lengths=lengths)
        return o
