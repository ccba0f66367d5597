"""Gated feed-forward block, ``act(x Wg^T) * (x Wu^T)`` times ``Wd^T`` plus a residual, as one node (kernels:
``csrc/gated_ffn.cu``; node: ``csrc/binding_block.cpp``).

CUDA tensors in bf16 of widths that are multiples of 8, and in fp32 of widths that the narrow layers' kernels take (inputs and
the middle multiples of 64, outputs of 4, at most 1,024), run the kernels.  Anything else — CPU tensors, other types and widths,
tracing, autocast, ``torch.func`` — is the same block as ``torch.nn.functional`` operations."""
from __future__ import annotations

from typing import Optional

import torch
from torch.nn import functional as F

from . import _cabi
from .linear import linear, plain_call

_ACTIVATIONS = {"silu": F.silu, "gelu": F.gelu, "relu": F.relu}


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                       activation: str = "silu", residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``(act(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T (+ residual)`` for ``x`` [..., in], ``w_gate`` and ``w_up`` [mid, in],
    ``w_down`` [out, mid], ``residual`` [..., out] and ``activation`` "silu", "gelu" (exact) or "relu".

    In bf16 the activation and its product with the up projection are taken from fp32 sums, as is the residual's addition;
    what the gradients need of the two projections is kept
    with 16 bits of their sums (6 bytes for a pair)."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(_ACTIVATIONS)}; got {activation!r}")
    if w_gate.dim() != 2 or w_up.shape != w_gate.shape or w_down.dim() != 2 or w_down.shape[1] != w_gate.shape[0] or \
            x.dim() < 1 or x.shape[-1] != w_gate.shape[1]:
        raise ValueError(f"x must be [..., in], w_gate and w_up [mid, in], w_down [out, mid]; got {tuple(x.shape)}, "
                         f"{tuple(w_gate.shape)}, {tuple(w_up.shape)}, {tuple(w_down.shape)}")
    if residual is not None and residual.shape != x.shape[:-1] + w_down.shape[:1]:
        raise ValueError(f"residual must be {tuple(x.shape[:-1] + w_down.shape[:1])}; got {tuple(residual.shape)}")
    if x.is_cuda and plain_call(x, w_gate, w_up, w_down, residual):
        y = _cabi.native().gated_feed_forward(x, w_gate, w_up, w_down, activation, residual)
        if y is not None:
            return y
    h = _ACTIVATIONS[activation](linear(x, w_gate, None)) * linear(x, w_up, None)
    y = linear(h, w_down, None)
    return y if residual is None else y + residual


class GatedFeedForward(torch.nn.Module):
    """``module(x, residual)`` with three learnt weights and no biases: ``gate`` and ``up`` [ffn_size, hidden_size], ``down``
    [hidden_size, ffn_size]."""

    def __init__(self, hidden_size: int, ffn_size: int, activation: str = "silu"):
        super().__init__()
        if activation not in _ACTIVATIONS:
            raise ValueError(f"activation must be one of {', '.join(_ACTIVATIONS)}; got {activation!r}")
        self.activation = activation
        self.gate = torch.nn.Parameter(torch.empty(ffn_size, hidden_size))
        self.up = torch.nn.Parameter(torch.empty(ffn_size, hidden_size))
        self.down = torch.nn.Parameter(torch.empty(hidden_size, ffn_size))
        for weight in (self.gate, self.up, self.down):
            torch.nn.init.normal_(weight, std=weight.shape[1] ** -0.5)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        return gated_feed_forward(x, self.gate, self.up, self.down, self.activation, residual)

    def extra_repr(self) -> str:
        return f"{self.gate.shape[1]}, {self.gate.shape[0]}, activation={self.activation!r}"
