"""``RMSNorm``: ``torch.nn.RMSNorm`` over the last dimension with the same parameter and ``state_dict`` key, alone, with the
residual addition in front of it, and with its result in 8 bits (kernels: ``csrc/rms_norm.cu``; node: ``csrc/binding_block.cpp``).

CUDA tensors in fp32 or bf16, weight of the same type, rows of up to 16,384 values run the kernels.  Anything else — CPU tensors,
other types, longer rows, no weight, tracing, autocast, ``torch.func`` — is ``torch.nn.functional.rms_norm`` itself, but for
:func:`rms_norm_quantized`, which raises."""
from __future__ import annotations

from typing import Optional

import torch

from . import _cabi
from .linear import plain_call, unobserved


def _eps(x: torch.Tensor, eps: Optional[float]) -> float:
    """``torch.nn.RMSNorm``'s default: the machine epsilon of the type that rows of ``x``'s are computed in."""
    return eps if eps is not None else torch.finfo(torch.float64 if x.dtype == torch.float64 else torch.float32).eps


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: Optional[float] = None) -> torch.Tensor:
    """``x / sqrt(mean(x ** 2) + eps) * weight`` over the last dimension."""
    if x.is_cuda and weight is not None and plain_call(x, weight):
        out = _cabi.native().add_rms_norm(x, None, weight, _eps(x, eps), False)
        if out is not None:
            return out[0]
    return torch.nn.functional.rms_norm(x, (x.shape[-1],), weight, eps)


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: Optional[float] = None,
                 want_sum: bool = True):
    """``(rms_norm(x + residual), x + residual)`` in one kernel each way.  The kernel's norm is that of the sum before it is
    rounded to the tensors' type.  The second is None when ``want_sum`` is false and nothing else needs it."""
    if x.is_cuda and weight is not None and plain_call(x, residual, weight):
        out = _cabi.native().add_rms_norm(x, residual, weight, _eps(x, eps), want_sum)
        if out is not None:
            return out
    x = x + residual
    return rms_norm(x, weight, eps), x


def rms_norm_quantized(x: torch.Tensor, weight: torch.Tensor, eps: Optional[float] = None,
                       residual: Optional[torch.Tensor] = None):
    """``(values, scales, sum)``: the norm of ``x`` (plus ``residual``) as ``float8_e4m3fn`` values of ``x``'s shape and one fp32
    scale a row, ``values * scales[..., None]`` standing for it, and ``x + residual`` (None without a residual).

    A row's scale is its largest magnitude / 448, at least 2^-126; a row with a NaN or an infinity has a NaN scale.  For
    inference: it raises where a gradient would be recorded, and for whatever the kernels do not cover."""
    for t in (x, weight, residual):
        if t is not None and not t.is_cuda:
            raise RuntimeError("rms_norm_quantized needs CUDA tensors (no CPU fallback)")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise RuntimeError("rms_norm_quantized has no gradient: call it under torch.no_grad()")
    if x.dtype not in (torch.float32, torch.bfloat16) or weight.dtype != x.dtype or \
            (residual is not None and residual.dtype != x.dtype):
        raise TypeError("x, weight and residual must all be float32 or all bfloat16")
    if weight.dim() != 1 or x.dim() < 1 or x.shape[-1] != weight.shape[0] or not 1 <= weight.shape[0] <= 16384:
        raise ValueError(f"x must be [..., hidden] for weight [hidden] of 1 to 16384 values; got {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual must have x's shape {tuple(x.shape)}; got {tuple(residual.shape)}")
    return _cabi.native().rms_norm_e4m3(x, weight, _eps(x, eps), residual)


class RMSNorm(torch.nn.RMSNorm):
    """Drop-in for ``nn.RMSNorm(hidden)``: same constructor, parameter and ``state_dict``."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if len(self.normalized_shape) == 1 and self.elementwise_affine and x.shape[-1:] == self.normalized_shape:
            return rms_norm(x, self.weight, self.eps)
        return super().forward(x)

    def add(self, x: torch.Tensor, residual: torch.Tensor, want_sum: bool = True):
        """``(self(x + residual), x + residual)``, one kernel each way unless somebody observes the module's calls."""
        if len(self.normalized_shape) == 1 and self.elementwise_affine and x.shape[-1:] == self.normalized_shape and \
                unobserved(self, RMSNorm):
            return add_rms_norm(x, residual, self.weight, self.eps, want_sum)
        x = x + residual
        return self(x), x
