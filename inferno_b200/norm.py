"""Host-side mirror of the reference's ``LayerNorm``: normalisation over the last axis, forward and backward.

``LayerNorm::forward`` in the reference saves mean and inverse deviation of each row and attaches a backward node
(src/inferno/modules/layernorm.cpp:25-98; kernels src/inferno/cuda/cudalayernorm.cu:16-400).  Here both directions run on the
kernels of ``csrc/layer_norm.cuh`` through the C ABI: fp32 or bf16 rows of up to 32 KB, weight and bias of either type, fp32 sums.
"""
from __future__ import annotations

import torch

from . import _capi


def layer_norm_forward(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5):
    """(y, mean, rstd) with y = (x - mean) * rstd * weight + bias over the last axis of x; mean and rstd are fp32, one per row.

    x may be a view whose rows lie one pitch apart (a slice of a wider tensor); it is then read in place.  y is dense."""
    return _capi.host().layer_norm_forward(x, weight, bias, eps)


def layer_norm_backward(x, dy, mean, rstd, weight=None, need_dx=True, need_dw=True, need_db=True):
    """(dx, dw, db) of ``layer_norm_forward``; dw and db in weight's type (fp32 without one); what is not needed comes back as None.
    All three repeat bit for bit."""
    return _capi.host().layer_norm_backward(x, dy, mean, rstd, weight, need_dx, need_dw, need_db)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last axis of x; differentiable once (backward node in csrc/host_ops.cpp), a second derivative raises
    NotImplementedError."""
    return _capi.host().layer_norm(x, weight, bias, eps)


class LayerNorm(torch.nn.Module):
    """``layer_norm`` with learned weight and bias, under the parameter names of ``torch.nn.LayerNorm``."""

    def __init__(self, features: int, eps: float = 1e-5, bias: bool = True):
        super().__init__()
        self.eps = eps
        self.weight = torch.nn.Parameter(torch.ones(features))
        self.bias = torch.nn.Parameter(torch.zeros(features)) if bias else None

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)
