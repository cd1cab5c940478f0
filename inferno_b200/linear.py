"""Host-side mirror of the reference's ``Linear`` for the two projections around attention.

``Linear::forward`` in the reference is ``matmul(x, W) + b`` with the weight stored ``[in, out]``
(src/inferno/modules/linear.cpp:19-106); its backward is MMBackward + the bias' sum_to_shape
(src/inferno/gradfn/mmbackward.cpp:36-98).  Here both directions run on the tcgen05 GEMM of
``csrc/linear_gemm.cuh`` through the C ABI (bf16 tensors, a bias of either type, fp32 accumulation).

``fused_linear`` adds the activation and the residual that follow a projection in a transformer block to its epilogue, and
``feed_forward`` joins two of them (InfernoApp/main.cpp:844-909: ff1 -> gelu -> ff2 -> + x; the reference's gelu is the tanh form,
src/inferno/functional/gelu_kernels.h:6-14).
"""
from __future__ import annotations

import torch

from . import _capi


def linear_forward(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """y = x @ w + bias with x [..., K], w [K, N] (the reference's [in, out] storage), bias [N]."""
    return _capi.host().linear_forward(x, w, bias)


def linear_backward(x, w, dy, need_dx=True, need_dw=True, need_db=True):
    """(dx, dw, db) of ``linear_forward``; db is fp32; what is not needed comes back as None.

    A dW whose tiles alone would not fill the GPU evenly is cut along the tokens and its parts are added up in fp32 in the order in
    which they finish: its bits can differ from run to run in the last place.  db repeats bit for bit, and so do dx beside a dW and
    y, unless they have few tiles and a contraction of 1024 or more: y is then cut like dW, and a dx that is asked for without dW is
    cut as well and its parts, at most eight, are rounded to bf16 as they are added (``ib200_linear_bwd_ws``)."""
    return _capi.host().linear_backward(x, w, dy, need_dx, need_dw, need_db)


class LinearFunction:
    """The differentiable projection (backward node in csrc/host_ops.cpp), under the name it had as an autograd function.  Second
    derivatives are refused (NotImplementedError)."""

    @staticmethod
    def apply(x, w, bias):
        return _capi.host().linear(x, w, bias)


def fused_linear_forward(x, w, bias=None, activation: str | None = None, residual=None, keep_slope: bool = False):
    """(y, slope) with y = act(x @ w + bias) + residual; activation is None or "gelu" (the tanh form), residual has y's shape.

    slope is what the backward needs: the activation's derivative at x @ w + bias, in fp16.  None without an activation, or
    when it is not kept."""
    return _capi.host().fused_linear_forward(x, w, bias, activation, residual, keep_slope)


def fused_linear_backward(x, w, dy, slope=None, activation: str | None = None, need_dx=True, need_dw=True, need_db=True):
    """(dx, dw, db) of ``fused_linear_forward``; db is fp32; what is not needed comes back as None.  The residual's gradient is dy.

    With an activation dz = dy * slope is rounded to bf16 ahead of the two products, db is summed before that.  dw is added up as in
    ``linear_backward``; dx and db repeat bit for bit."""
    return _capi.host().fused_linear_backward(x, w, dy, slope, activation, need_dx, need_dw, need_db)


def fused_linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, activation: str | None = None,
                 residual: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x @ w + bias) + residual`` in one kernel; differentiable (backward node in csrc/host_ops.cpp).  bf16 tensors, a bias of
    either type; in_features and out_features are multiples of 8, the number of rows is free.  Second derivatives are refused (NotImplementedError)."""
    return _capi.host().fused_linear(x, w, bias, activation, residual)


def feed_forward(x: torch.Tensor, w1: torch.Tensor, b1: torch.Tensor | None, w2: torch.Tensor, b2: torch.Tensor | None,
                 residual: torch.Tensor | None = None) -> torch.Tensor:
    """``gelu(x @ w1 + b1) @ w2 + b2 + residual``; differentiable.  w1 [C, H], w2 [H, C]; biases and residual may be None.

    Two kernels forward; backward the gradient of the hidden layer is multiplied by gelu' in the epilogue of the product that
    makes it.  The hidden layer is rounded to bf16 between the products, and so is its gradient.  Second derivatives are
    refused (NotImplementedError)."""
    return _capi.host().feed_forward(x, w1, b1, w2, b2, residual)


class Linear(torch.nn.Module):
    """``x @ W + b`` with W stored [in, out] like the reference's Linear; bf16 weight, fp32-accumulated GEMM.
    With an activation ("gelu") or a residual given to forward, these are part of the kernel's epilogue."""

    activation: str | None = None      # (also of a module that was pickled before it could have one)

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: str | None = None):
        super().__init__()
        self.activation = activation
        self.weight = torch.nn.Parameter(torch.empty(in_features, out_features))
        self.bias = torch.nn.Parameter(torch.zeros(out_features)) if bias else None
        torch.nn.init.normal_(self.weight, 0.0, 0.02)

    def forward(self, x, residual=None):
        if self.activation is None and residual is None:
            return _capi.host().linear(x, self.weight, self.bias)
        return fused_linear(x, self.weight, self.bias, self.activation, residual)


class FeedForward(torch.nn.Module):
    """``feed_forward`` with its two projections as ``ff1`` and ``ff2``."""

    def __init__(self, features: int, hidden: int, bias: bool = True):
        super().__init__()
        self.ff1, self.ff2 = Linear(features, hidden, bias), Linear(hidden, features, bias)

    def forward(self, x, residual=None):
        return feed_forward(x, self.ff1.weight, self.ff1.bias, self.ff2.weight, self.ff2.bias, residual)


def _time_shape(M: int, K: int, N: int, iters: int = 20):
    """Forward and backward of one projection on synthetic bf16 data, timed with CUDA events."""
    g = torch.Generator(device="cuda").manual_seed(M + K + N)
    x = torch.randn(M, K, device="cuda", generator=g).to(torch.bfloat16)
    w = (torch.randn(K, N, device="cuda", generator=g) / K ** 0.5).to(torch.bfloat16)
    b = torch.randn(N, device="cuda", generator=g)
    dy = torch.randn(M, N, device="cuda", generator=g).to(torch.bfloat16)

    def timed(fn):
        for _ in range(3):
            fn()
        torch.cuda.synchronize()
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        for _ in range(iters):
            fn()
        e1.record()
        torch.cuda.synchronize()
        return e0.elapsed_time(e1) / iters

    fwd = timed(lambda: linear_forward(x, w, b))
    bwd = timed(lambda: linear_backward(x, w, dy))
    flop = 2.0 * M * K * N
    return dict(M=M, K=K, N=N, fwd_ms=fwd, fwd_tflops=flop / fwd / 1e9, bwd_ms=bwd, bwd_tflops=2 * flop / bwd / 1e9)


if __name__ == "__main__":
    import argparse
    import json

    ap = argparse.ArgumentParser(description="time y = x W + b and its backward (dX, dW, db) on one GPU")
    ap.add_argument("M", type=int, nargs="?", default=16384)
    ap.add_argument("K", type=int, nargs="?", default=768)
    ap.add_argument("N", type=int, nargs="?", default=2304)
    ap.add_argument("--iters", type=int, default=20)
    a = ap.parse_args()
    print(json.dumps(_time_shape(a.M, a.K, a.N, a.iters)))
