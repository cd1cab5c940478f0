"""Forms of the fused projections that their sizes choose, each with its values checked, and the bias gradient of the hidden layer with a bound tight
enough to miss no block of rows."""
import os
import subprocess
import sys

import pytest
import torch
from test_fused_linear_gpu import ONE, check, check_ff, ff_problem, gelu64, problem

from inferno_b200 import linear as L

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# Few rows: blocks of a cluster split K in two from 2048 of it (at most 74 strips of 64 columns), in four from 4096 (at most 37 strips); up to 16 rows and
# up to 32 have a kernel each.  Depths that leave the last block a shorter share, and widths that end inside a strip.
FEW = [(1, 1992, 520), (16, 1984, 4800),                                            # not split
       (3, 2056, 136), (16, 2048, 4096), (9, 3000, 4736),                           # in two, 16 rows
       (17, 2056, 136), (31, 2056, 4096), (32, 4096, 4096),                         # in two, 32 rows
       (1, 4096, 8), (5, 4104, 264), (16, 8200, 2368),                              # in four, 16 rows
       (17, 4104, 264), (24, 8200, 2368), (32, 4096, 1024), (32, 4160, 72)]         # in four, 32 rows


@pytest.mark.parametrize("M,K,N", FEW)
@pytest.mark.parametrize("act,with_res", [(True, False), (False, True), (True, True), (False, False)])
def test_few_rows(M, K, N, act, with_res):
    x, w, b, res, dy = problem(M, K, N, seed=M + K + N)
    y, _ = check(x, w, b, res if with_res else None, dy, act)
    # element by element: half a step of bf16, and fp32 sums of K terms, each off by 2^-24 of the terms so far, behind a slope of at most 1.13;
    # the exponential and the products behind it
    d = [t.detach().double() for t in (x, w, b, res)]
    z = d[0] @ d[1] + d[2]
    want = (gelu64(z)[0] if act else z) + (d[3] if with_res else 0)
    size = d[0].abs() @ d[1].abs() + d[2].abs() + (d[3].abs() if with_res else 0)
    assert bool(((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + (1.13 * (K + 2) * 2.0 ** -24 + 2.0 ** -18) * size).all())
    assert torch.equal(y, L.fused_linear(x.detach(), w.detach(), b.detach(), "gelu" if act else None, res.detach() if with_res else None))


@pytest.mark.parametrize("M,C,H", [(17, 1024, 4096), (32, 512, 4160), (20, 2048, 8192), (16, 1024, 4104)])
def test_feed_forward_of_few_rows(M, C, H):
    check_ff(*ff_problem(M, C, H, seed=M + C))


@pytest.mark.parametrize("bias_type", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,C,H", [(33, 264, 520), (1023, 1024, 4096), (5000, 256, 1024), (9000, 136, 520), (40000, 64, 264)])
def test_bias_gradient_of_the_hidden_layer(M, C, H, bias_type):
    """db1 is the column sum of dz = (dy w2^T) gelu'(z) before dz is rounded.  What is off in a term: the slope, by half a step of fp16 (2^-11 of itself, or
    2^-25 where it is below 2^-14), of either sign, so that M of them add up to the root of their squares; fp32 sums and the slope's own evaluation,
    2^-18 of the terms' magnitudes.  Then the result's rounding.  32 rows left out, sqrt(32 / M) of the norm, are more than twice the bound."""
    x, w1, b1, w2, b2, res, dy = ff_problem(M, C, H, seed=M + H)
    b1 = b1.to(bias_type).requires_grad_()
    g, = torch.autograd.grad(L.feed_forward(x, w1, b1, w2, b2, res), b1, dy)
    dh, slope = dy.double() @ w2.double().t(), gelu64(x.double() @ w1.double() + b1.detach().double())[1]
    dz = dh * slope
    want = dz.sum(0)
    slope_off = (dh * (slope.abs() * 2.0 ** -11).clamp_min(2.0 ** -25)).square().sum(0).sqrt()
    tol = float(slope_off.norm()) + 2.0 ** -18 * float(dz.abs().sum(0).norm()) + (ONE * float(want.norm()) if bias_type == torch.bfloat16 else 0.0)
    assert g.dtype == bias_type and float((g.double() - want).norm()) <= tol
    lost = float(dz[M // 64 * 32:M // 64 * 32 + 32].sum(0).norm())      # a block of 32 rows in the middle would be noticed
    assert lost > 2 * tol


# The kernel that a process meets first may be met in a capture: each of the product's forms in a process of its own.
FORMS = {"bias": "lambda: L.linear_forward(x, w, b)", "plain": "lambda: L.linear_forward(x, w)", "residual": "lambda: L.fused_linear_forward(x, w, b, None, r)[0]",
         "gelu": "lambda: L.fused_linear_forward(x, w, b, 'gelu', r, True)[0]", "slabs": "lambda: L.fused_linear_backward(x[:40], w, r[:40])[0]",
         "cut": "lambda: L.linear_backward(x, w, r)[0]", "few": "lambda: L.fused_linear(x[:5], w, b, 'gelu')", "norm": "lambda: N.layer_norm(x)"}

_FIRST = r"""
import sys, torch
from inferno_b200 import linear as L, norm as N
bf16 = lambda *s: torch.randn(*s, device="cuda").to(torch.bfloat16)
x, w, b, r = bf16(2000, 512), bf16(512, 4096), bf16(4096), bf16(2000, 4096)
call = eval(sys.argv[1])
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = call()
want = call().clone()
for _ in range(2):
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and bool(want.any())
print("the same")
"""


@pytest.mark.parametrize("form", FORMS)
def test_first_call_of_a_process_captured(form):
    res = subprocess.run([sys.executable, "-c", _FIRST, FORMS[form]], env=dict(os.environ, PYTHONPATH=ROOT), cwd=ROOT, capture_output=True, text=True, timeout=150)
    assert res.returncode == 0 and "the same" in res.stdout, res.stdout[-500:] + res.stderr[-2000:]
