"""Layer norm, fused projections and the feed-forward block where calls meet: more elements than 32 bits count, several host threads, a capture that
torch has to refuse, saved-tensor hooks, in-place changes, other shapes on one scratch."""
import os
import subprocess
import sys
import threading

import pytest
import torch

from inferno_b200 import linear as L
from inferno_b200 import norm as N

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def bf16(*shape, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g, dtype=torch.bfloat16) * std)


def rel(got, want):
    return float((got.double() - want.double()).norm() / want.double().norm())


def test_layer_norm_past_32_bits():
    """270000 x 8192 elements: the last rows' results, and weight gradients that every row is part of.  Their tolerance: half a step of bf16, and sums of
    1824 rows a block (2^-24 each of the sum of magnitudes, which is sqrt(270000) = 520 times the result's size: 2^-4 of a step at most)."""
    M, C = 270000, 8192
    x, dy = bf16(M, C, seed=1), bf16(M, C, seed=2, std=0.1)
    w, b = bf16(C, seed=3), bf16(C, seed=4)
    y, mean, rstd = N.layer_norm_forward(x, w, b)
    dx, dw, db = N.layer_norm_backward(x, dy, mean, rstd, w)
    wdw, wdb = torch.zeros(C, device="cuda", dtype=torch.float64), torch.zeros(C, device="cuda", dtype=torch.float64)
    for i in range(0, M, 10000):
        xd, gd = x[i:i + 10000].double(), dy[i:i + 10000].double()
        var, mu = torch.var_mean(xd, dim=1, correction=0, keepdim=True)
        xh = (xd - mu) * torch.rsqrt(var + 1e-5)
        wdw += (gd * xh).sum(0)
        wdb += gd.sum(0)
        if i + 10000 >= M or i == 0:
            g = gd * w.double()
            part = slice(i, i + 10000)
            assert rel(y[part], xh * w.double() + b.double()) <= 1.1 * 2 ** -8
            assert rel(dx[part], torch.rsqrt(var + 1e-5) * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))) <= 1.1 * 2 ** -8
    assert rel(dw, wdw) <= 1.1 * 2 ** -8 and rel(db, wdb) <= 1.1 * 2 ** -8


def test_projection_past_32_bits():
    """600000 x 4096 outputs (and as many slopes, residuals, gradients): rows from both ends.  Roundings as in the tests of ordinary sizes."""
    M, K, H = 600000, 64, 4096
    x, w, b, res, dy = bf16(M, K, seed=1), bf16(K, H, seed=2, std=K ** -0.5), bf16(H, seed=3), bf16(M, H, seed=4), bf16(M, H, seed=5, std=0.1)
    y, slope = L.fused_linear_forward(x, w, b, "gelu", res, True)
    dx, dw, db = L.fused_linear_backward(x, w, dy, slope, "gelu")
    for part in (slice(0, 300), slice(M - 300, M)):
        z = x[part].double() @ w.double() + b.double()
        zt = z.clone().requires_grad_()
        h = torch.nn.functional.gelu(zt, approximate="tanh")
        s, = torch.autograd.grad(h.sum(), zt)
        assert rel(y[part], h.detach() + res[part].double()) <= 1.1 * 2 ** -8 and rel(slope[part], s) <= 2 ** -10
        assert rel(dx[part], (dy[part].double() * s) @ w.double().t()) <= 1.1 * 2 ** 0.5 * 2 ** -8
    wdw, wdb = torch.zeros(K, H, device="cuda", dtype=torch.float64), torch.zeros(H, device="cuda", dtype=torch.float64)
    for i in range(0, M, 30000):
        dz = dy[i:i + 30000].double() * slope[i:i + 30000].double()
        wdw += x[i:i + 30000].double().t() @ dz
        wdb += dz.sum(0)
    # dz rounded (2^-8), the slope taken as it was kept; fp32 sums of 600000 terms in parts: 2^-24 of the sum of magnitudes a term, 2^-9 of the result
    assert rel(dw, wdw) <= 1.1 * 2 ** 0.5 * 2 ** -8 and rel(db, wdb) <= 2 ** -9


def test_feed_forward_past_32_bits():
    M, C, H = 540000, 64, 4096
    x, w1, b1, w2, b2 = bf16(M, C, seed=1), bf16(C, H, seed=2, std=C ** -0.5), bf16(H, seed=3), bf16(H, C, seed=4, std=H ** -0.5), bf16(C, seed=5)
    dy = bf16(M, C, seed=6, std=0.1)
    x.requires_grad_(); b1.requires_grad_()
    y = L.feed_forward(x, w1, b1, w2, b2, x)
    dx, db1 = torch.autograd.grad(y, (x, b1), dy)
    wdb = torch.zeros(H, device="cuda", dtype=torch.float64)
    mag = torch.zeros(H, device="cuda", dtype=torch.float64)
    for i in range(0, M, 20000):
        part = slice(i, i + 20000)
        zt = (x.detach()[part].double() @ w1.double() + b1.detach().double()).requires_grad_()
        h = torch.nn.functional.gelu(zt, approximate="tanh")
        dz, = torch.autograd.grad(h, zt, dy[part].double() @ w2.double().t())
        wdb += dz.sum(0)
        mag += dz.square().sum(0)
        if i == 0 or i + 20000 >= M:
            assert rel(y.detach()[part], x.detach()[part].double() + h.detach() @ w2.double() + b2.double()) <= 2 * 1.1 * 2 ** -8
            assert rel(dx[part], dy[part].double() + dz @ w1.double().t()) <= 2 * 1.1 * 2 ** -8
    # the result's rounding; slopes in fp16 and fp32 products: independent errors of at most 2^-11 a term
    assert float((db1.double() - wdb).norm()) <= 1.1 * 2 ** -8 * float(wdb.norm()) + 2 ** -11 * float(mag.sqrt().norm()) * 4


def step_of(M, seed):
    x, w1, b1, w2, b2 = bf16(M, 256, seed=seed), bf16(256, 520, seed=seed + 1, std=0.06), bf16(520, seed=seed + 2), bf16(520, 256, seed=seed + 3, std=0.04), bf16(256, seed=seed + 4)
    lw, lb, dy = bf16(256, seed=seed + 5), bf16(256, seed=seed + 6), bf16(M, 256, seed=seed + 7)
    leaves = [t.requires_grad_() for t in (x, lw, lb, w1, b1, w2, b2)]

    def step():
        n = N.layer_norm(x, lw, lb)
        y = L.feed_forward(n, w1, b1, w2, b2, x)
        y = L.fused_linear(L.fused_linear(y, w1, b1, "gelu"), w2, b2, None, y)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
    return step


@pytest.mark.parametrize("own_stream", [False, True])
def test_several_host_threads(own_stream):
    """Four threads, on one stream or each on its own, problems of different size: everybody gets what a call alone gives (weight gradients to their own
    repeatability, everything that does not follow from one bit for bit)."""
    steps = [step_of(M, 100 * M) for M in (3, 70, 500, 1111)]
    want = [[t.clone() for t in s()] for s in steps]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        s = torch.cuda.Stream() if own_stream else torch.cuda.default_stream()
        with torch.cuda.stream(s):
            for _ in range(15):
                got = steps[i]()
                s.synchronize()
                if not torch.equal(got[0], want[i][0]) or not torch.equal(got[1], want[i][1]) or any(rel(a, b) > 2 ** -8 for a, b in zip(got, want[i])):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


_LIVING_GRAPH = r"""
import torch
from inferno_b200 import linear as L, norm as N
bf16 = lambda *s: torch.randn(*s, device="cuda").to(torch.bfloat16)
x, lw, lb, w, b, w2, dy = bf16(100, 64), bf16(64), bf16(64), bf16(64, 128), bf16(128), bf16(128, 64), bf16(100, 64)
leaves = [t.requires_grad_() for t in (x, lw, lb, w, b, w2)]
def forward():
    n = N.layer_norm(x, lw, lb)
    return L.fused_linear(L.feed_forward(n, w, b, w2, None, x), w, b, "gelu") @ w2
y = forward()                       # an eager graph of the leaves, which lives on
want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
try:
    with torch.cuda.graph(g):
        torch.autograd.grad(forward(), leaves, dy)
    print("captured")
except RuntimeError as e:
    print("refused")
del g
got = torch.autograd.grad(forward(), leaves, dy)
torch.cuda.synchronize()
for a, c in zip(got, want):
    assert float((a.float() - c.float()).norm()) <= 2 ** -7 * float(c.float().norm())
print("goes on")
"""


def test_backward_captured_beside_a_living_eager_graph_does_not_end_the_process():
    """torch ties a leaf's gradient to the stream of the graph that lives, and the capture breaks: an exception, not the end of the process, and eager
    calls go on."""
    res = subprocess.run([sys.executable, "-c", _LIVING_GRAPH], env=dict(os.environ, PYTHONPATH=ROOT), cwd=ROOT, capture_output=True, text=True, timeout=150)
    assert res.returncode == 0 and "goes on" in res.stdout, res.stdout[-500:] + res.stderr[-2000:]


def test_saved_tensors():
    """What is saved passes through hooks (here: to the host and back, and through other strides), and an operand changed in place is noticed."""
    step = step_of(200, 7)
    want = step()
    with torch.autograd.graph.save_on_cpu():
        got = step()
    assert all(rel(a, b) <= 2 ** -8 for a, b in zip(got, want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 else t):
        got = step()
    assert all(rel(a, b) <= 2 ** -8 for a, b in zip(got, want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.float()):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            step()
    x, w = bf16(40, 64, seed=1), bf16(64, 64, seed=2).requires_grad_()
    x2 = x.clone()
    y = L.fused_linear(x2, w, None, "gelu")
    x2.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    x2 = x.clone().requires_grad_() * 1.0
    y = N.layer_norm(x2)
    x2.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


def test_one_input_in_several_places():
    """x as its own residual, one weight in both projections, a tensor as weight and input: gradients add up."""
    w = bf16(128, 128, seed=3, std=0.09).requires_grad_()
    dy = bf16(128, 128, seed=4)
    y = L.fused_linear(w, w, None, "gelu", w)
    g, = torch.autograd.grad(y, w, dy)
    d = w.detach().double().requires_grad_()
    want, = torch.autograd.grad(torch.nn.functional.gelu(d @ d, approximate="tanh") + d, d, dy.double())
    assert rel(g, want) <= 3 * 2 ** -8         # three rounded gradients, and their rounded sum
    y = L.feed_forward(w, w, None, w, None, w)
    g, = torch.autograd.grad(y, w, dy)
    want, = torch.autograd.grad(torch.nn.functional.gelu(d @ d, approximate="tanh") @ d + d, d, dy.double())
    assert rel(g, want) <= 4 * 2 ** -8
    b = bf16(128, seed=5).requires_grad_()
    y = N.layer_norm(w, b, b)
    g, = torch.autograd.grad(y, b, dy)
    db = b.detach().double().requires_grad_()
    want, = torch.autograd.grad(torch.nn.functional.layer_norm(d.detach(), (128,), db, db, 1e-5), db, dy.double())
    assert rel(g, want) <= 3 * 2 ** -8


def test_second_derivatives_are_refused():
    """create_graph gives the same first gradients; going through them again raises, whichever tensor is asked for, also beside a residual's own path."""
    x, w1, b1, w2 = bf16(40, 64, seed=1), bf16(64, 128, seed=2, std=0.1), bf16(128, seed=3), bf16(128, 64, seed=4, std=0.1)
    res, lw, lb = bf16(40, 128, seed=5), bf16(64, seed=6), bf16(64, seed=7)
    for call, leaves in ((lambda: L.fused_linear(x, w1, b1, "gelu", res), (x, w1, b1, res)), (lambda: L.fused_linear(x, w1, None, None, res), (x, w1)),
                         (lambda: L.feed_forward(x, w1, b1, w2, None, x), (x, w1, b1, w2)), (lambda: N.layer_norm(x, lw, lb), (x, lw, lb)), (lambda: N.layer_norm(x), (x,))):
        for t in leaves:
            t.requires_grad_()
        dy = torch.ones_like(call().detach()).requires_grad_()
        want = torch.autograd.grad(call(), leaves, dy)
        got = torch.autograd.grad(call(), leaves, dy, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))                 # (40 rows: no sum is cut, all of them repeat)
        for of in leaves + (dy,):
            if of is not b1 and of is not res and of is not lb:                  # (the first gradients do not depend on what is only added)
                with pytest.raises(NotImplementedError, match="second derivatives"):
                    torch.autograd.grad(sum((g.float() ** 2).sum() for g in got), of, retain_graph=True)
        for t in leaves:
            t.requires_grad_(False)
    y = L.fused_linear(x, w1, b1, "gelu")                                        # without any leaf, and without create_graph, nothing is in the way
    assert not y.requires_grad and all(not g.requires_grad for g in want)
