"""Projections with GELU and residual in their epilogue, and the feed-forward block, against the formulas in 64 bits.

Tolerances, on the norm of each result.  A rounding to bf16 is off by at most 2^-8 of the value, so a result that is rounded once is off by at most
2^-8 of its norm; the fp32 sums behind it (K 2^-23 of the sum of magnitudes at most, in practice sqrt(K) of it) are covered by the factor 1.1.
Where an operand was rounded before (the hidden layer, its gradient, the gradient behind gelu'), two independent roundings meet: sqrt(2) 2^-8.  gelu'(z)
is kept in fp16, off by at most 2^-11 of itself: in sums that are not rounded to bf16 afterwards (fp32 db) that is 2^-11 of the sum of magnitudes."""
import os
import subprocess
import sys

import pytest
import torch

from inferno_b200 import linear as L

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ONE, TWO = 1.1 * 2.0 ** -8, 1.1 * 2.0 ** 0.5 * 2.0 ** -8


def normal(*shape, seed, std=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def gelu64(z):
    c = (2 / torch.pi) ** 0.5
    t = torch.tanh(c * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def rel(got, want):
    n = float(want.norm())
    return float((got.double() - want).norm()) / n if n else float(got.double().norm())


def problem(M, K, N, seed=0):
    return (normal(M, K, seed=seed), normal(K, N, seed=seed + 1, std=K ** -0.5), normal(N, seed=seed + 2, std=0.5), normal(M, N, seed=seed + 3),
            normal(M, N, seed=seed + 4, std=0.1))


def reference(x, w, b, res, dy, act):
    x, w, dy = x.double(), w.double(), dy.double()
    z = x @ w + (b.double() if b is not None else 0)
    y, slope = gelu64(z) if act else (z, torch.ones_like(z))
    dz = dy * slope
    return z, y + (res.double() if res is not None else 0), dz @ w.t(), x.t() @ dz, dz.sum(0), dz.abs().sum(0)


def check(x, w, b, res, dy, act):
    leaves = [t for t in (x, w, b, res) if t is not None]
    for t in leaves:
        t.requires_grad_()
    y = L.fused_linear(x, w, b, "gelu" if act else None, res)
    grads = dict(zip([id(t) for t in leaves], torch.autograd.grad(y, leaves, dy)))
    d = [None if t is None else t.detach() for t in (x, w, b, res)]
    _, wy, wdx, wdw, wdb, sdb = reference(*d, dy, act)
    assert y.dtype == torch.bfloat16 and rel(y.detach(), wy) <= ONE
    two = TWO if act else ONE
    assert rel(grads[id(x)], wdx) <= two and rel(grads[id(w)], wdw) <= two
    if b is not None:
        g = grads[id(b)]
        assert g.dtype == b.dtype
        tol = 2.0 ** -11 * float(sdb.norm()) + (ONE if b.dtype == torch.bfloat16 else 2.0 ** -18) * float(wdb.norm()) + 2.0 ** -18 * float(sdb.norm())
        assert float((g.double() - wdb).norm()) <= tol
    if res is not None:
        assert torch.equal(grads[id(res)], dy)
    return y.detach(), grads


# Rows on either side of every border (one warp's 32, a CTA's 128, a pair's 256), columns and depths at the tiles' edges, products cut along K.
@pytest.mark.parametrize("M", [1, 2, 3, 5, 8, 15, 16, 17, 31, 33, 64, 65, 127, 129, 255, 257, 777])
@pytest.mark.parametrize("act,with_res", [(True, False), (False, True), (True, True)])
def test_rows(M, act, with_res):
    x, w, b, res, dy = problem(M, 200, 328, seed=M)
    check(x, w, b, res if with_res else None, dy, act)


@pytest.mark.parametrize("M,K,N", [(8, 8, 8), (5, 8, 264), (256, 64, 256), (264, 72, 520), (3, 4104, 264), (130, 2056, 72), (4097, 136, 264), (1000, 768, 768),
                                   (2047, 1000, 2008), (9479, 1032, 2056), (20, 4096, 4096), (1, 8192, 1024)])
@pytest.mark.parametrize("act,with_res", [(True, False), (False, True), (True, True)])
def test_shapes(M, K, N, act, with_res):
    x, w, b, res, dy = problem(M, K, N, seed=M + K + N)
    check(x, w, b, res if with_res else None, dy, act)


@pytest.mark.parametrize("M", [4, 300])
@pytest.mark.parametrize("act,with_res", [(True, False), (False, True), (True, True), (False, False)])
def test_biases_of_either_type_or_none(M, act, with_res):
    x, w, b, res, dy = problem(M, 256, 520, seed=7)
    for bias in (None, b, b.float()):
        x, w, res = (t.detach().clone() for t in (x, w, res))
        check(x, w, None if bias is None else bias.detach().clone(), res if with_res else None, dy, act)


@pytest.mark.parametrize("M,K,N", [(6, 1024, 512), (513, 1024, 512)])
def test_kept_slope(M, K, N):
    x, w, b, res, dy = problem(M, K, N, seed=9)
    b = b.float()
    b[:5] = torch.tensor([100.0, -100.0, 16.5, -3e38, 3e38], device="cuda")
    y, slope = L.fused_linear_forward(x, w, b, "gelu", res, keep_slope=True)
    z, wy, *_ = reference(x, w, b, res, dy, True)
    assert slope.dtype == torch.float16 and slope.shape == y.shape
    # half a step of fp16; |gelu''| < 1.2 times what fp32 sums leave of z; the exponential and the products behind it
    want = gelu64(z.clamp(-16, 16))[1]
    assert bool(((slope.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -18 + 1.2 * K * 2.0 ** -23 * (x.double().abs() @ w.double().abs())).all())
    keep = [i for i in range(N) if i not in (3, 4)]
    assert rel(y[:, keep], wy[:, keep]) <= ONE and torch.equal(y[:, 3], res[:, 3]) and bool((y[:, 4] > 2e38).all())
    assert L.fused_linear_forward(x, w, b, "gelu", res)[1] is None and L.fused_linear_forward(x, w, b, None, res, True)[1] is None
    dx, dw, db = L.fused_linear_backward(x, w, dy, slope, "gelu")
    assert all(bool(torch.isfinite(t).all()) for t in (dx, dw, db))
    # far out the slope is 1 or 0 exactly
    assert bool((db[[1, 3]] == 0).all()) and torch.allclose(db[[0, 2, 4]], dy[:, [0, 2, 4]].float().sum(0), rtol=1e-5, atol=1e-5)


def test_gelu_keeps_its_relative_precision_in_the_tail():
    """Element by element: half a step of bf16, and an exponential's error of 2^-21 of its argument (at most 40 here)."""
    z = torch.linspace(-9, 9, 4096, device="cuda").to(torch.bfloat16)
    x, w = z.view(-1, 1) * torch.eye(1, 8, device="cuda").to(torch.bfloat16), torch.zeros(8, 64, device="cuda", dtype=torch.bfloat16)
    w[0] = 1.0
    y = L.fused_linear_forward(x, w, None, "gelu")[0]
    want = gelu64(z.double())[0]
    # tanh in 64 bits loses the tail itself: below -4 the logistic form
    u = 0.7978845608028654 * (z.double() + 0.044715 * z.double() ** 3)
    want = torch.where(z < -4, z.double() / (1 + torch.exp(-2 * u)), want)
    tol = (2.0 ** -8 + 2.0 ** -14) * want.abs() + 2.0 ** -126
    assert bool(((y.double() - want[:, None]).abs() <= tol[:, None]).all())


def test_rows_do_not_touch_each_other():
    """A row with NaN or infinities leaves the others as they were, and so do rows past the last one."""
    for M, K, N in ((7, 1024, 512), (300, 512, 264)):
        x, w, b, res, dy = problem(M, K, N, seed=11)
        y0 = L.fused_linear_forward(x, w, b, "gelu", res)[0]
        x2 = x.clone()
        x2[3, 5], x2[5, 6] = float("nan"), float("inf")
        y = L.fused_linear_forward(x2, w, b, "gelu", res)[0]
        same = [i for i in range(M) if i not in (3, 5)]
        assert torch.equal(y[same], y0[same]) and bool(torch.isnan(y[3]).all()) and bool((~torch.isfinite(y[5])).any())
        buf = torch.full((M + 3, N), 7.0, device="cuda", dtype=torch.bfloat16)
        from inferno_b200 import _capi
        s = torch.cuda.current_stream().cuda_stream
        need = _capi.lib().ib200_fused_linear_workspace_bytes(M, K, N, 1, 0)
        ws = torch.empty(max(need, 256), device="cuda", dtype=torch.uint8)
        assert _capi.lib().ib200_fused_linear_fwd(x.data_ptr(), w.data_ptr(), b.data_ptr(), 1, res.data_ptr(), 1, buf.data_ptr(), None, M, K, N, ws.data_ptr(),
                                                  need, s) == _capi.OK
        assert torch.equal(buf[:M], y0) and bool((buf[M:] == 7.0).all())


def test_parts_views_and_repeats():
    x, w, b, res, dy = problem(333, 264, 520, seed=13)
    y, slope = L.fused_linear_forward(x, w, b, "gelu", res, True)
    full = L.fused_linear_backward(x, w, dy, slope, "gelu")
    for need in ((True, False, False), (False, True, False), (False, False, True), (True, False, True), (False, True, True), (True, True, False), (False,) * 3):
        for have, g, f in zip(need, L.fused_linear_backward(x, w, dy, slope, "gelu", *need), full):
            assert (g is None) != have and (not have or rel(g, f.double()) <= 2.0 ** -8)
    dx, _, db = L.fused_linear_backward(x, w, dy, slope, "gelu")
    assert torch.equal(dx, full[0]) and torch.equal(db, full[2]) and torch.equal(L.fused_linear_forward(x, w, b, "gelu", res)[0], y)
    # operands that are slices of wider tensors, begin off 16 bytes, are transposed, or lie in more axes
    wide = normal(333, 600, seed=1)
    view = wide[:, 3:523]
    assert torch.equal(L.fused_linear(x, w, b, "gelu", view), L.fused_linear(x, w, b, "gelu", view.contiguous()))
    off = normal(333 * 264 + 1, seed=2)[1:].view(333, 264)
    assert torch.equal(L.fused_linear(off, w, b, "gelu"), L.fused_linear(off.clone(), w, b, "gelu"))
    wt = normal(520, 264, seed=3, std=0.06).t()
    assert torch.equal(L.fused_linear(x, wt, b[:520], "gelu"), L.fused_linear(x, wt.contiguous(), b, "gelu"))
    bias = normal(523, seed=4)[3:]
    assert torch.equal(L.fused_linear(x, w, bias, None, res), L.fused_linear(x, w, bias.clone(), None, res))
    assert torch.equal(L.fused_linear(x.view(3, 111, 264), w, b, "gelu", res.view(3, 111, 520)).view(333, 520), y)
    assert torch.equal(L.fused_linear(x[0], w, b, "gelu", res[0]), L.fused_linear(x[:1], w, b, "gelu", res[:1])[0])
    # a broadcast gradient and a broadcast residual
    r = res[:1].clone().requires_grad_()
    x.requires_grad_()
    out = L.fused_linear(x, w, b, None, r.expand(333, 520))
    gx, gr = torch.autograd.grad(out.sum(), (x, r))
    ones = torch.ones(333, 520, device="cuda", dtype=torch.float64)
    assert rel(gx, ones @ w.double().t()) <= ONE and bool((gr == 333).all() or rel(gr, ones.sum(0, keepdim=True)) <= 2.0 ** -8)


def test_no_rows():
    w, b = normal(64, 128, seed=1).requires_grad_(), normal(128, seed=2).requires_grad_()
    x = torch.empty(0, 3, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = L.fused_linear(x, w, b, "gelu")
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == (0, 3, 128) and dx.shape == x.shape and not dw.any() and not db.any() and dw.shape == w.shape
    ff = L.FeedForward(64, 128).cuda().to(torch.bfloat16)
    z = ff(x, x)
    g = torch.autograd.grad(z, [x] + list(ff.parameters()), torch.empty_like(z))
    assert z.shape == x.shape and all(not t.any() for t in g)


# ---- the feed-forward block -------------------------------------------------------------------------

def ff_problem(M, C, H, seed):
    return (normal(M, C, seed=seed), normal(C, H, seed=seed + 1, std=C ** -0.5), normal(H, seed=seed + 2, std=0.3), normal(H, C, seed=seed + 3, std=H ** -0.5),
            normal(C, seed=seed + 4, std=0.3), normal(M, C, seed=seed + 5), normal(M, C, seed=seed + 6, std=0.1))


def ff_reference(x, w1, b1, w2, b2, res, dy):
    x, w1, w2, dy = x.double(), w1.double(), w2.double(), dy.double()
    h, slope = gelu64(x @ w1 + (0 if b1 is None else b1.double()))
    y = h @ w2 + (0 if b2 is None else b2.double())
    part = y
    if res is not None:
        y = y + res.double()
    dz = (dy @ w2.t()) * slope
    return y, part, dz @ w1.t(), x.t() @ dz, dz.sum(0), h.t() @ dy, dy.sum(0), dz.abs().sum(0)


def check_ff(x, w1, b1, w2, b2, res, dy):
    leaves = [t for t in (x, w1, b1, w2, b2, res) if t is not None]
    for t in leaves:
        t.requires_grad_()
    y = L.feed_forward(x, w1, b1, w2, b2, res)
    g = dict(zip([id(t) for t in leaves], torch.autograd.grad(y, leaves, dy)))
    wy, part, wdx, wdw1, wdb1, wdw2, wdb2, s1 = ff_reference(*(None if t is None else t.detach() for t in (x, w1, b1, w2, b2, res)), dy)
    assert float((y.detach().double() - wy).norm()) <= ONE * float(wy.norm()) + ONE * float(part.norm())
    assert rel(g[id(x)], wdx) <= TWO and rel(g[id(w1)], wdw1) <= TWO and rel(g[id(w2)], wdw2) <= TWO
    if b1 is not None:         # dz is rounded before its columns are summed: at most 2^-8 of the sum of magnitudes
        assert g[id(b1)].dtype == b1.dtype and float((g[id(b1)].double() - wdb1).norm()) <= ONE * float(wdb1.norm()) + ONE * float(s1.norm())
    if b2 is not None:
        assert g[id(b2)].dtype == b2.dtype and rel(g[id(b2)], wdb2) <= (ONE if b2.dtype == torch.bfloat16 else 2.0 ** -14)
    if res is not None:
        assert torch.equal(g[id(res)], dy)


@pytest.mark.parametrize("M", [1, 2, 5, 16, 17, 31, 32, 33, 128, 129, 257, 1023])
def test_feed_forward_rows(M):
    check_ff(*ff_problem(M, 200, 808, seed=M))


@pytest.mark.parametrize("M,C,H", [(7, 8, 8), (300, 64, 256), (100, 264, 72), (2000, 512, 2048), (5000, 256, 1024), (513, 1024, 4096), (3, 2048, 8192), (9000, 136, 520)])
def test_feed_forward_shapes(M, C, H):
    check_ff(*ff_problem(M, C, H, seed=M + C))


@pytest.mark.parametrize("M", [3, 400])
def test_feed_forward_biases_and_residual(M):
    x, w1, b1, w2, b2, res, dy = ff_problem(M, 136, 520, seed=3)
    for a, c, r in ((None, None, None), (b1, None, res), (None, b2, res), (b1.float(), b2, None), (b1, b2.float(), res)):
        check_ff(x.detach().clone(), w1.detach().clone(), None if a is None else a.detach().clone(), w2.detach().clone(), None if c is None else c.detach().clone(),
                 None if r is None else r.detach().clone(), dy)


def test_feed_forward_with_its_input_as_residual_and_parts():
    x, w1, b1, w2, b2, _, dy = ff_problem(500, 136, 520, seed=5)
    x.requires_grad_()
    dx, = torch.autograd.grad(L.feed_forward(x, w1, b1, w2, b2, x), x, dy)
    want = ff_reference(x.detach(), w1, b1, w2, b2, None, dy)
    assert rel(dx, want[2] + dy.double()) <= TWO
    leaves = (x, w1, b1, w2, b2)
    for t in leaves:
        t.requires_grad_()
    want = (want[2], want[3], want[4], want[5], want[6])
    for pick in ([0], [1], [2], [3], [4], [0, 1], [1, 2], [3, 4], [0, 3], [0, 2, 4], [1, 4]):
        y = L.feed_forward(*(t if i in pick else t.detach() for i, t in enumerate(leaves)))
        for i, g in zip(pick, torch.autograd.grad(y, [leaves[i] for i in pick], dy)):
            assert rel(g, want[i]) <= 2 * TWO, (pick, i)      # (the sums of dz: two roundings of terms that largely cancel)


def test_gradient_against_differences():
    """Central differences along the gradient itself, from the outputs in bf16: with steps of 2^-4 of a deviation the truncation is below 2^-7 of the
    difference, and the outputs' rounding (2^-8 each, independent over 600 x 264 of them) is far below it."""
    x, w1, b1, w2, b2, _, dy = ff_problem(600, 264, 520, seed=21)
    x.requires_grad_()
    dx, = torch.autograd.grad(L.feed_forward(x, w1, b1, w2, b2), x, dy)
    v = dx.float() / dx.float().std()
    with torch.no_grad():
        up, down = (x.float() + v / 16).to(torch.bfloat16), (x.float() - v / 16).to(torch.bfloat16)
        num = ((L.feed_forward(up, w1, b1, w2, b2).double() - L.feed_forward(down, w1, b1, w2, b2).double()) * dy.double()).sum()
        want = ((up.double() - down.double()) * dx.double()).sum()
    assert abs(float(num - want)) <= 2.0 ** -6 * abs(float(want))


# ---- streams, graphs, the checked build, and the operators together -----------------------------------------------

def test_streams_and_captured_graphs():
    x, w1, b1, w2, b2, res, dy = ff_problem(700, 264, 1032, seed=31)
    leaves = (x, w1, b1, w2, b2, res)
    for t in leaves:
        t.requires_grad_()

    def step():
        y = L.feed_forward(*leaves)
        h = L.fused_linear(x, w1, b1, "gelu")
        return (y.detach(), h.detach()) + torch.autograd.grad(y, leaves, dy, retain_graph=False) + torch.autograd.grad(h, (x, w1, b1), dh)
    dh = normal(700, 1032, seed=37, std=0.1)
    want = [t.clone() for t in step()]
    near = lambda got: all(rel(a, c.double()) <= 2.0 ** -8 for a, c in zip(got, want))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    s.synchronize()
    assert near(got) and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    big = L.FeedForward(1024, 4096).cuda().to(torch.bfloat16)
    xb = normal(2048, 1024, seed=5).requires_grad_()
    torch.autograd.grad(big(xb), [xb] + list(big.parameters()), normal(2048, 1024, seed=6))
    for g, out in graphs + graphs:
        for t in out:
            if t.data_ptr() != dy.data_ptr():      # the residual's gradient is dy itself
                t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert near(out)


_FIRST = r"""
import sys, torch
from inferno_b200 import _capi, linear as L, norm as N
from inferno_b200.attention import causal_attention_packed
bf16 = lambda *s: torch.randn(*s, device="cuda").to(torch.bfloat16)
ln, ff, up = N.LayerNorm(264).cuda().to(torch.bfloat16), L.FeedForward(264, 520).cuda().to(torch.bfloat16), L.Linear(264, 520, activation="gelu").cuda().to(torch.bfloat16)
x, dy, dh = bf16(333, 264).requires_grad_(), bf16(333, 264), bf16(333, 520)
params = [x] + list(ln.parameters()) + list(ff.parameters()) + list(up.parameters())
def step():
    n = ln(x)
    return torch.autograd.grad((ff(n, x), up(n)), params, (dy, dh))
def run():
    if sys.argv[1] == "capture":
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        g.replay()
        return out
    return step()
got = run()
torch.cuda.synchronize()
for a, b in zip(got, step()):
    assert float((a.float() - b.float()).norm()) <= 2 ** -7 * float(b.float().norm()) + 1e-6
import ctypes
code = ctypes.c_int(-1)
assert _capi.lib().ib200_attn_check_static(torch.cuda.current_stream().cuda_stream, ctypes.byref(code)) == _capi.OK, code.value
for M in (1, 3, 40, 300):                # the checked build goes through every form
    for K, N2 in ((264, 520), (2056, 136)):
        w, b = bf16(K, N2), bf16(N2)
        for act in (None, "gelu"):
            for res in (None, bf16(M, N2)):
                x2 = bf16(M, K).requires_grad_()
                torch.autograd.grad(L.fused_linear(x2, w, b, act, res), x2, bf16(M, N2))
torch.cuda.synchronize()
assert _capi.lib().ib200_attn_check_static(torch.cuda.current_stream().cuda_stream, ctypes.byref(code)) == _capi.OK, code.value
print("steps agree", _capi.lib()._name)
"""


def _child(arg, **env):
    res = subprocess.run([sys.executable, "-c", _FIRST, arg], env=dict(os.environ, PYTHONPATH=ROOT, **env), cwd=ROOT, capture_output=True, text=True, timeout=200)
    assert res.returncode == 0 and "steps agree" in res.stdout, res.stdout[-500:] + res.stderr[-2000:]
    return res.stdout


def test_checked_build_finds_nothing():
    from inferno_b200 import build
    assert "bounds" in _child("eager", IB200_LIB=build.build(bounds=True))


def test_first_call_of_a_process_can_be_captured():
    _child("capture")


def test_a_transformer_block_of_these_operators():
    """ln -> packed attention -> output projection + x -> ln -> feed-forward + x, forward and backward, against the composition in 64 bits.  Each of the
    block's seven tensors between operators is rounded to bf16 (2^-8, independent), and attention's own tolerance is 2e-2: that is what is allowed."""
    from inferno_b200.attention import causal_attention_packed
    from inferno_b200.norm import LayerNorm
    torch.manual_seed(3)
    B, T, C, H = 2, 200, 256, 4
    mods = torch.nn.ModuleDict(dict(ln1=LayerNorm(C), qkv=L.Linear(C, 3 * C), out=L.Linear(C, C), ln2=LayerNorm(C), ff=L.FeedForward(C, 4 * C))).cuda()
    with torch.no_grad():
        for p in mods.parameters():
            p.add_(torch.randn_like(p) * 0.04)
    mods = mods.to(torch.bfloat16)
    x, dy = normal(B, T, C, seed=41).requires_grad_(), normal(B, T, C, seed=42)
    y = mods["out"](causal_attention_packed(mods["qkv"](mods["ln1"](x)), H), residual=x)
    y = mods["ff"](mods["ln2"](y), residual=y)
    params = list(mods.parameters())
    grads = torch.autograd.grad(y, [x] + params, dy)

    p = {k: v.detach().double().requires_grad_() for k, v in mods.named_parameters()}
    xd = x.detach().double().requires_grad_()
    ln = lambda t, n: torch.nn.functional.layer_norm(t, (C,), p[n + ".weight"], p[n + ".bias"], 1e-5)
    lin = lambda t, n: t @ p[n + ".weight"] + p[n + ".bias"]
    q, k, v = (t.view(B, T, H, C // H).transpose(1, 2) for t in lin(ln(xd, "ln1"), "qkv").split(C, 2))
    s = (q @ k.transpose(-1, -2)) / (C // H) ** 0.5
    s = s.masked_fill(torch.triu(torch.ones(T, T, device="cuda", dtype=torch.bool), 1), float("-inf"))
    yd = xd + lin((torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B, T, C), "out")
    yd = yd + lin(torch.nn.functional.gelu(lin(ln(yd, "ln2"), "ff.ff1"), approximate="tanh"), "ff.ff2")
    want = torch.autograd.grad(yd, [xd] + list(p.values()), dy.double())
    assert rel(y.detach(), yd.detach()) <= 2e-2
    for (name, g), wg in zip([("x", grads[0])] + list(zip(p, grads[1:])), want):
        assert rel(g, wg) <= 2e-2, (name, rel(g, wg))


@pytest.mark.parametrize("M", [1, 3, 33, 1001])
def test_plain_projection_takes_any_number_of_rows(M):
    x, w, b, _, dy = problem(M, 136, 264, seed=M)
    for t in (x, w, b):
        t.requires_grad_()
    y = L.LinearFunction.apply(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    _, wy, wdx, wdw, wdb, _ = reference(x.detach(), w.detach(), b.detach(), None, dy, False)
    assert rel(y.detach(), wy) <= ONE and rel(dx, wdx) <= ONE and rel(dw, wdw) <= ONE and rel(db, wdb) <= ONE


@pytest.mark.parametrize("M,K,N", [(1, 264, 4096), (5, 1024, 4096), (40, 2048, 8192), (300, 512, 4104), (600, 256, 2056)])
def test_few_rows_backward(M, K, N):
    """dX of few rows is cut along its long contraction and added up in fp32: rounded once, with weights that need gradients or not, and repeats."""
    x, w, b, res, dy = problem(M, K, N, seed=M + N)
    for act in (False, True):
        slope = L.fused_linear_forward(x, w, b, "gelu", None, True)[1] if act else None
        _, _, wdx, wdw, wdb, sdb = reference(x, w, b, None, dy, act)
        name = "gelu" if act else None
        full = L.fused_linear_backward(x, w, dy, slope, name)
        alone = L.fused_linear_backward(x, w, dy, slope, name, True, False, False)[0]
        assert rel(full[0], wdx) <= (TWO if act else ONE) and rel(full[1], wdw) <= (TWO if act else ONE)
        assert float((full[2].double() - wdb).norm()) <= (2.0 ** -11 if act else 2.0 ** -18) * float(sdb.norm()) + 2.0 ** -18 * float(wdb.norm())
        assert rel(alone, wdx) <= (TWO if act else ONE) and torch.equal(full[0], L.fused_linear_backward(x, w, dy, slope, name)[0])
    C, H = K, N
    x, w1, b1, w2, b2, res, dy = ff_problem(M, C, H, seed=M)
    x.requires_grad_()
    dx, = torch.autograd.grad(L.feed_forward(x, w1, b1, w2, b2, res), x, dy)
    want = ff_reference(x.detach(), w1, b1, w2, b2, res, dy)
    assert rel(dx, want[2]) <= TWO
    check_ff(x.detach().clone(), w1, b1, w2, b2, res, dy)
