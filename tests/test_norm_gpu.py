"""Layer norm, forward and backward, against the formulas in 64 bits.

Tolerances.  A result is rounded once to its type: half a step, finfo(t).eps / 2 of the value.  Before that everything is fp32.  A row's
sums are at most 64 terms a thread and nine levels of a tree deep, so off by less than 2^-24 (64 + 9) < 2^-17 of the sum of magnitudes;
`SUM` allows that, and covers the handful of roundings of the element-wise steps as well.  The rows' sums of dw and db are chains of at
most a block's rows, the block's eight warps, an eighth of the blocks and eight parts: under 128 at these sizes, 2^-17 again."""
import pytest
import torch

from inferno_b200 import norm as N

pytestmark = pytest.mark.gpu
SUM = 2.0 ** -17
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def half_step(t):
    return torch.finfo(t.dtype).eps / 2


def make(M, C, dtype, param, seed, mean=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    x = (r(M, C) * torch.exp(0.5 * r(M, 1)) + mean * r(M, 1)).to(DT[dtype])
    return x, (1 + 0.2 * r(C)).to(DT[param]), (0.1 * r(C)).to(DT[param]), r(M, C).to(DT[dtype])


def reference(x, w, b, dy, eps=1e-5):
    """y, dx, dw, db in 64 bits, and for each how large the terms are that its fp32 evaluation adds up."""
    x, dy = x.double(), dy.double()
    C = x.shape[-1]
    w = torch.ones(C, device=x.device, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(C, device=x.device, dtype=torch.float64) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    size = xh.abs() + x.abs().mean(-1, keepdim=True) * rstd      # of xh: the error of the mean is relative to the row's size
    g = dy * w
    y = xh * w + b
    m1, m2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    dx = rstd * (g - m1 - xh * m2)
    dx_size = rstd * (g.abs() + g.abs().mean(-1, keepdim=True) + size * (g * size).abs().mean(-1, keepdim=True))
    rows = tuple(range(x.dim() - 1))
    return ((y, dx, (dy * xh).sum(rows), dy.sum(rows)),
            (size * w.abs() + b.abs(), dx_size, (dy.abs() * size).sum(rows), dy.abs().sum(rows)))


def close(got, want, size, what):
    tol = half_step(got) * want.abs() * (1 + 2 ** -7) + SUM * size + 2.0 ** -126
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), f"{what}: {float((off / tol).max()):.2f} of the tolerance"


def check(x, w, b, dy, eps=1e-5):
    leaves = [t for t in (x, w, b) if t is not None]
    for t in leaves:
        t.requires_grad_()
    y = N.layer_norm(x, w, b, eps)
    grads = dict(zip([id(t) for t in leaves], torch.autograd.grad(y, leaves, dy)))
    want, size = reference(x.detach(), None if w is None else w.detach(), None if b is None else b.detach(), dy, eps)
    assert y.dtype == x.dtype and y.is_contiguous()
    close(y.detach(), want[0], size[0], "y")
    for t, k, name in ((x, 1, "dx"), (w, 2, "dw"), (b, 3, "db")):
        if t is not None:
            got = grads[id(t)]
            assert got.dtype == t.dtype and got.shape == t.shape
            close(got, want[k], size[k], name)


# Widths at every border of the shapes: one warp, 128 and 512 threads a row, one to four chunks each, and rows that are not whole chunks.
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("C", [1, 2, 7, 8, 31, 64, 250, 256, 264, 512, 520, 768, 1000, 1024, 1025, 1032, 2048, 4096, 4104, 5000, 8191, 8192])
def test_widths(dtype, C):
    for M in (1, 37):
        check(*make(M, C, dtype, dtype, 7 * C + M))


@pytest.mark.parametrize("C", [8200, 12288, 16376, 16384, 16383])
def test_widest_bf16_rows(C):
    check(*make(5, C, "bf16", "bf16", C))


@pytest.mark.parametrize("M,C,dtype", [(2331, 1000, "f32"), (5000, 768, "bf16"), (3, 768, "bf16"), (2367, 256, "bf16"), (2369, 64, "f32"), (601, 4096, "bf16"),
                                       (300, 8192, "bf16"), (149, 8192, "f32")])
def test_more_rows_than_blocks(M, C, dtype):
    check(*make(M, C, dtype, dtype, M))


@pytest.mark.parametrize("dtype,param", [("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("C", [768, 777])
def test_parameters_of_the_other_type(dtype, param, C):
    check(*make(100, C, dtype, param, C))


@pytest.mark.parametrize("with_w,with_b", [(True, False), (False, True), (False, False)])
def test_without_weight_or_bias(with_w, with_b):
    x, w, b, dy = make(50, 768, "bf16", "bf16", 3)
    check(x, w if with_w else None, b if with_b else None, dy)


def test_leading_axes_and_row_views():
    x, w, b, dy = make(6 * 40, 768, "bf16", "bf16", 5)
    check(x.view(6, 40, 768), w, b, dy.view(6, 40, 768))
    # rows one pitch apart: a slice of a packed projection, read in place, aligned and not
    for lo in (0, 768, 1, 4):
        wide = torch.randn(6, 40, 3 * 768 + 8, device="cuda").to(torch.bfloat16)
        view = wide[..., lo:lo + 768]
        y, mean, rstd = N.layer_norm_forward(view, w.detach(), b.detach())
        y2, mean2, rstd2 = N.layer_norm_forward(view.contiguous(), w.detach(), b.detach())
        (want, _, _, _), (size, _, _, _) = reference(view, w.detach(), b.detach(), view)
        close(y, want, size, f"y of a slice at {lo}")
        assert (mean - mean2).abs().max() <= SUM * 4 and (rstd - rstd2).abs().max() <= SUM * 8 and mean.shape == (6, 40)
        check(view.detach(), w.detach().clone(), b.detach().clone(), wide[..., lo + 8:lo + 776] if lo else dy.view(6, 40, 768))
    # axes that are not one pitch apart, a transposed tensor, a broadcast row and a broadcast gradient
    t = torch.randn(40, 6, 768, device="cuda")
    check(t.transpose(0, 1), w.detach().float(), b.detach().float(), torch.randn(6, 40, 768, device="cuda"))
    check(torch.randn(96, 50, device="cuda").t(), None, None, torch.randn(50, 96, device="cuda"))
    check(torch.randn(1, 96, device="cuda").expand(9, 96).detach(), None, None, torch.randn(1, 1, device="cuda").expand(9, 96))
    check(torch.randn(96, device="cuda"), None, None, torch.randn(96, device="cuda"))


def test_no_rows():
    x = torch.empty(0, 5, 768, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    m = N.LayerNorm(768).cuda().to(torch.bfloat16)
    y = m(x)
    dx, dw, db = torch.autograd.grad(y, (x, m.weight, m.bias), torch.empty_like(y))
    assert y.shape == x.shape and dx.shape == x.shape and not dw.any() and not db.any() and dw.shape == (768,)


def test_rows_of_one_value_infinities_and_nan():
    x, w, b, dy = make(8, 768, "f32", "f32", 9)
    x[0] = 0.0
    x[1] = 5.0                       # no spread: eps alone decides, y is the bias
    x[2, 5] = float("inf")
    x[3, 6] = float("nan")
    x[4] *= 1e-20                    # squares underflow
    y, mean, rstd = N.layer_norm_forward(x, w, b)
    assert torch.equal(y[0], b) and torch.allclose(y[1], b, atol=1e-6) and torch.allclose(y[4], b, atol=1e-12)
    assert bool(torch.isnan(y[2:4]).any(1).all()) and bool(torch.isfinite(y[5:]).all())
    dx, dw, db = N.layer_norm_backward(x, dy, mean, rstd, w)
    assert bool(torch.isfinite(dx[5:]).all()) and bool(torch.isfinite(dx[:2]).all()) and bool(torch.isfinite(db).all())
    assert bool(torch.isnan(dw).any())


def test_mean_far_above_the_spread():
    """A mean of 10^4 spreads: 2^-24 of the mean is 6e-4 of a spread, which bounds what any fp32 evaluation can know of x itself; the inputs are exact
    here, so only the statistics count, and what rounding leaves of the mean is added back."""
    x, w, b, dy = make(16, 4096, "f32", "f32", 11, mean=0.0)
    x = x + 1e4
    y, _, _ = N.layer_norm_forward(x, w, b)
    (want, _, _, _), _ = reference(x, w, b, dy)
    assert float((y.double() - want).norm() / want.norm()) < 1e-5


def test_gradient_against_differences():
    """Central differences of the fp32 forward along a random direction.  Third derivatives are of order 1 / sigma^3: with steps of 2^-6 of a deviation the
    truncation is about 2^-12; the forward's rounding, 2^-22 of |y| |dy| / (2 h), is 2^-17."""
    x, w, b, dy = make(64, 500, "f32", "f32", 13)
    v = torch.randn_like(x) * x.std(1, keepdim=True)
    y, mean, rstd = N.layer_norm_forward(x, w, b)
    dx, dw, db = N.layer_norm_backward(x, dy, mean, rstd, w)
    h = 2.0 ** -6
    f = lambda *a: N.layer_norm_forward(*a)[0].double()
    d = lambda plus, minus: ((f(*plus) - f(*minus)) * dy.double()).sum(1) / (2 * h)
    num = d((x + h * v, w, b), (x - h * v, w, b))
    want = (dx.double() * v.double()).sum(1)
    scale = (dx.double().norm(dim=1) * v.double().norm(dim=1))
    assert bool(((num - want).abs() <= 2.0 ** -9 * scale).all())
    u = torch.randn_like(w)
    num = d((x, w + h * u, b), (x, w - h * u, b)).sum()
    assert abs(float(num - (dw.double() * u).sum())) <= 2.0 ** -12 * float(dw.double().norm() * u.double().norm())
    num = d((x, w, b + h * u), (x, w, b - h * u)).sum()
    assert abs(float(num - (db.double() * u).sum())) <= 2.0 ** -12 * float(db.double().norm() * u.double().norm())


def test_parts_and_repeats():
    x, w, b, dy = make(1200, 768, "bf16", "bf16", 17)
    _, mean, rstd = N.layer_norm_forward(x, w, b)
    full = N.layer_norm_backward(x, dy, mean, rstd, w)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True), (False, False, False)):
        part = N.layer_norm_backward(x, dy, mean, rstd, w, *need)
        for have, g, f in zip(need, part, full):
            assert (g is None) != have and (not have or torch.equal(g, f))
    assert all(torch.equal(a, c) for a, c in zip(full, N.layer_norm_backward(x, dy, mean, rstd, w)))
    assert N.layer_norm_backward(x, dy, mean, rstd)[1].dtype == torch.float32


def test_other_stream_and_capture():
    x, w, b, dy = make(700, 768, "bf16", "bf16", 19)
    x.requires_grad_(); w.requires_grad_(); b.requires_grad_()
    step = lambda: (lambda y: (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy))(N.layer_norm(x, w, b))
    want = [t.clone() for t in step()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    s.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    graphs = []
    for _ in range(2):                                   # two graphs over one stream's scratch, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    big = make(40000, 1024, "bf16", "bf16", 23)
    N.layer_norm_backward(big[0], big[3], *N.layer_norm_forward(*big[:3])[1:], big[1])
    for g, out in graphs + graphs:
        for t in out:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_module_matches_torch_names():
    m, t = N.LayerNorm(96), torch.nn.LayerNorm(96)
    m.load_state_dict(t.state_dict())
    m.cuda()
    x = torch.randn(10, 96, device="cuda")
    ref = t.cuda()(x)
    assert torch.allclose(m(x), ref, atol=1e-5)
    assert N.LayerNorm(96, bias=False).bias is None
