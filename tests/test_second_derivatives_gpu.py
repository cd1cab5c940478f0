"""Gradients made with create_graph are refused a second derivative by everything that they depend on.  The slope of a GELU is taken at x w + b, so
behind one they depend on the bias as well, also where the bias is all that needs a gradient; without one they do not."""
import pytest
import torch

from inferno_b200 import attention as A
from inferno_b200 import linear as L

pytestmark = pytest.mark.gpu


def bf16(*shape, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(torch.bfloat16)


def problem():
    return bf16(40, 64, seed=1), bf16(64, 128, seed=2, std=0.1), bf16(128, seed=3), bf16(128, 64, seed=4, std=0.1), bf16(64, seed=5)


def refused(grads, of):
    """Through the gradients and through a path of its own: the gradients' part must not be left out."""
    with pytest.raises(NotImplementedError, match="second derivatives"):
        torch.autograd.grad(sum((g.float() ** 2).sum() for g in grads) + (of.float() ** 2).sum(), of, retain_graph=True)


@pytest.mark.parametrize("bias_type", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("leaves", ["b", "xb", "wb", "xwb"])
def test_bias_ahead_of_gelu(leaves, bias_type):
    x, w, b, _, _ = problem()
    t = dict(x=x, w=w, b=b.to(bias_type))
    for n in leaves:
        t[n].requires_grad_()
    call = lambda: L.fused_linear(t["x"], t["w"], t["b"], "gelu")
    dy = bf16(40, 128, seed=6)
    want = torch.autograd.grad(call(), [t[n] for n in leaves], dy)
    got = torch.autograd.grad(call(), [t[n] for n in leaves], dy, create_graph=True)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    for g in got:
        assert g.requires_grad
        refused([g], t["b"])
    with pytest.raises(NotImplementedError, match="second derivatives"):
        (sum((g.float() ** 2).sum() for g in got) + (t["b"].float() ** 2).sum()).backward()


@pytest.mark.parametrize("leaves", [("b1",), ("x", "b1"), ("w1", "b1"), ("b1", "w2"), ("b1", "b2"), ("x", "w1", "b1", "w2", "b2")])
def test_first_bias_of_the_feed_forward_block(leaves):
    t = dict(zip(("x", "w1", "b1", "w2", "b2"), problem()))
    for n in leaves:
        t[n].requires_grad_()
    call = lambda: L.feed_forward(t["x"], t["w1"], t["b1"], t["w2"], t["b2"], t["x"])
    dy = bf16(40, 64, seed=7)
    want = torch.autograd.grad(call(), [t[n] for n in leaves], dy)
    got = torch.autograd.grad(call(), [t[n] for n in leaves], dy, create_graph=True)
    for n, g, c in zip(leaves, got, want):
        assert torch.equal(g, c)
        if n != "b2":                              # (db2 is the sum of dy)
            refused([g], t["b1"])


def test_a_bias_that_is_only_added_is_free():
    """Nothing depends on it, and a second path through it gives what it should."""
    x, w, b, _, _ = problem()
    for t in (x, w, b):
        t.requires_grad_()
    gx, gw = torch.autograd.grad(L.fused_linear(x, w, b, None, x.new_zeros(40, 128)), (x, w), bf16(40, 128, seed=6), create_graph=True)
    g, = torch.autograd.grad((gx.float() ** 2).sum() + (gw.float() ** 2).sum() + (b.float() ** 2).sum(), b, retain_graph=True)
    assert torch.equal(g, 2 * b.detach())
    refused([gx], w)
    refused([gw], x)


@pytest.mark.parametrize("form", ["function", "module"])
def test_plain_projection(form):
    """A projection without activation and residual refuses what one with them refuses."""
    x, w, b, _, _ = problem()
    if form == "module":
        lin = L.Linear(64, 128).cuda().to(torch.bfloat16)
        w, b, call = lin.weight, lin.bias, lambda: lin(x)
    else:
        call = lambda: L.LinearFunction.apply(x, w, b)
    leaves = (x, w, b)
    for t in leaves:
        t.requires_grad_()
    dy = bf16(40, 128, seed=6).requires_grad_()
    want = torch.autograd.grad(call(), leaves, dy)
    assert all(not g.requires_grad for g in want)
    got = torch.autograd.grad(call(), leaves, dy, create_graph=True)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    refused([got[0]], w)
    refused([got[1]], x)
    for g in got:
        refused([g], dy)
    g, = torch.autograd.grad(sum((t.float() ** 2).sum() for t in got[:2]) + (b.float() ** 2).sum(), b, retain_graph=True)      # only added: nothing depends on it
    assert torch.equal(g, 2 * b.detach())
    y = call()                                     # a gradient penalty beside the loss itself
    gx, = torch.autograd.grad(y, x, dy, create_graph=True)
    with pytest.raises(NotImplementedError, match="second derivatives"):
        (y.float().sum() + (gx.float() ** 2).sum()).backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form", ["qkv", "slices", "packed"])
def test_attention(form, dtype):
    """Gradients of the queries depend on keys and values, and the other way round."""
    dense = bf16(2, 40, 3 * 128, seed=8).to(dtype).requires_grad_()
    if form == "packed":
        leaves, call, shape = (dense,), lambda: A.causal_attention_packed(dense, 2), (2, 40, 128)
    else:
        q, k, v = (t.detach().transpose(1, 2) for t in dense.view(2, 40, 3, 2, 64).unbind(2))
        leaves = tuple((t if form == "slices" else t.contiguous()).requires_grad_() for t in (q, k, v))
        call, shape = lambda: A.causal_attention(*leaves), (2, 2, 40, 64)
    dy = bf16(*shape, seed=9).to(dtype).requires_grad_()
    want = torch.autograd.grad(call(), leaves, dy)
    assert all(not g.requires_grad for g in want)
    got = torch.autograd.grad(call(), leaves, dy, create_graph=True)
    for g, c in zip(got, want):
        assert float((g.detach().double() - c.double()).norm()) <= 1e-3 * float(c.double().norm())      # (dq is added up in an order that varies)
        for of in leaves + (dy,):
            refused([g], of)
