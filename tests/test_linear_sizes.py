"""The sizes at which the plain projection has to say no, or to do nothing: what its kernels cannot number, and no rows at all."""
import pytest
import torch

from inferno_b200 import linear as L

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def z(*s, device):
    return torch.zeros(s, dtype=torch.bfloat16, device=device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("M", [2**31 - 256, 2**31, 2**32 + 16, 2**33])
def test_rows_that_an_int_cannot_number(built_lib, device, M):
    """One row, over and over, so that nothing is allocated for them.  2^32 + 16 rows are not 16."""
    x, dy, w = z(1, 8, device=device).expand(M, 8), z(1, 8, device=device).expand(M, 8), z(8, 8, device=device)
    lin = L.Linear(8, 8).to(device=device, dtype=torch.bfloat16)
    for call in (lambda: L.linear_forward(x, w), lambda: L.LinearFunction.apply(x, w, None), lambda: lin(x), lambda: L.linear_backward(x, w, dy)):
        with pytest.raises(ValueError, match="too many rows"):
            call()


@pytest.mark.parametrize("device", DEVICES)
def test_weights_that_are_empty_or_too_wide(built_lib, device):
    for K, N in ((0, 8), (8, 0), (8, 2**31 - 256), (2**32 + 8, 8)):
        w, x, dy = z(1, 1, device=device).expand(K, N), z(1, 1, device=device).expand(4, K), z(1, 1, device=device).expand(4, N)
        for call in (lambda: L.linear_forward(x, w), lambda: L.LinearFunction.apply(x, w, None), lambda: L.linear_backward(x, w, dy)):
            with pytest.raises(ValueError, match="rows and columns"):
                call()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 64), (3, 0, 64), (0, 5, 64)])
@pytest.mark.parametrize("bias_type", [torch.bfloat16, torch.float32, None])
def test_no_rows(shape, bias_type):
    """An empty output, an empty dx, and gradients of zero, as with an activation or a residual."""
    x, w = z(*shape, device="cuda").requires_grad_(), torch.ones(64, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    b = None if bias_type is None else torch.ones(128, device="cuda", dtype=bias_type, requires_grad=True)
    y = L.LinearFunction.apply(x, w, b)
    assert y.shape == shape[:-1] + (128,) and L.linear_forward(x.detach(), w.detach(), b).shape == y.shape
    leaves = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, leaves, torch.empty_like(y))
    for t, g in zip(leaves, grads):
        assert g.shape == t.shape and g.dtype == t.dtype and not g.any()
    dx, dw, db = L.linear_backward(x.detach(), w.detach(), torch.empty_like(y))
    assert dx.shape == x.shape and not dw.any() and not db.any() and db.dtype == torch.float32
    for g, have in zip(L.linear_backward(x.detach(), w.detach(), torch.empty_like(y), False, True, False), (False, True, False)):
        assert (g is not None) == have


@pytest.mark.gpu
def test_module_without_rows_in_every_form():
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)
    for lin in (L.Linear(64, 128), L.Linear(64, 128, bias=False), L.Linear(64, 128, activation="gelu")):
        lin = lin.cuda().to(torch.bfloat16)
        for res in (None, torch.empty(0, 128, device="cuda", dtype=torch.bfloat16)):
            y = lin(x, res)
            assert y.shape == (0, 128)
            y.sum().backward()
            assert all(not p.grad.any() for p in lin.parameters())


def test_module_saved_before_it_had_an_activation(built_lib):
    """A module that was pickled whole has only the attributes of its time."""
    import pickle
    lin = L.Linear(32, 64).bfloat16()
    del lin.__dict__["activation"]
    lin = pickle.loads(pickle.dumps(lin))
    x = z(4, 32, device="cpu")
    for call in (lambda: lin(x), lambda: lin(x, z(4, 64, device="cpu"))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
