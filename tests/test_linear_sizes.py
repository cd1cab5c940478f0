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
