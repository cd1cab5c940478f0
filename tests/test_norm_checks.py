"""What layer norm refuses, before anything is allocated or launched.  Shapes come ahead of the device, so the same cases run on CPU tensors."""
import math

import pytest
import torch

from inferno_b200 import _capi
from inferno_b200 import norm as N

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_shapes(built_lib, device):
    z = lambda *s, dt=torch.float32: torch.zeros(s, device=device, dtype=dt)
    for x in (z(), z(3, 0)):
        with pytest.raises(ValueError, match="last axis"):
            N.layer_norm(x)
    for w in (z(4), z(0), z(1, 8), z()):
        with pytest.raises(ValueError, match="weight and bias"):
            N.layer_norm(z(3, 8), w)
        with pytest.raises(ValueError, match="weight and bias"):
            N.layer_norm_forward(z(3, 8), None, w)
        with pytest.raises(ValueError, match="weight and bias"):
            N.layer_norm_backward(z(3, 8), z(3, 8), z(3), z(3), w)


def test_a_cpu_tensor_is_refused(built_lib):
    x = torch.zeros(3, 8)
    for call in (lambda: N.layer_norm(x), lambda: N.layer_norm_forward(x), lambda: N.layer_norm_backward(x, x, x[:, 0], x[:, 0]), lambda: N.LayerNorm(8)(x)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(TypeError):
        N.layer_norm([1.0, 2.0])


@pytest.mark.gpu
def test_types_devices_and_statistics():
    x, w = torch.zeros(3, 8, device="cuda"), torch.ones(8, device="cuda")
    for bad in (x.half(), x.double(), x.int()):
        with pytest.raises(TypeError, match="float32 or bfloat16"):
            N.layer_norm(bad)
        with pytest.raises(TypeError, match="float32 or bfloat16"):
            N.layer_norm(x, bad[0])
    with pytest.raises(TypeError, match="same dtype"):
        N.layer_norm(x, w, w.bfloat16())
    with pytest.raises(ValueError, match="device"):
        N.layer_norm(x, w.cpu())
    for eps in (-1e-5, math.inf, math.nan):
        with pytest.raises(ValueError, match="eps"):
            N.layer_norm(x, w, eps=eps)
    s = torch.zeros(3, device="cuda")
    for dy in (x[:2], x[:, :4], x.cpu()):
        with pytest.raises(ValueError, match="dy must"):
            N.layer_norm_backward(x, dy, s, s)
    with pytest.raises(TypeError, match="dy must"):
        N.layer_norm_backward(x, x.bfloat16(), s, s)
    for bad in (s[:2], s.double(), s.cpu()):
        with pytest.raises(ValueError, match="mean and rstd"):
            N.layer_norm_backward(x, x, bad, s)
    with pytest.raises(_capi.Ib200Error) as e:
        N.layer_norm(torch.zeros(1, 8193, device="cuda"))
    assert e.value.status == _capi.ERR_UNSUPPORTED
    with pytest.raises(_capi.Ib200Error):
        N.layer_norm(torch.zeros(1, 16385, device="cuda", dtype=torch.bfloat16))
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level():
        with pytest.raises(NotImplementedError):
            N.layer_norm(fwAD.make_dual(x, x))


def test_c_abi_validation(built_lib):
    """Fake addresses, never dereferenced: every refusal happens on the host."""
    L = _capi.lib()
    F, B = _capi.DTYPE_F32, _capi.DTYPE_BF16
    x, w, b, y, m, r, dy = (0x10000 * i for i in range(1, 8))
    fwd = lambda x=x, w=w, p=F, y=y, m=m, r=r, M=4, C=64, eps=1e-5, dt=F, pitch=64: L.ib200_layer_norm_fwd(x, pitch, w, b, p, y, m, r, M, C, eps, dt, None)
    bad = _capi.ERR_INVALID_ARGUMENT
    assert fwd(x=None) == bad and fwd(y=None) == bad and fwd(m=None) == bad and fwd(M=0) == bad and fwd(C=0) == bad and fwd(M=-1) == bad
    assert fwd(eps=-1.0) == bad and fwd(eps=math.nan) == bad and fwd(dt=3) == bad and fwd(p=2) == bad and fwd(pitch=-8) == bad
    assert fwd(C=8193) == _capi.ERR_UNSUPPORTED and fwd(C=16385, dt=B) == _capi.ERR_UNSUPPORTED
    assert fwd(x=x + 2) == _capi.ERR_MISALIGNED and fwd(x=x + 1, dt=B) == _capi.ERR_MISALIGNED and fwd(w=w + 2) == _capi.ERR_MISALIGNED
    need = L.ib200_layer_norm_workspace_bytes(1000, 64, F)
    assert need > 0 and need % (2 * 64 * 4) == 0
    assert L.ib200_layer_norm_workspace_bytes(0, 64, F) == 0 and L.ib200_layer_norm_workspace_bytes(4, 16385, B) == 0
    bwd = lambda x=x, dy=dy, m=m, ws=0x900000, n=need, dw=0xA0000, dx=0xB0000: L.ib200_layer_norm_bwd(x, 64, w, dy, 64, m, r, dx, dw, 0xC0000, F, 1000, 64, F, ws, n, None)
    assert bwd(x=None) == bad and bwd(dy=None) == bad and bwd(m=None) == bad
    assert bwd(ws=None) == _capi.ERR_WORKSPACE and bwd(n=need - 1) == _capi.ERR_WORKSPACE and bwd(ws=0x900008) == _capi.ERR_WORKSPACE
    assert bwd(dw=0xA0002) == _capi.ERR_MISALIGNED
    assert L.ib200_layer_norm_bwd(x, 64, w, dy, 64, m, r, None, None, None, F, 1000, 64, F, None, 0, None) == _capi.OK
    import torch
    if not torch.cuda.is_available():
        assert fwd() == _capi.ERR_NO_DEVICE and bwd() == _capi.ERR_NO_DEVICE
