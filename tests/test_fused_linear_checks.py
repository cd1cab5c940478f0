"""What the fused projections and the feed-forward block refuse, before anything is allocated or launched.  Shapes come ahead of the device."""
import pytest
import torch

from inferno_b200 import _capi
from inferno_b200 import linear as L

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def z(*s, device, dtype=torch.bfloat16):
    return torch.zeros(s, dtype=dtype, device=device)


@pytest.mark.parametrize("device", DEVICES)
def test_shapes(built_lib, device):
    x, w, b = z(16, 32, device=device), z(32, 64, device=device), z(64, device=device)
    for bad in (z(16, 64, device=device), z(32, 16, device=device), z(device=device), z(33, device=device)):
        for call in (lambda: L.fused_linear(bad, w, b, "gelu"), lambda: L.fused_linear_backward(bad, w, z(16, 64, device=device)),
                     lambda: L.feed_forward(bad, w, b, z(64, 32, device=device), None)):
            with pytest.raises(ValueError, match="last axis"):
                call()
    for bad in (z(63, device=device), z(1, 64, device=device), z(0, device=device), z(device=device)):
        with pytest.raises(ValueError, match="bias"):
            L.fused_linear(x, w, bad, "gelu")
        with pytest.raises(ValueError, match="bias"):
            L.feed_forward(x, w, bad, z(64, 32, device=device), None)
    for bad in (z(16, 63, device=device), z(8, 64, device=device), z(64, device=device), z(1, 16, 64, device=device), z(1, 64, device=device)):
        with pytest.raises(ValueError, match="residual"):
            L.fused_linear(x, w, b, None, bad)
        with pytest.raises(ValueError, match="dy must"):
            L.fused_linear_backward(x, w, bad)
    for bad in (z(64, 64, device=device), z(32, 64, device=device), z(64, 40, device=device), z(64, device=device)):
        with pytest.raises(ValueError, match="w2|last axis"):
            L.feed_forward(x, w, b, bad, None)
    with pytest.raises(ValueError, match="residual"):
        L.feed_forward(x, w, b, z(64, 32, device=device), None, z(16, 64, device=device))
    for M in (2**31 - 256, 2**31, 2**33):                                      # one row, over and over: nothing is allocated for them
        rows = z(1, 32, device=device).expand(M, 32)
        for call in (lambda: L.fused_linear(rows, w, b, "gelu"), lambda: L.feed_forward(rows, w, b, z(64, 32, device=device), None)):
            with pytest.raises(ValueError, match="too many rows"):
                call()
    with pytest.raises(ValueError, match="rows and columns"):
        L.fused_linear(z(4, 0, device=device), z(0, 8, device=device))
    for name in ("relu", "GELU", "", 3, True):
        with pytest.raises(ValueError, match="activation"):
            L.fused_linear(x, w, b, name)


def test_a_cpu_tensor_is_refused(built_lib):
    x, w, b = z(16, 32, device="cpu"), z(32, 64, device="cpu"), z(64, device="cpu")
    for call in (lambda: L.fused_linear(x, w, b, "gelu"), lambda: L.fused_linear_forward(x, w), lambda: L.fused_linear_backward(x, w, z(16, 64, device="cpu")),
                 lambda: L.feed_forward(x, w, b, w.t(), None), lambda: L.Linear(32, 64, activation="gelu").bfloat16()(x), lambda: L.FeedForward(32, 64).bfloat16()(x)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


@pytest.mark.gpu
def test_types_devices_and_sizes():
    d = "cuda"
    x, w, b, r = z(16, 32, device=d), z(32, 64, device=d), z(64, device=d), z(16, 64, device=d)
    for call in (lambda t: L.fused_linear(t(x), w, b, "gelu"), lambda t: L.fused_linear(x, t(w), b, "gelu"), lambda t: L.fused_linear(x, w, b, None, t(r)),
                 lambda t: L.fused_linear_backward(x, w, t(r)), lambda t: L.feed_forward(x, w, b, t(z(64, 32, device=d)), None)):
        for t in (lambda v: v.float(), lambda v: v.half()):
            with pytest.raises(TypeError, match="bfloat16"):
                call(t)
        with pytest.raises((ValueError, RuntimeError)):
            call(lambda v: v.cpu())
    with pytest.raises(TypeError, match="bias"):
        L.fused_linear(x, w, b.half(), "gelu")
    with pytest.raises(ValueError, match="the bias is on cpu"):
        L.fused_linear(x, w, b.cpu(), "gelu")
    for bad in (None, r, r.half()[:8], r.half().cpu()):
        with pytest.raises((ValueError, TypeError)):
            L.fused_linear_backward(x, w, r, bad, "gelu")
    for K, N in ((30, 64), (32, 60)):
        with pytest.raises(_capi.Ib200Error) as e:
            L.fused_linear(z(16, K, device=d), z(K, N, device=d), None, "gelu")
        assert e.value.status == _capi.ERR_UNSUPPORTED
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level():
        with pytest.raises(NotImplementedError):
            L.fused_linear(fwAD.make_dual(x, x), w, b, "gelu")


def test_c_abi_validation(built_lib):
    """Fake addresses, never dereferenced: every refusal happens on the host."""
    C = _capi.lib()
    bad, B = _capi.ERR_INVALID_ARGUMENT, _capi.DTYPE_BF16
    x, w, b, r, y, p, ws = (0x100000 * i for i in range(1, 8))
    fwd = lambda x=x, w=w, b=b, bd=B, r=r, act=1, y=y, p=p, M=16, K=32, N=64, ws=ws, n=1 << 20: C.ib200_fused_linear_fwd(x, w, b, bd, r, act, y, p, M, K, N, ws, n, None)
    assert fwd(x=None) == bad and fwd(w=None) == bad and fwd(y=None) == bad and fwd(bd=2) == bad and fwd(act=2) == bad and fwd(act=-1) == bad
    assert fwd(act=0) == bad and fwd(M=0) == bad and fwd(K=-8) == bad and fwd(N=0) == bad            # a slope without an activation
    assert fwd(K=36) == _capi.ERR_UNSUPPORTED and fwd(N=60) == _capi.ERR_UNSUPPORTED
    for k in ("x", "w", "y", "r", "p", "b"):
        assert fwd(**{k: 0x900008}) == _capi.ERR_MISALIGNED
    assert fwd(ws=0x900008) == _capi.ERR_WORKSPACE
    size = C.ib200_fused_linear_workspace_bytes
    assert size(16, 32, 64, 1, _capi.PASS_BWD) >= size(16, 32, 64, 0, _capi.PASS_BWD) + 16 * 64 * 2 and size(0, 32, 64, 1, 1) == 0
    need = size(16, 32, 64, 1, _capi.PASS_BWD)
    bwd = lambda x=x, w=w, dy=r, p=p, act=1, dx=y, dbt=B, M=16, N=64, ws=ws, n=need: C.ib200_fused_linear_bwd(x, w, dy, p, act, dx, 0x800000, 0x900000, dbt, M, 32, N, ws, n, None)
    assert bwd(x=None) == bad and bwd(dy=None) == bad and bwd(p=None) == bad and bwd(act=0) == bad and bwd(dbt=5) == bad and bwd(M=0) == bad
    assert bwd(ws=None) == _capi.ERR_WORKSPACE and bwd(n=need - 1) == _capi.ERR_WORKSPACE and bwd(ws=ws + 8) == _capi.ERR_WORKSPACE
    assert bwd(p=p + 8) == _capi.ERR_MISALIGNED and bwd(N=60, n=1 << 24) == _capi.ERR_UNSUPPORTED
    need = C.ib200_feed_forward_workspace_bytes(16, 32, 64)
    assert need > 2 * 32 * 64 * 4 and C.ib200_feed_forward_workspace_bytes(0, 32, 64) == 0
    ff = lambda x=x, p=p, dy=r, d1=B, M=16, Cc=32, n=need, ws=ws: C.ib200_feed_forward_bwd(x, w, p, 0xA00000, 0xB00000, dy, 0xC00000, 0xD00000, 0xE00000, d1, 0xF00000,
                                                                                         0x1000000, B, M, Cc, 64, ws, n, None)
    assert ff(x=None) == bad and ff(p=None) == bad and ff(dy=None) == bad and ff(d1=9) == bad and ff(M=0) == bad
    assert ff(Cc=36, n=1 << 24) == _capi.ERR_UNSUPPORTED and ff(n=need - 1) == _capi.ERR_WORKSPACE and ff(ws=None) == _capi.ERR_WORKSPACE
    if not torch.cuda.is_available():
        assert fwd() in (_capi.ERR_NO_DEVICE, _capi.ERR_CUDA) and bwd() in (_capi.ERR_NO_DEVICE, _capi.ERR_CUDA) and ff() == _capi.ERR_NO_DEVICE


def test_c_abi_sizes_at_the_end_of_an_int(built_lib):
    """Fake addresses again: sizes whose tiles or rows an int cannot number are refused, and no size makes a workspace's formula divide by zero."""
    C = _capi.lib()
    big, un = 2**31 - 1, _capi.ERR_UNSUPPORTED
    fwd = lambda M, K, N: C.ib200_fused_linear_fwd(0x100000, 0x200000, None, 0, None, 1, 0x300000, None, M, K, N, None, 0, None)
    bwd = lambda M, K, N, db=0x700000: C.ib200_fused_linear_bwd(0x100000, 0x200000, 0x300000, 0x400000, 1, 0x500000, 0x600000, db, 0, M, K, N, 0x800000, 2**63, None)
    ff = lambda M, Cc, H, d1=0xA00000: C.ib200_feed_forward_bwd(0x100000, 0x200000, 0x300000, 0x400000, 0x500000, 0x600000, 0x700000, 0x800000, d1, 0, 0x900000, 0xB00000, 0, M, Cc,
                                                               H, 0xC00000, 2**63, None)
    for M, K, N in ((big, 64, 64), (64, big - 7, 64), (64, 64, big - 7), (2**31 - 256, 64, 64), (2**30, 64, 2**30)):
        assert fwd(M, K, N) == un, (M, K, N)
    for M, K, N in ((big, 64, 64), (64, big - 7, 64), (64, 64, big - 7), (2**31 - 256, 64, 64)):
        assert bwd(M, K, N) == un and ff(M, K, N) == un, (M, K, N)
    assert fwd(33, 2**31 - 260, 64) == un                                         # not a multiple of 8
    for M in (1, 33, 2**24, big):
        for K in (8, 2**24, big):
            for N in (8, 2**24, big):
                for act in (0, 1):
                    C.ib200_fused_linear_workspace_bytes(M, K, N, act, _capi.PASS_FWD)
                    assert C.ib200_fused_linear_workspace_bytes(M, K, N, act, _capi.PASS_BWD) > 0
                assert C.ib200_feed_forward_workspace_bytes(M, K, N) > 0
    assert bwd(16, 32, 64, db=0x700002) == _capi.ERR_MISALIGNED and ff(16, 32, 64, d1=0xA00001) == _capi.ERR_MISALIGNED
