"""The scratch of the feed-forward block's backward: no more than is used, and nothing past its end."""
import pytest
import torch

from inferno_b200 import _capi


def up(n):
    return (n + 255) // 256 * 256


def without_accumulators(M, C, H):
    """Column sums of dy and of dz, and dz."""
    return up(128 * C * 4) + up((M + 31) // 32 * H * 4) + up(M * H * 2)


@pytest.mark.parametrize("M,C,H", [(16384, 2048, 8192), (4096, 4096, 16384), (1100, 2560, 4096), (1025, 64, 256 * 149), (200000, 256, 38400)])
def test_weight_gradients_that_are_not_cut_have_no_accumulators(built_lib, M, C, H):
    """More tiles of dW than two rounds of the GPU's pairs of SMs: it runs in whole tiles."""
    assert _capi.lib().ib200_feed_forward_workspace_bytes(M, C, H) == without_accumulators(M, C, H)


@pytest.mark.parametrize("M,C,H", [(8192, 1024, 4096), (1100, 64, 256), (16384, 768, 2056)])
def test_weight_gradients_that_are_cut_keep_them(built_lib, M, C, H):
    assert _capi.lib().ib200_feed_forward_workspace_bytes(M, C, H) == without_accumulators(M, C, H) + 2 * up(C * H * 4)


@pytest.mark.gpu
@pytest.mark.parametrize("M,C,H", [(1100, 2560, 4096), (300, 264, 520), (2000, 264, 520), (1, 2048, 8192), (33, 64, 256 * 149)])
@pytest.mark.parametrize("asked", [(1, 1, 1, 1, 1), (0, 1, 0, 0, 0), (0, 0, 0, 1, 0), (1, 0, 0, 1, 0), (0, 0, 1, 0, 1), (0, 1, 0, 1, 0)])
def test_nothing_past_the_end(M, C, H, asked):
    g = torch.Generator(device="cuda").manual_seed(M + C)
    bf16 = lambda *s, std=1.0: (torch.randn(*s, device="cuda", generator=g) * std).to(torch.bfloat16)
    x, w1, w2, h, dy = bf16(M, C), bf16(C, H, std=C ** -0.5), bf16(H, C, std=H ** -0.5), bf16(M, H), bf16(M, C, std=0.1)
    slope = torch.rand(M, H, device="cuda", generator=g).half()
    dz = (dy.double() @ w2.double().t()) * slope.double()
    want = (dz @ w1.double().t(), x.double().t() @ dz, dz.sum(0), h.double().t() @ dy.double(), dy.double().sum(0))
    outs = [torch.empty(s, device="cuda", dtype=torch.bfloat16) if a else None for a, s in zip(asked, ((M, C), (C, H), (H,), (H, C), (C,)))]
    need = _capi.lib().ib200_feed_forward_workspace_bytes(M, C, H)
    ws = torch.full((need + 4096,), 0xA5, device="cuda", dtype=torch.uint8)
    ptr = lambda t: None if t is None else t.data_ptr()
    rc = _capi.lib().ib200_feed_forward_bwd(x.data_ptr(), w1.data_ptr(), slope.data_ptr(), h.data_ptr(), w2.data_ptr(), dy.data_ptr(), ptr(outs[0]), ptr(outs[1]),
                                            ptr(outs[2]), _capi.DTYPE_BF16, ptr(outs[3]), ptr(outs[4]), _capi.DTYPE_BF16, M, C, H, ws.data_ptr(), need,
                                            torch.cuda.current_stream().cuda_stream)
    assert rc == _capi.OK
    assert bool((ws[need:] == 0xA5).all())
    for o, wnt in zip(outs, want):      # two roundings to bf16 (dz's and the result's), the slope's is in both; the sums of dz may cancel
        if o is not None:
            assert float((o.double() - wnt).norm()) <= 1.1 * 2.0 ** 0.5 * 2.0 ** -8 * float(wnt.norm())
