"""The in-situ GPT with whole blocks on this library: outputs and gradients against the plain PyTorch composition."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_block_variant_matches_torch_composition():
    """The same weights in both models, bf16.  Tolerance as for the other variants of this model: 5e-2 on each gradient (bf16 everywhere, four blocks'
    worth of roundings on either side), 2e-2 on the loss."""
    from inferno_b200.insitu_gpt import GPT
    torch.manual_seed(1)
    dev = torch.device("cuda")
    cfg = dict(vocab=512, T=256, C=128, H=2, layers=2)
    block = GPT(attn_impl="ib200_block", **cfg).to(dev).to(torch.bfloat16)
    ref = GPT(attn_impl="torch", **cfg).to(dev).to(torch.bfloat16)
    own = {n: n.replace(".ff1.", ".ff.ff1.").replace(".ff2.", ".ff.ff2.") for n in ref.state_dict()}
    turned = lambda n: n.endswith(".weight") and any(k in n for k in (".wqkv.", ".wout.", ".ff1.", ".ff2."))      # stored [in, out] here
    sd = block.state_dict()
    ref.load_state_dict({n: sd[m].t().contiguous() if turned(n) else sd[m] for n, m in own.items()})
    idx = torch.randint(0, cfg["vocab"], (2, cfg["T"]), device=dev)
    tgt = torch.randint(0, cfg["vocab"], (2, cfg["T"]), device=dev)
    losses = []
    for m in (block, ref):
        loss = torch.nn.functional.cross_entropy(m(idx).float().view(-1, cfg["vocab"]), tgt.view(-1))
        loss.backward()
        losses.append(float(loss.detach()))
    assert abs(losses[0] - losses[1]) < 2e-2
    params = dict(block.named_parameters())
    for n, p in ref.named_parameters():
        g = params[own[n]].grad.float()
        g = g.t() if turned(n) else g
        rel = float((g - p.grad.float()).norm() / p.grad.float().norm())
        assert rel < 5e-2, (n, rel)


def test_block_variant_runs_in_the_harness_and_without_gradients():
    from inferno_b200.insitu_gpt import GPT, run
    out = run(layers=2, C=256, H=4, vocab=1024, T=512, B=2, steps=2, warmup=1, attn_impl="ib200_block")
    assert out["config"]["attn_impl"] == "ib200_block" and out["attn_fwd_ms"] > 0 and out["step_ms"] > 0
    m = GPT(vocab=512, T=64, C=128, H=2, layers=2, attn_impl="ib200_block").cuda().to(torch.bfloat16)
    idx = torch.randint(0, 512, (1, 64), device="cuda")
    full = m(idx).detach()
    with torch.no_grad():
        for n in (1, 7, 33):                   # prompts short enough for the few-row kernel, and longer ones
            part = m(idx[:, :n])
            # causal: a prefix gives the prefix of the outputs, up to bf16 roundings in a different summation order
            assert float((part.float() - full[:, :n].float()).norm() / full[:, :n].float().norm()) < 2e-2
