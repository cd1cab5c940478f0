"""The operators of a transformer block around its attention, as timed cases: layer norm, a projection with bias, GELU and
residual in its epilogue, and the feed-forward block that is made of two of them.

Kinds of case:
  ln    `layer_norm`: y, and with step the gradients of x, weight and bias
  lin   `fused_linear`: y = act(x w + b) + residual, and with step the gradients of x, w, b and residual
  ff    `feed_forward`: y = gelu(x w1 + b1) w2 + b2 + residual, and with step the gradients of all of them
GELU is the tanh form throughout.
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}
_EPS = 1e-5


def listed():
    return [
        # the norm of one decoded token: latency is all there is
        dict(name="ln_token", kind="ln", M=1, C=768, dtype="bf16", step=False),
        # a norm of the 12-layer GPT at its training batch
        dict(name="ln_gpt_step", kind="ln", M=16384, C=768, dtype="bf16", step=True),
        # fp32 training on a ragged batch with a width that no power of two divides evenly
        dict(name="ln_ragged_step_f32", kind="ln", M=2331, C=1000, dtype="f32", step=True),
        # a wide model's norm over a long batch
        dict(name="ln_wide_step", kind="ln", M=16384, C=8192, dtype="bf16", step=True),
        # the up projection of a few tokens that are decoded together
        dict(name="lin_gelu_tokens", kind="lin", M=5, K=1024, N=4096, act=True, res=False, step=False),
        # an output projection of a ragged prompt, added to the residual stream
        dict(name="lin_residual_prompt", kind="lin", M=777, K=1000, N=2008, act=False, res=True, step=False),
        # the attention's output projection of the 12-layer GPT at its training batch, with the residual
        dict(name="lin_residual_step", kind="lin", M=16384, K=768, N=768, act=False, res=True, step=True),
        # an up projection with its GELU, trained
        dict(name="lin_gelu_step", kind="lin", M=8192, K=1024, N=4096, act=True, res=False, step=True),
        # the feed-forward block of one decoded token: the weights' bytes are what it costs
        dict(name="ff_token", kind="ff", M=1, C=2048, H=8192, res=True, step=False),
        # scoring one prompt of odd length
        dict(name="ff_prompt", kind="ff", M=1023, C=1024, H=4096, res=True, step=False),
        # the feed-forward block of a small model, trained
        dict(name="ff_step", kind="ff", M=8192, C=1024, H=4096, res=True, step=True),
        # the largest: a wider model's feed-forward block over a whole batch
        dict(name="ff_large_step", kind="ff", M=16384, C=2048, H=8192, res=True, step=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _features(rng, lo, hi):
    """Feature sizes: multiples of 8, half of them multiples of 64."""
    n = _log_int(rng, lo, hi)
    unit = 64 if n >= 256 and rng.random() < 0.5 else 8
    return max(unit, n // unit * unit)


def draw(rng):
    kind = rng.choice(["ln", "ln", "lin", "lin", "ff"])
    step = rng.random() < 0.6
    M = _log_int(rng, 1, 16384)
    if kind == "ln":
        C = _log_int(rng, 64, 8192) if rng.random() < 0.3 else _features(rng, 64, 8192)
        return dict(kind="ln", M=M, C=C, dtype=rng.choice(["bf16", "f32"]) if C <= 4096 else "bf16", step=step)
    if kind == "lin":
        act = rng.random() < 0.5
        return dict(kind="lin", M=M, K=_features(rng, 64, 4096), N=_features(rng, 64, 4096), act=act, res=not act or rng.random() < 0.3, step=step)
    C = _features(rng, 128, 2048)
    return dict(kind="ff", M=M, C=C, H=4 * C, res=rng.random() < 0.8, step=step)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)

    M, step = case["M"], case["step"]
    s = dict(case)
    if case["kind"] == "ln":
        C, dt = case["C"], _DT[case["dtype"]]
        # a residual stream: rows of different size, and a mean of their own
        x = torch.randn(M, C, device="cuda", generator=g)
        x = x * torch.exp(0.5 * torch.randn(M, 1, device="cuda", generator=g)) + 0.3 * torch.randn(M, 1, device="cuda", generator=g)
        s["x"] = x.to(dt)
        s["weight"] = (1.0 + 0.2 * torch.randn(C, device="cuda", generator=g)).to(dt)
        s["bias"] = normal(C, std=0.1, dtype=dt)
        leaves = ["x", "weight", "bias"]
        out = (M, C)
    elif case["kind"] == "lin":
        K, N = case["K"], case["N"]
        s["x"], s["w"], s["b"] = normal(M, K), normal(K, N, std=K ** -0.5), normal(N, std=0.1)
        s["residual"] = normal(M, N) if case["res"] else None
        leaves = ["x", "w", "b"] + (["residual"] if case["res"] else [])
        out, dt = (M, N), torch.bfloat16
    else:
        C, H = case["C"], case["H"]
        s["x"] = normal(M, C)
        s["w1"], s["b1"] = normal(C, H, std=C ** -0.5), normal(H, std=0.1)
        s["w2"], s["b2"] = normal(H, C, std=H ** -0.5), normal(C, std=0.1)
        s["residual"] = normal(M, C) if case["res"] else None
        leaves = ["x", "w1", "b1", "w2", "b2"] + (["residual"] if case["res"] else [])
        out, dt = (M, C), torch.bfloat16
    if step:
        s["dy"] = normal(*out, std=0.1, dtype=dt)
        for name in leaves:
            s[name].requires_grad_()
    s["leaves"] = leaves
    return s


# ---- the plain forms: 32 bits, each result rounded once at the end ------------------------------

def _gelu(z):
    u = 0.7978845608028654 * (z + 0.044715 * z * z * z)
    return z / (1 + torch.exp(-2 * u))


def _gelu_slope(z):
    u = 0.7978845608028654 * (z + 0.044715 * z * z * z)
    du = 0.7978845608028654 * (1 + 3 * 0.044715 * z * z)
    s = 1 / (1 + torch.exp(-2 * u))
    return s + 2 * z * du * s * (1 - s)


def _plain_ln(s):
    x, w, b = s["x"].detach().float(), s["weight"].detach().float(), s["bias"].detach().float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    r = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + _EPS)
    xh = d * r
    dt = s["x"].dtype
    y = (xh * w + b).to(dt)
    if not s["step"]:
        return y
    dy = s["dy"].float()
    g = dy * w
    dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return y, dx.to(dt), (dy * xh).sum(0).to(dt), dy.sum(0).to(dt)


def _plain_lin(s):
    dt = s["x"].dtype
    x, w, b = s["x"].detach().float(), s["w"].detach().float(), s["b"].detach().float()
    z = x @ w + b
    y = _gelu(z) if s["act"] else z
    if s["res"]:
        y = y + s["residual"].detach().float()
    if not s["step"]:
        return y.to(dt)
    dy = s["dy"].float()
    dz = dy * _gelu_slope(z) if s["act"] else dy
    out = [y, dz @ w.t(), x.t() @ dz, dz.sum(0)] + ([dy] if s["res"] else [])
    return tuple(t.to(dt) for t in out)


def _plain_ff(s):
    dt = s["x"].dtype
    x, w1, b1, w2, b2 = (s[k].detach().float() for k in ("x", "w1", "b1", "w2", "b2"))
    z = x @ w1 + b1
    h = _gelu(z)
    y = h @ w2 + b2
    if s["res"]:
        y = y + s["residual"].detach().float()
    if not s["step"]:
        return y.to(dt)
    dy = s["dy"].float()
    dz = (dy @ w2.t()) * _gelu_slope(z)
    out = [y, dz @ w1.t(), x.t() @ dz, dz.sum(0), h.t() @ dy, dy.sum(0)] + ([dy] if s["res"] else [])
    return tuple(t.to(dt) for t in out)


def _own(s):
    from inferno_b200.linear import feed_forward, fused_linear
    from inferno_b200.norm import layer_norm
    if s["kind"] == "ln":
        y = layer_norm(s["x"], s["weight"], s["bias"], eps=_EPS)
    elif s["kind"] == "lin":
        y = fused_linear(s["x"], s["w"], s["b"], activation="gelu" if s["act"] else None, residual=s["residual"])
    else:
        y = feed_forward(s["x"], s["w1"], s["b1"], s["w2"], s["b2"], residual=s["residual"])
    if not s["step"]:
        return y
    return (y.detach(),) + torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["dy"])


def run(state):
    if own:
        return _own(state)
    return {"ln": _plain_ln, "lin": _plain_lin, "ff": _plain_ff}[state["kind"]](state)


# ---- from the definition, in 64 bits ---------------------------------------------------------------

def _act64(z):
    """gelu and its derivative by way of the hyperbolic tangent."""
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * z * (1.0 + 0.044715 * z.square()))
    return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t.square()) * c * (1.0 + 0.134145 * z.square())


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    step = case["step"]
    if case["kind"] == "ln":
        C = case["C"]
        var, mean = torch.var_mean(d["x"], dim=1, correction=0, keepdim=True)
        rstd = torch.rsqrt(var + _EPS)
        xh = (d["x"] - mean) * rstd
        y = torch.addcmul(d["bias"], xh, d["weight"])
        if not step:
            return y
        wdy = d["dy"] * d["weight"]
        c1 = (wdy * xh).sum(1, keepdim=True) / C
        c2 = wdy.sum(1, keepdim=True) / C
        return y, (wdy - c2 - xh * c1) * rstd, torch.einsum("mc,mc->c", d["dy"], xh), torch.einsum("mc->c", d["dy"])
    if case["kind"] == "lin":
        z = torch.addmm(d["b"], d["x"], d["w"])
        y, slope = _act64(z) if case["act"] else (z, torch.ones_like(z))
        y = y + d["residual"] if case["res"] else y
        if not step:
            return y
        dz = slope * d["dy"]
        return (y, torch.einsum("mn,kn->mk", dz, d["w"]), torch.einsum("mk,mn->kn", d["x"], dz), torch.einsum("mn->n", dz)) + ((d["dy"],) if case["res"] else ())
    z = torch.addmm(d["b1"], d["x"], d["w1"])
    h, slope = _act64(z)
    y = torch.addmm(d["b2"], h, d["w2"])
    y = y + d["residual"] if case["res"] else y
    if not step:
        return y
    dz = torch.einsum("mc,hc->mh", d["dy"], d["w2"]) * slope
    return (y, torch.einsum("mh,ch->mc", dz, d["w1"]), torch.einsum("mc,mh->ch", d["x"], dz), torch.einsum("mh->h", dz),
            torch.einsum("mh,mc->hc", h, d["dy"]), torch.einsum("mc->c", d["dy"])) + ((d["dy"],) if case["res"] else ())


def work(case):
    """Each input once, each output once.  A residual's gradient is dy itself: neither written nor read again."""
    M, step = case["M"], case["step"]
    if case["kind"] == "ln":
        C, e = case["C"], _SIZE[case["dtype"]]
        bytes_ = e * (2 * M * C + 2 * C)
        flops = 8 * M * C
        if step:
            bytes_ += e * (2 * M * C + 2 * C)       # dy in, dx out, and the gradients of weight and bias
            flops += 14 * M * C
        return {"bytes": bytes_, "flops": flops}
    if case["kind"] == "lin":
        K, N = case["K"], case["N"]
        bytes_ = 2 * (M * K + K * N + N + M * N * (2 if case["res"] else 1))
        flops = 2 * M * K * N
        if step:
            bytes_ += 2 * (M * N + M * K + K * N + N)
            flops *= 3
        return {"bytes": bytes_, "flops": flops}
    C, H = case["C"], case["H"]
    bytes_ = 2 * (M * C * (3 if case["res"] else 2) + 2 * C * H + C + H)
    flops = 4 * M * C * H
    if step:
        bytes_ += 2 * (2 * M * C + 2 * C * H + C + H)
        flops *= 3
    return {"bytes": bytes_, "flops": flops}
