"""Plain forms of weights held in 4 bits, in 64 bits and on any device, and the bounds that results are held to."""
from __future__ import annotations

import torch


def plain_values(w: torch.Tensor, group: int) -> torch.Tensor:
    """What ``w`` [.., K] keeps: per ``group`` elements s = max |w| / 7 rounded to five significant bits (ties to even; 0 below
    7 * 2^-126), each element q s with q = w / s rounded (ties to even)."""
    K = w.shape[-1]
    v = torch.nn.functional.pad(w.double(), (0, -K % group)).reshape(*w.shape[:-1], -1, group)
    top = v.abs().amax(dim=-1, keepdim=True)
    m, e = torch.frexp(top / 7)
    s = torch.ldexp((m * 32).round(), e - 5)
    s = torch.where(top < 7 * 2.0 ** -126, 0.0, s)
    q = torch.where(s > 0, (v / torch.where(s > 0, s, 1.0)).round(), 0.0)
    return (q * s).reshape(*w.shape[:-1], -1)[..., :K]


def values_by_place(w4) -> torch.Tensor:
    """[G, N, K] float64: every element of a ``Weight4`` fetched by its own place."""
    codes, scales = w4.codes.reshape(-1).cpu(), w4.scales.double().reshape(-1).cpu()
    G, N, K, group = w4.G, w4.N, w4.K, w4.group
    half = N // 2 if w4.pair else N
    strips, blocks, groups = (2 if w4.pair else 1) * -(-half // 16), -(-K // 64), -(-K // group)
    g, n, k = torch.arange(G).view(-1, 1, 1), torch.arange(N).view(1, -1, 1), torch.arange(K).view(1, 1, -1)
    strip, r = n % half // 16 + n // half * (strips // 2 if w4.pair else 0), n % half % 16
    at = g * strips + strip
    c = k % 64
    byte = (at * blocks + k // 64) * 512 + (r % 8) * 64 + c % 16 // 4 * 16 + c // 16 * 4 + c % 2 * 2 + c % 4 // 2
    q = (codes[byte].int() >> (r // 8 * 4).int() & 15).double() - 8
    return q * scales[((at * groups + k // group) * 8 + r % 8) * 2 + r // 8]


ACTS = {
    "silu": lambda g, p: g * torch.sigmoid(g),
    "gelu_tanh": lambda g, p: torch.nn.functional.gelu(g, approximate="tanh"),
}


def gated(act: str, g: torch.Tensor, u: torch.Tensor, param: float = 0.0) -> torch.Tensor:
    if act == "clamped_sigmoid":
        g, u = g.clamp(max=param), u.clamp(-param, param)
        return g * torch.sigmoid(1.702 * g) * (u + 1)
    return ACTS[act](g, param) * u


def plain_act(act: str, y: torch.Tensor) -> torch.Tensor:
    if act == "relu2":
        return y.clamp(min=0).square()
    if act == "gelu":
        return torch.nn.functional.gelu(y)
    return y


def sum_bound(x: torch.Tensor, W: torch.Tensor) -> torch.Tensor:
    """How far a product's 32-bit sums may be off.  The products x q s are exact in 32 bits.  They are added 16 at a time in the tensor core,
    one addition onto the last sum (rounded or cut: at most 2^-23 of it) and the 16 among themselves (likewise, with room for four), then pieces of K by
    at most a few dozen additions: (K / 16 + 80) 2^-23 of the sum of magnitudes bounds it all."""
    return (x.shape[-1] / 16 + 80) * 2.0 ** -23 * (x.abs() @ W.abs().transpose(-1, -2))


def out_step(y: torch.Tensor, dtype) -> torch.Tensor:
    """Half a step of the output's type."""
    return y.abs() * (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24) + 1e-37


def check_product(got: torch.Tensor, x: torch.Tensor, W: torch.Tensor, *, bias=None, swiglu=False, act="silu", param=0.0):
    """``got`` against x W^T (and what follows it) in 64 bits."""
    x, W = x.double(), W.double()
    if not swiglu:
        y, off = x @ W.t(), sum_bound(x, W)
        if bias is not None:
            y = y + bias.double()
            off = off + 2.0 ** -23 * (y.abs() + bias.double().abs())
        z = plain_act(act, y)
        # |relu(x)^2|' <= 2 |x|, |gelu'| <= 1.13; both computed to a few 2^-24 of their terms
        slope = 2 * (y.abs() + off) if act == "relu2" else 1.13
        off = slope * off + 2.0 ** -21 * z.abs() + (2.0 ** -22 * y.abs() if act == "gelu" else 0)
    else:
        half = W.shape[0] // 2
        g, u = x @ W[:half].t(), x @ W[half:].t()
        dg, du = sum_bound(x, W[:half]), sum_bound(x, W[half:])
        z = gated(act, g, u, param)
        # |silu'| <= 1.1, |gelu'| <= 1.13, |(g sigmoid(1.702 g))'| <= 1.13; the function to 2^-19 of itself (a quick exponential and quotient, or tanh)
        h = gated(act, g, torch.ones_like(u) if act != "clamped_sigmoid" else torch.zeros_like(u), param).abs()
        top = u.abs() + du if act != "clamped_sigmoid" else torch.full_like(u, param + 1)
        off = 1.13 * dg * top + (h + 1.13 * dg) * du + 2.0 ** -19 * (z.abs() + h) + 2.0 ** -19 * g.abs() * top * (act == "gelu_tanh")
    off = off + out_step(z, got.dtype) * 1.01
    far = (got.double() - z).abs()
    assert bool((far <= off).all()), f"off by {float((far / off).max()):.2f} of what rounding allows at {int((far / off).argmax())}"
