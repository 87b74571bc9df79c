"""64-bit formulas of the sublayer operators and the bounds their outputs are
held to (test infrastructure).

Roundings to a type are off by at most half a step, H = eps / 2 relative to
the value; their relative errors are spread over [-H, H], so the 2-norm of
many is at most H / sqrt(3) of the result's, and n independent ones
sqrt(n) H / sqrt(3).  fp32 sums of K terms add at most sqrt(K) 2^-24 on top in
the same sense.  Where there are too few values for a norm to say much, every
rounding counts with its full H.  Single elements are held to eight times the
norm's bound."""

from __future__ import annotations

import math

import torch

ULP32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close2(got, want, dtype, roundings, terms, what):
    """got against want (64 bits) in 2-norm and element by element."""
    assert tuple(got.shape) == tuple(want.shape), (what, tuple(got.shape), tuple(want.shape))
    assert got.dtype == dtype, (what, got.dtype)
    h = half_step(dtype)
    many = want.numel() >= 1000 and terms >= 64
    tol = (math.sqrt(roundings) * h / math.sqrt(3.0) if many else roundings * h) + ULP32 * (math.sqrt(terms) + 4)
    e = (got.double().cpu() - want.cpu())
    w = want.cpu()
    norm = float(w.norm())
    rel = float(e.norm()) / max(norm, 1e-300)
    assert rel <= tol, f"{what}: 2-norm error {rel:.3e} > {tol:.3e}"
    rms = norm / math.sqrt(max(1, w.numel()))
    over = e.abs() - (8 * tol * rms + h * w.abs())
    assert float(over.max()) <= 0.0, f"{what}: an element is {float(over.max()):.3e} beyond its bound"


# ---- layer norm ----------------------------------------------------------------

def norm_fwd(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + eps)
    y = (x - mean) * rstd
    y = y if w is None else y * w.double()
    return (y if b is None else y + b.double()), mean, rstd


def norm_bwd(gy, x, w, eps):
    _, mean, rstd = norm_fwd(x, None, None, eps)
    h = (x.double() - mean) * rstd
    gy = gy.double()
    g = gy if w is None else gy * w.double()
    gx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    lead = tuple(range(x.dim() - 1))
    return gx, (gy * h).sum(lead), gy.sum(lead), (gy * h).abs().sum(lead), gy.abs().sum(lead)


# ---- feed-forward block ----------------------------------------------------------

def act(kind, z):
    if kind == "silu":
        e = torch.sigmoid(z)
        return z * e, e + z * e * (1 - e)
    if kind == "gelu":
        p = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)
    return z.clamp(min=0), (z > 0).double()


def ffn_fwd(x, wg, wu, wd, kind):
    x, wg, wu, wd = (t.double() for t in (x, wg, wu, wd))
    g, u = x @ wg.t().contiguous(), x @ wu.t().contiguous()
    h = act(kind, g)[0] * u
    return h @ wd.t().contiguous(), g, u, h


def ffn_bwd(go, x, wg, wu, wd, kind):
    _, g, u, h = ffn_fwd(x, wg, wu, wd, kind)
    go, x, wg, wu, wd = (t.double() for t in (go, x, wg, wu, wd))
    dh = go @ wd
    a, d = act(kind, g)
    dg, du = dh * u * d, dh * a
    return (dg @ wg + du @ wu, dg.t().contiguous() @ x, du.t().contiguous() @ x, go.t().contiguous() @ h)


# ---- dropout ---------------------------------------------------------------------

def philox(group, seed, offset):
    """The four words of one group, in Python integers."""
    c = [group & 0xFFFFFFFF, group >> 32, offset & 0xFFFFFFFF, offset >> 32]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k[1], p0 & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c
