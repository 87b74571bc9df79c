"""The activations and their derivatives far from zero, one by one: x holds one
1 a token, so gates are single weights, exactly; w_up and grad_out are 1 and
w_down is the identity, so hidden, out, and the gradients of the weights are
the activation's values and slopes with no sum on the way."""

from __future__ import annotations

import math

import pytest
import torch

import sublayer_ref as R
from FlagOS_mhc import sublayer as S
from test_gpu_sublayer import DEV, DT

pytestmark = pytest.mark.gpu


def _act(kind, g):
    """act(g) and act'(g), in 64 bits without 1 + tanh (which would be left with
    2^-53 of the gate, more than the tail's own size)."""
    if kind != "gelu_tanh":
        return R.act(kind, g)
    k = math.sqrt(2 / math.pi)
    z = 2 * k * (g + 0.044715 * g ** 3)
    s = torch.sigmoid(z)
    return g * s, s + g * s * torch.sigmoid(-z) * 2 * k * (1 + 3 * 0.044715 * g * g)


def _errors(kind, g):
    """What act(g) and act'(g) in fp32 may be off by, before rounding to the type.

    Sigmoid s of z (silu: g; gelu_tanh: 2 v, v a cubic of four roundings): its
    exponent is off by |z| 2^-24 (2 v: by |z| 2^-21 with the cubic's), at most
    90 of them before s is 0; 2^-17 and 2^-14 of s in all.  Above z = 0 what
    counts is 1 - s, off by 2^-22 at most, times what the slope has beside it.  gelu:
    1 + erf cancels: 2^-22 of the gate (slope: of 1); exp(-g^2 / 2), by its
    argument's rounding, 88 2^-23 < 2^-16.  Below 2^-126 nothing is held: 100
    times that."""
    floor = 100 * 2.0 ** -126
    a, d = (t.abs() for t in _act(kind, g))
    s = lambda z: torch.sigmoid(z)
    if kind == "silu":
        return 2.0 ** -16 * a + floor, 2.0 ** -16 * d + (g.abs() + 4) * 2.0 ** -21 * s(g) + floor
    if kind == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        z = 2 * k * (g + 0.044715 * g ** 3)
        slope = 2 * k * g.abs() * (1 + 3 * 0.044715 * g * g)
        return 2.0 ** -14 * a + floor, 2.0 ** -14 * (s(z) + slope * s(z) * s(-z)) + 2.0 ** -21 * slope * s(z) + 100 * floor
    if kind == "gelu":
        return 2.0 ** -22 * g.abs() + 2.0 ** -20 * a, 2.0 ** -22 + 2.0 ** -16 * (d + g.abs() * torch.exp(-g * g / 2)) + floor
    return torch.zeros_like(g), torch.zeros_like(g)


# few tokens, tiles of 64 rows, tiles for more
@pytest.mark.parametrize("T", [4, 64, 300])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh", "relu"])
def test_far_out(kind, dtype, T):
    dt, D, F = DT[dtype], 320, 512
    span = torch.linspace(-100, 100, T * F, device=DEV).reshape(F, T)
    span[0, 0], span[1, 0], span[2, 0], span[3, 0] = 0.0, -87.5, -88.5, -89.5  # subnormal and vanishing sigmoids
    wg = torch.zeros(F, D, device=DEV)
    wg[:, :T] = span
    wg = wg.to(dt)
    x, wu = torch.eye(T, D, device=DEV, dtype=dt), torch.ones(F, D, device=DEV, dtype=dt)
    wd, go = torch.eye(F, device=DEV, dtype=dt), torch.ones(T, F, device=DEV, dtype=dt)
    f = S.gated_ffn(x, wg, wu, wd, kind, need_backward=True)
    _, gwg, gwu, _ = S.gated_ffn_backward(go, x, wg, wu, wd, f["gate"], f["up"], f["hidden"], kind)
    g = wg[:, :T].t().double()
    assert torch.equal(f["gate"].double(), g) and bool((f["up"] == 1).all())
    a, d = _act(kind, g)
    ea, ed = _errors(kind, g)
    h, tiny = R.half_step(dt), torch.finfo(dt).tiny
    bound = lambda v, e: 1.01 * (e + h * v.abs().clamp(min=tiny))
    for name, got, want, e in (("hidden", f["hidden"], a, ea), ("out", f["out"], a, ea), ("grad_w_up", gwu[:, :T].t(), a, ea),
                               ("grad_w_gate", gwg[:, :T].t(), d, ed)):
        over = (got.double() - want).abs() - bound(want, e)
        i = int(over.argmax())
        assert float(over.max()) <= 0, f"{name}: {float(over.max()):.3e} beyond at gate {float(g.flatten()[i])}"
    assert not gwg[:, T:].any() and not gwu[:, T:].any()
