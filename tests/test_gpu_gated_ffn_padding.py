"""Rows that hold an infinity or a NaN where a hidden row is longer than F
(F % 8 != 0): the columns past F stay zero, and what the formula makes
infinite is not NaN.  All operands are positive, so that the sums with one
infinite term are +infinity."""

from __future__ import annotations

import math

import pytest
import torch

from FlagOS_mhc import sublayer as S
from test_gpu_sublayer import DEV, DT, _gen

pytestmark = pytest.mark.gpu

CASES = [
    (5, 16, 12, 16, "f32"),             # direct loads, four columns past F
    (70, 40, 36, 24, "f32"),
    (600, 1024, 1028, 1024, "f32"),
    (300, 1003, 2677, 1001, "f16"),     # padded copies
    (2051, 1003, 2821, 1003, "bf16"),
    (200, 1003, 2677, 1001, "bf16"),    # through registers
    (4, 1003, 2677, 1001, "f16"),       # few tokens
]


@pytest.mark.parametrize("T,D,F,O,dtype", CASES)
@pytest.mark.parametrize("kind", ["relu", "silu"])
def test_infinities(T, D, F, O, dtype, kind):
    print(f"[gated_ffn padding] T={T} D={D} F={F} O={O} {dtype} {kind}", flush=True)
    g = _gen(T + F)
    u = lambda *s, scale=1.0: ((0.5 + torch.rand(*s, device=DEV, generator=g)) * scale).to(DT[dtype])
    x, wg, wu, wd, go = u(T, D), u(F, D, scale=1 / D), u(F, D, scale=1 / D), u(O, F, scale=1 / F), u(T, O)
    f = S.gated_ffn(x, wg, wu, wd, kind, need_backward=True)
    back = lambda gr: S.gated_ffn_backward(gr, x, wg, wu, wd, f["gate"], f["up"], f["hidden"], kind)
    grads = back(go)
    assert all(bool(t.isfinite().all()) for t in (f["out"], *grads))
    x2, go2 = x.clone(), go.clone()
    x2[1, 0], x2[3, D - 1], go2[2, 0] = math.inf, math.nan, math.inf
    f2 = S.gated_ffn(x2, wg, wu, wd, kind, need_backward=True)
    assert not f2["hidden"][:, F:].any()
    for out in (f2["out"], S.gated_ffn(x2, wg, wu, wd, kind)["out"]):
        assert bool((out[1] == math.inf).all()) and bool(out[3].isnan().all())
        rest = [t for t in range(T) if t not in (1, 3)]
        assert torch.equal(out[rest], f["out"][rest])
    gx, gwg, gwu, gwd = back(go2)
    assert bool((gx[2] == math.inf).all()) and bool((gwg == math.inf).all()) and bool((gwu == math.inf).all())
    assert bool((gwd[0] == math.inf).all()) and torch.equal(gwd[1:], grads[3][1:])
    rest = [t for t in range(T) if t != 2]
    assert torch.equal(gx[rest], grads[0][rest])
