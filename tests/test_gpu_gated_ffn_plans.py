"""The gated feed-forward block with every kernel in every role: each of its
products by each tile that a plan may choose for it, whole and in runs of k,
direct to LDS and through registers, and the tails.  tests/test_gemm_plan_reach.py
keeps the list of shapes complete as the plans' costs change.

Two bounds.  Element by element, every rounding counts in full where it occurs
and is carried through the next product with the absolute values of its terms
(_bounds).  In 2-norm, roundings are spread over their range and the sums' too:
that of sublayer_ref.close2, for results that are many, of many terms."""

from __future__ import annotations

import math

import pytest
import torch

import sublayer_ref as R
from FlagOS_mhc import sublayer as S
from test_gpu_sublayer import DT, _ffn_inputs

# T, D, F, O, dtype
SHAPES = [
    (1, 1100, 515, 264, "bf16"), (2, 4100, 1030, 258, "f32"), (3, 515, 264, 1003, "f16"), (4, 72, 96, 128, "f32"),
    (2312, 576, 896, 896, "f32"), (1283, 214, 6457, 221, "bf16"), (3844, 2143, 180, 152, "f16"),
    (2049, 1216, 256, 4096, "f32"), (5, 69, 76, 93, "bf16"), (5, 85, 83, 101, "f32"), (5, 128, 448, 7232, "f16"),
    (5, 1386, 1219, 2479, "bf16"), (6, 1920, 2176, 3840, "f32"), (10, 1878, 1898, 3875, "f32"),
    (1808, 1657, 69, 2435, "f16"), (1282, 1792, 6400, 192, "f32"), (5, 104, 64, 84, "f32"),
    (17, 66, 64, 111, "bf16"), (17, 90, 84, 79, "f32"), (33, 76, 65, 444, "f32"), (34, 136, 69, 753, "f16"),
    (19, 384, 384, 128, "f32"), (5, 1728, 1984, 128, "bf16"), (18, 2048, 1728, 128, "f16"),
    (3686, 2027, 65, 184, "f32"), (67, 2816, 2029, 4910, "bf16"), (5196, 3288, 64, 3349, "f16"),
    (67, 8431, 4265, 76, "bf16"), (1801, 3520, 2304, 3840, "f16"), (73, 5851, 8686, 8068, "f32"),
    (18, 373, 527, 119, "f32"), (17, 883, 916, 121, "bf16"), (1050, 1728, 7936, 2048, "f16"),
    (257, 431, 8105, 82, "f32"), (75, 70, 4252, 5688, "bf16"), (2352, 6981, 274, 93, "f16"),
    (2068, 3968, 1984, 128, "f32"), (1854, 256, 4544, 5120, "f32"), (2561, 628, 64, 3423, "f32"),
    (521, 229, 7992, 272, "bf16"), (523, 377, 7746, 180, "f32"), (67, 2880, 4544, 6720, "f32"),
    (2050, 8064, 192, 256, "f32"), (1541, 4773, 443, 5200, "f32"), (5135, 640, 704, 6400, "f16"),
    (4599, 192, 896, 1600, "f32"), (2607, 6561, 1782, 263, "bf16"), (1483, 3584, 2944, 192, "f32"),
    (527, 704, 8000, 5888, "f16"), (4130, 8581, 1988, 2005, "bf16"), (17, 182, 72, 428, "f32"),
    (18, 192, 64, 2368, "f16"), (231, 136, 4291, 64, "f32"), (491, 160, 7948, 120, "bf16"),
    (4361, 1801, 2860, 3690, "f16"), (3076, 8576, 896, 5312, "f32"), (6153, 192, 94, 8292, "bf16"),
    (1063, 256, 704, 7232, "f16"), (1329, 1427, 3242, 75, "f32"), (3616, 8621, 227, 246, "bf16"),
    (133, 128, 8256, 6912, "f16"), (517, 1572, 7792, 415, "bf16"), (6402, 2230, 162, 7792, "f32"),
    (549, 2843, 7793, 174, "f16"), (6427, 128, 8448, 128, "f32"), (3088, 320, 2816, 6976, "f32"),
    (1043, 3579, 1610, 8163, "f32"), (2561, 85, 6167, 1590, "f32"), (5125, 4480, 1620, 120, "bf16"),
    (4024, 128, 6080, 2752, "f16"), (7870, 320, 2816, 4032, "f32"),
]


def _mm(a, b):
    return a @ b.contiguous()


def _bounds(x, wg, wu, wd, go, kind, gate):
    """name -> (the 64-bit result, what the kernels' may be off by).

    U = 2^-24 is a rounding to fp32, H one to the type (half a step; below the
    smallest normal number, that number's).  A sum of K terms in fp32, in any
    order: (K + 2) U of the terms' sizes.  The activations have slopes below
    1.13 and second derivatives below 0.8 (relu: its slope is off by 1 where the
    gate's sum may have the other sign, and is that of the saved gate there, from
    which the backward is defined: one such slope, right or wrong, is more than
    all roundings in the 2-norm); their own arithmetic is off by 32 U
    (16-bit results: 2^-16) of the value and, where 1 + erf or an exponent's
    argument cancels, 4 U of the gate.  Products of two errors: 1% on top."""
    dt = x.dtype
    H, U, tiny = R.half_step(dt), R.ULP32, torch.finfo(dt).tiny
    X, G, W, V, Y = (t.double() for t in (x, wg, wu, wd, go))
    D, F, O, T = X.shape[1], G.shape[0], V.shape[0], X.shape[0]
    ab = lambda a, b: _mm(a.abs(), b.abs())
    g, u, dh = _mm(X, G.t()), _mm(X, W.t()), _mm(Y, V)
    eg, eu, edh = (D + 2) * U * ab(X, G.t()), (D + 2) * U * ab(X, W.t()), (O + 2) * U * ab(Y, V)
    a, d = R.act(kind, g)
    if kind == "relu":
        d = torch.where(g.abs() <= eg, (gate > 0).double(), d)
    own = 2.0 ** -16 if dt.itemsize == 2 else 32 * U
    ea = own * a.abs() + 4 * U * g.abs() + 1.13 * eg
    ed = own * d.abs() + 8 * U * (1 + g.abs()) + (0.8 * eg if kind != "relu" else (g.abs() <= eg).double())
    rounded = lambda v: H * v.abs().clamp(min=tiny) + 4 * U * v.abs()
    h, dg, du = a * u, dh * u * d, dh * a
    eh = 1.01 * (rounded(h) + u.abs() * ea + a.abs() * eu)
    edg = 1.01 * (rounded(dg) + (u * d).abs() * edh + (dh * d).abs() * eu + (dh * u).abs() * ed)
    edu = 1.01 * (rounded(du) + a.abs() * edh + dh.abs() * ea)

    def product(left, right, e_left):
        want = _mm(left, right)
        return want, _mm(e_left, right.abs()) + H * want.abs().clamp(min=tiny) + (left.shape[1] + 2) * U * ab(left, right)

    res = {"gate": (g, eg), "up": (u, eu), "hidden": (h, eh), "out": product(h, V.t(), eh),
           "grad_x": product(torch.cat((dg, du), 1), torch.cat((G, W), 0), torch.cat((edg, edu), 1)),
           "grad_w_gate": product(dg.t().contiguous(), X, edg.t().contiguous()),
           "grad_w_up": product(du.t().contiguous(), X, edu.t().contiguous())}
    want, e = product(h.t().contiguous(), Y, eh.t().contiguous())
    res["grad_w_down"] = (want.t(), e.t())
    return res


OTHER = {"bf16": "f16", "f16": "bf16"}


@pytest.mark.gpu
@pytest.mark.parametrize("T,D,F,O,dtype", SHAPES + [(*s[:4], OTHER[s[4]]) for s in SHAPES if s[4] in OTHER])
def test_every_kernel_in_every_role(T, D, F, O, dtype):
    print(f"[gated_ffn plans] T={T} D={D} F={F} O={O} {dtype}", flush=True)
    kind = ("silu", "gelu", "gelu_tanh", "relu")[(T + F) % 4]
    args = _ffn_inputs(T, D, F, O, DT[dtype], 12)
    x, wg, wu, wd, go = args
    f = S.gated_ffn(x, wg, wu, wd, kind, need_backward=True)
    grads = S.gated_ffn_backward(go, x, wg, wu, wd, f["gate"], f["up"], f["hidden"], kind)
    torch.cuda.synchronize()
    assert torch.equal(S.gated_ffn(x, wg, wu, wd, kind)["out"], f["out"])
    assert not f["hidden"][:, F:].any()
    got = {"gate": f["gate"], "up": f["up"], "hidden": f["hidden"][:, :F], "out": f["out"],
           **dict(zip(("grad_x", "grad_w_gate", "grad_w_up", "grad_w_down"), grads))}
    roundings = {"gate": 1, "up": 1, "hidden": 1}
    terms = {"gate": D, "up": D, "hidden": D, "out": D + F, "grad_x": D + O + 2 * F, "grad_w_down": D + T}
    for name, (want, bound) in _bounds(*args, kind, f["gate"]).items():
        e = (got[name].double() - want).abs_()
        assert bool((e <= bound).all()), f"{name}: {float((e - bound).max()):.3e} beyond its bound"
        if min(want.shape) >= 64:
            h = R.half_step(got[name].dtype)
            tol = math.sqrt(roundings.get(name, 2)) * h / math.sqrt(3.0) + R.ULP32 * (math.sqrt(terms.get(name, D + O + T)) + 4)
            rel = float(e.norm() / want.norm())
            assert rel <= tol, f"{name}: 2-norm error {rel:.3e} > {tol:.3e}"
