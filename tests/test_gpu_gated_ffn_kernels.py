"""The gated feed-forward block at sizes that reach each of its kernels: large
tiles (whole, cut into runs of k, with a tail of few rows), padded copies of
odd rows, products through registers, few tokens.  Against 64-bit formulas;
bounds: tests/sublayer_ref.py."""

from __future__ import annotations

import pytest
import torch

import sublayer_ref as R
from FlagOS_mhc import sublayer as S
from test_gpu_sublayer import DT, _check_ffn, _ffn_inputs

pytestmark = pytest.mark.gpu

# what tests/test_gemm_plan.py counts over many shapes, here by example (256 CUs)
SHAPES = [
    (2051, 1024, 2816, 1024, "bf16"),  # 256 x 256 and 128 x 256 tiles, runs of k
    (2304, 520, 4104, 520, "bf16"),    # 256 x 256 with the gated gradient; 128 x 128 in runs
    (4099, 512, 1536, 2048, "f16"),    # 3 rows past whole tiles
    (2048, 512, 4096, 512, "f32"),     # large fp32 tiles
    (300, 1003, 2677, 1001, "f16"),    # every operand's rows are copied
    (1100, 501, 1003, 503, "f32"),
    (600, 1003, 1024, 1000, "bf16"),   # x's, w_gate's and w_up's are
    (513, 1024, 1003, 264, "bf16"),    # w_down's is
    (200, 1003, 2677, 1001, "bf16"),   # through registers
    (64, 333, 1001, 335, "f32"),
    (16, 333, 1001, 335, "f16"),
    (4, 1100, 515, 37, "bf16"),        # few tokens: KB runs with a cut end
    (3, 4100, 1030, 258, "f32"),
    (40, 2048, 5632, 2048, "bf16"),
]


@pytest.mark.parametrize("T,D,F,O,dtype", SHAPES)
def test_kernels(T, D, F, O, dtype):
    print(f"[gated_ffn kernels] T={T} D={D} F={F} O={O} {dtype}", flush=True)
    kind = ("silu", "gelu", "gelu_tanh", "relu")[(T + D) % 4]
    _check_ffn(*_ffn_inputs(T, D, F, O, DT[dtype]), kind, f"{kind} {dtype}")


@pytest.mark.parametrize("T,D,F,O,dtype", [(2, 513, 4099, 1, "f16"), (5, 72, 4096, 3000, "bf16"), (9, 40, 264, 56, "f32")])
def test_few_tokens_or_outputs_element_by_element(T, D, F, O, dtype):
    """Sums of few terms, or few sums that may be small by chance beside their
    terms: a norm of the results says nothing of a single one, so every rounding
    is counted where it occurs, in full.  gate, up and the gradient of hidden:
    fp32 sums; hidden and the gradients of gate and up: one rounding to the type
    (H); every result: one more.  The activations' first and second derivatives
    are below 1.2; their own fp32 arithmetic is 2^-17 at worst for 16-bit
    results, which H covers eight times over, and 32 ulps for fp32.  Half a step
    below a type's smallest normal number is that number's."""
    dt = DT[dtype]
    x, wg, wu, wd, go = _ffn_inputs(T, D, F, O, dt)
    f = S.gated_ffn(x, wg, wu, wd, "gelu", need_backward=True)
    grads = S.gated_ffn_backward(go, x, wg, wu, wd, f["gate"], f["up"], f["hidden"], "gelu")
    H, U = R.half_step(dt), R.ULP32
    _, g, u, h = R.ffn_fwd(x, wg, wu, wd, "gelu")
    X, G, W, V, Y = (t.double() for t in (x, wg, wu, wd, go))
    mm = lambda a, b: a @ b.contiguous()
    ab = lambda a, b: mm(a.abs(), b.abs())  # sums of the terms' sizes
    a, d = R.act("gelu", g)
    dh = mm(Y, V)
    dg, du = dh * u * d, dh * a
    eg, eu, edh = D * U * ab(X, G.t()), D * U * ab(X, W.t()), O * U * ab(Y, V)
    tiny = torch.finfo(dt).tiny
    own = lambda v: H * v.abs().clamp(min=tiny) + 32 * U * v.abs()
    eh = own(h) + eu * a.abs() + 1.2 * u.abs() * eg
    edg = own(dg) + 1.2 * edh * u.abs() + dh.abs() * (1.2 * eu + 1.2 * u.abs() * eg)
    edu = own(du) + edh * a.abs() + 1.2 * dh.abs() * eg

    def check(name, got, left, right, e_left):
        """got = left @ right, left off by e_left."""
        want = mm(left, right)
        K = left.shape[1]
        bound = (1 + H) * mm(e_left, right.abs()) + H * want.abs().clamp(min=tiny) + (K + 2) * U * ab(left, right)
        assert bool(((got.double() - want).abs() <= bound).all()), name

    check("out", f["out"], h, V.t(), eh)
    check("grad_w_down", grads[3].t(), h.t(), Y, eh.t())
    check("grad_w_gate", grads[1], dg.t(), X, edg.t())
    check("grad_w_up", grads[2], du.t(), X, edu.t())
    check("grad_x", grads[0], torch.cat((dg, du), 1), torch.cat((G, W), 0), torch.cat((edg, edu), 1))


@pytest.mark.parametrize("T,D,F,O", [(2051, 1024, 2816, 1024), (300, 1003, 2677, 1001), (1, 520, 1032, 520)])
def test_other_streams_and_repeats_bit_for_bit(T, D, F, O):
    """Runs, joins and copies have a fixed order, and take their workspaces from
    the stream that the call is on."""
    a = _ffn_inputs(T, D, F, O, torch.bfloat16, 7)
    runs = []
    for _ in range(3):
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            f = S.gated_ffn(*a[:4], need_backward=True)
            grads = S.gated_ffn_backward(a[4], *a[:4], f["gate"], f["up"], f["hidden"])
        s.synchronize()
        runs.append((f["out"], f["gate"], f["up"], f["hidden"], *grads))
    for r in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(r, runs[0]))


def test_without_the_weights_gradients():
    x, wg, wu, wd, go = _ffn_inputs(70, 136, 264, 72, torch.bfloat16, 8)
    f = S.gated_ffn(x, wg, wu, wd, need_backward=True)
    want = S.gated_ffn_backward(go, x, wg, wu, wd, f["gate"], f["up"], f["hidden"])
    got = S.gated_ffn_backward(go, x, wg, wu, wd, f["gate"], f["up"], f["hidden"], need_weights=False)
    assert torch.equal(got[0], want[0]) and got[1:] == (None, None, None)
    xr = x.clone().requires_grad_(True)
    S.gated_ffn_fn(xr, wg, wu, wd).backward(go)  # frozen weights
    assert torch.equal(xr.grad, want[0])


@pytest.mark.parametrize("T,dtype", [(2051, "bf16"), (300, "f16"), (2048, "f32")])
def test_nan_and_infinity_stay_in_their_token(T, dtype):
    """.. in the large tiles and the padded copies too: forward, and the gradient
    with respect to x."""
    D, F, O = (1024, 2816, 1024) if T > 300 else (1003, 2677, 1001)
    x, wg, wu, wd, go = _ffn_inputs(T, D, F, O, DT[dtype], 9)
    f = S.gated_ffn(x, wg, wu, wd, need_backward=True)
    gx = S.gated_ffn_backward(go, x, wg, wu, wd, f["gate"], f["up"], f["hidden"], need_weights=False)[0]
    x2, go2 = x.clone(), go.clone()
    x2[1, D - 1], x2[T - 1, 0], go2[7, O - 1] = float("nan"), float("inf"), float("nan")
    f2 = S.gated_ffn(x2, wg, wu, wd, need_backward=True)
    gx2 = S.gated_ffn_backward(go2, x2, wg, wu, wd, f2["gate"], f2["up"], f2["hidden"], need_weights=False)[0]
    keep = torch.ones(T, dtype=torch.bool, device=x.device)
    keep[1] = keep[T - 1] = False
    assert torch.equal(f2["out"][keep], f["out"][keep]) and bool(f2["out"][1].isnan().all())
    keep[7] = False
    assert torch.equal(gx2[keep], gx[keep]) and bool(gx2[7].isnan().all())


def test_gradient_against_differences():
    """fp32: the gradient of a scalar against the 64-bit formula's differences."""
    x, wg, wu, wd, go = _ffn_inputs(260, 130, 260, 130, torch.float32, 10)
    f = S.gated_ffn(x, wg, wu, wd, "gelu", need_backward=True)
    grads = S.gated_ffn_backward(go, x, wg, wu, wd, f["gate"], f["up"], f["hidden"], "gelu")
    t = [x, wg, wu, wd]
    g = torch.Generator(device=x.device)
    g.manual_seed(11)
    for i, gr in enumerate(grads):
        v = torch.randn(t[i].shape, device=x.device, generator=g).double()
        at = lambda s: float((R.ffn_fwd(*[a.double() + s * v if j == i else a for j, a in enumerate(t)], "gelu")[0]
                              * go.double()).sum())
        num = (at(1e-6) - at(-1e-6)) / 2e-6
        # 64-bit differences are good to 1e-6 of the norms; the fp32 gradient to about sqrt(K) 2^-24 of them
        assert abs(num - float((gr.double() * v).sum())) <= (1e-6 + 64 * R.ULP32) * float(gr.double().norm() * v.norm())
