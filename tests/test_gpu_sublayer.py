"""Layer norm, gated feed-forward block and dropout on the GPU against 64-bit
formulas (bounds: tests/sublayer_ref.py)."""

from __future__ import annotations

import math

import pytest
import torch

import sublayer_ref as R
from FlagOS_mhc import sublayer as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


# ---- layer norm ----------------------------------------------------------------

# one vector, waves, blocks of 256 and 1024, the loop; widths that end inside a vector
NORM_SHAPES = [(1, 1), (3, 7), (5, 8), (1, 7168), (37, 64), (130, 255), (9, 513), (65, 1003), (33, 2049), (17, 4095),
               (1030, 256), (300, 7168), (5, 8200), (3, 16385), (2, 33001)]


def _check_norm(x, w, b, gy, eps=1e-5):
    D, dt = x.shape[-1], x.dtype
    h = R.half_step(dt)
    f = S.layer_norm(x, w, b, eps, need_backward=True)
    torch.cuda.synchronize()
    y, mean, rstd = R.norm_fwd(x, w, b, eps)
    # sums over a row: 32 values a lane at most, the wave's and the waves' levels (the loop: D / 1024)
    depth = 64 + D // 1024
    xm = x.double().abs().amax(-1, keepdim=True)
    wm = 1.0 if w is None else float(w.double().abs().max())
    bm = 0.0 if b is None else float(b.double().abs().max())
    bound = h * y.abs() + depth * R.ULP32 * (4 * xm * rstd * wm + bm)
    assert f["y"].shape == x.shape and f["y"].dtype == dt
    assert bool(((f["y"].double() - y).abs() <= bound).all()), float(((f["y"].double() - y).abs() - bound).max())
    assert bool(((f["mean"].double() - mean.reshape(-1)).abs() <= depth * R.ULP32 * xm.reshape(-1)).all())
    assert bool(((f["rstd"].double() / rstd.reshape(-1) - 1).abs() <= depth * R.ULP32 * (2 + xm * rstd).reshape(-1)).all())
    gx, gw, gb = S.layer_norm_backward(gy, x, w, f["mean"], f["rstd"])
    torch.cuda.synchronize()
    wx, ww, wb, aw, ab = R.norm_bwd(gy, x, w, eps)
    gm = gy.double().abs().amax(-1, keepdim=True) * wm
    hm = (2 * xm * rstd).clamp(min=1.0, max=math.sqrt(D))
    bound = h * wx.abs() + depth * R.ULP32 * 4 * rstd * gm * (1 + hm * hm + xm * rstd)
    assert gx.shape == x.shape and gx.dtype == dt
    assert bool(((gx.double() - wx).abs() <= bound).all()), float(((gx.double() - wx).abs() - bound).max())
    T = x.numel() // D
    chain = depth + T / 256 + 128 + 16
    hd = depth * R.ULP32 * 4 * ((xm * rstd) * gy.double().abs()).reshape(-1, D).sum(0)  # xhat's own error
    assert bool(((gw.double() - ww).abs() <= chain * R.ULP32 * aw + hd).all())
    assert bool(((gb.double() - wb).abs() <= chain * R.ULP32 * ab).all())
    return f, gx, gw, gb


@pytest.mark.parametrize("T,D", NORM_SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_layer_norm(T, D, dtype):
    print(f"[layer_norm] T={T} D={D} {dtype}", flush=True)
    g, dt = _gen(T * 31 + D), DT[dtype]
    x = (_randn(g, T, D) * 2 + 0.5).to(dt)
    w, b = _randn(g, D) * 0.2 + 1, _randn(g, D)
    gy = _randn(g, T, D, dtype=dt)
    _check_norm(x, w, b, gy)
    _check_norm(x, w.to(dt), b.to(dt), gy)
    _check_norm(x, None, None, gy)


def test_layer_norm_far_mean_and_constant_rows():
    g = _gen(5)
    x = _randn(g, 40, 1000) + 300.0
    x[3] = 7.0  # no variance: rstd is eps^-1/2
    x[5] = 0.0
    _check_norm(x, _randn(g, 1000), _randn(g, 1000), _randn(g, 40, 1000))


def test_layer_norm_nan_stays_in_its_row():
    g = _gen(6)
    x = _randn(g, 6, 300, dtype=torch.bfloat16)
    x[2, 5] = float("nan")
    x[4, 7] = float("inf")
    y = S.layer_norm(x)["y"]
    bad = y.isnan().any(-1).tolist()
    assert bad == [False, False, True, False, True, False]


def test_layer_norm_views_streams_and_empty():
    g = _gen(7)
    base = _randn(g, 20, 3, 130, dtype=torch.bfloat16)
    for x in (base[:, 1, :], base.transpose(0, 1), base.reshape(-1)[1:1 + 19 * 130].view(19, 130)):
        _check_norm(x, None, None, torch.ones_like(x))
    side = torch.cuda.Stream()
    x = _randn(g, 64, 512)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        y = S.layer_norm(x)["y"]
    side.synchronize()
    assert torch.equal(y, S.layer_norm(x)["y"])
    e = S.layer_norm(x[:0], need_backward=True)
    gx, gw, gb = S.layer_norm_backward(x[:0], x[:0], None, e["mean"], e["rstd"])
    assert e["y"].shape == (0, 512) and gx.shape == (0, 512) and not gw.any() and not gb.any()


def test_layer_norm_repeats_bit_for_bit():
    g = _gen(8)
    x, gy, w = _randn(g, 3001, 640, dtype=torch.bfloat16), _randn(g, 3001, 640, dtype=torch.bfloat16), _randn(g, 640)
    runs = [_check_norm(x, w, w, gy) for _ in range(3)]
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r[1:], runs[0][1:]))


def test_layer_norm_autograd():
    g = _gen(9)
    x = _randn(g, 2, 9, 96, dtype=torch.bfloat16).requires_grad_(True)
    w, b = _randn(g, 96, dtype=torch.bfloat16).requires_grad_(True), _randn(g, 96).requires_grad_(True)
    gy = _randn(g, 2, 9, 96, dtype=torch.bfloat16)
    S.layer_norm_fn(x, w, b).backward(gy)
    f = S.layer_norm(x.detach(), w.detach(), b.detach(), need_backward=True)
    gx, gw, gb = S.layer_norm_backward(gy, x.detach(), w.detach(), f["mean"], f["rstd"])
    assert torch.equal(x.grad, gx) and torch.equal(w.grad, gw.to(w.dtype)) and torch.equal(b.grad, gb)


def test_layer_norm_refusals():
    x = torch.zeros(4, 8, device=DEV)
    with pytest.raises(ValueError, match="weight"):
        S.layer_norm(x, torch.zeros(7, device=DEV))
    with pytest.raises(NotImplementedError, match="dtype"):
        S.layer_norm(x.double())
    with pytest.raises(ValueError, match="grad_y"):
        S.layer_norm_backward(x[:2], x, None, x[:, 0], x[:, 0])
    with pytest.raises(ValueError, match="means"):
        S.layer_norm_backward(x, x, None, x[:2, 0], x[:, 0])


# ---- gated feed-forward block ------------------------------------------------------

FFN_SHAPES = [(1, 1, 1, 1), (2, 3, 5, 7), (1, 64, 128, 64), (7, 200, 264, 200), (16, 256, 512, 128), (17, 136, 72, 40),
              (64, 1024, 2048, 1024), (65, 255, 513, 255), (130, 128, 320, 256), (300, 500, 1000, 500),
              (513, 264, 520, 1032), (1000, 1003, 2677, 1003)]


def _ffn_inputs(T, D, F, O, dt, seed=0):
    g = _gen(seed + T + D)
    return (_randn(g, T, D, dtype=dt), _randn(g, F, D, dtype=dt, scale=D ** -0.5),
            _randn(g, F, D, dtype=dt, scale=D ** -0.5), _randn(g, O, F, dtype=dt, scale=F ** -0.5),
            _randn(g, T, O, dtype=dt))


def _check_ffn(x, wg, wu, wd, go, kind, what=""):
    dt, F = x.dtype, wg.shape[0]
    T, D, O = x.numel() // x.shape[-1], x.shape[-1], wd.shape[0]
    f = S.gated_ffn(x, wg, wu, wd, kind, need_backward=True)
    out = S.gated_ffn(x, wg, wu, wd, kind)["out"]
    grads = S.gated_ffn_backward(go, x, wg, wu, wd, f["gate"], f["up"], f["hidden"], kind)
    torch.cuda.synchronize()
    want, g, u, h = R.ffn_fwd(x.reshape(T, D), wg, wu, wd, kind)
    R.close2(out.reshape(T, O), want, dt, 2, D + F, what + " out")
    R.close2(f["out"].reshape(T, O), want, dt, 2, D + F, what + " out (saved)")
    R.close2(f["gate"], g, torch.float32, 1, D, what + " gate")
    R.close2(f["up"], u, torch.float32, 1, D, what + " up")
    R.close2(f["hidden"][:, :F], h, dt, 1, D, what + " hidden")
    assert not f["hidden"][:, F:].any()
    wants = R.ffn_bwd(go.reshape(T, O), x.reshape(T, D), wg, wu, wd, kind)
    for name, got, w, terms in zip(("x", "w_gate", "w_up", "w_down"), grads, wants,
                                   (D + O + 2 * F, D + O + T, D + O + T, D + T)):
        R.close2(got.reshape(w.shape), w, dt, 2, terms, f"{what} grad_{name}")
    return out, f, grads


@pytest.mark.parametrize("T,D,F,O", FFN_SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_gated_ffn(T, D, F, O, dtype):
    print(f"[gated_ffn] T={T} D={D} F={F} O={O} {dtype}", flush=True)
    kind = ("silu", "gelu", "gelu_tanh", "relu")[(T + D) % 4]
    _check_ffn(*_ffn_inputs(T, D, F, O, DT[dtype]), kind, f"{kind} {dtype}")


@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh", "relu"])
def test_gated_ffn_activations_far_out(kind):
    """Gates far from zero: the activations' tails and their derivatives."""
    x, wg, wu, wd, go = _ffn_inputs(40, 64, 96, 64, torch.float32, 3)
    _check_ffn(x, wg * 20, wu, wd, go, kind, kind)


def test_gated_ffn_views_leading_dims_and_empty():
    g = _gen(4)
    dt = torch.bfloat16
    big = _randn(g, 2 * 70, 72, dtype=dt, scale=0.1)  # one tensor for gate and up
    wd = _randn(g, 48, 70, dtype=dt, scale=0.1)
    base = _randn(g, 3, 5, 145, dtype=dt)
    x, go = base[..., 1:73], _randn(g, 48, 5, 3, dtype=dt).permute(2, 1, 0)
    out, f, grads = _check_ffn(x, big[:70], big[70:], wd, go, "silu")
    assert out.shape == (3, 5, 48) and grads[0].shape == x.shape
    unaligned = big.reshape(-1)[3:3 + 70 * 72].view(70, 72)
    _check_ffn(x, unaligned, big[70:], wd, go, "silu")
    e = S.gated_ffn(x[:0], big[:70], big[70:], wd, need_backward=True)
    grads = S.gated_ffn_backward(go[:0], x[:0], big[:70], big[70:], wd, e["gate"], e["up"], e["hidden"])
    assert e["out"].shape == (0, 5, 48) and grads[0].shape == (0, 5, 72)
    assert not any(t.any() for t in grads[1:])


def test_gated_ffn_nan_stays_in_its_token():
    """A token that holds a NaN or an infinity leaves every other token as it is."""
    for T in (5, 40, 300):
        for dt in DT.values():
            x, wg, wu, wd, _ = _ffn_inputs(T, 72, 136, 72, dt)
            want = S.gated_ffn(x, wg, wu, wd)["out"]
            x[1, 3], x[T - 1, 71] = float("nan"), float("inf")
            got = S.gated_ffn(x, wg, wu, wd)["out"]
            assert torch.equal(got[2:T - 1], want[2:T - 1]) and torch.equal(got[0], want[0])
            assert bool(got[1].isnan().all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gated_ffn_repeats_bit_for_bit_and_streams(dtype):
    a = _ffn_inputs(333, 264, 520, 264, DT[dtype], 5)
    runs = []
    for i in range(3):
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            f = S.gated_ffn(*a[:4], need_backward=True)
            grads = S.gated_ffn_backward(a[4], *a[:4], f["gate"], f["up"], f["hidden"])
        s.synchronize()
        runs.append((f["out"], *grads))
    for r in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(r, runs[0]))


def test_gated_ffn_autograd():
    x, wg, wu, wd, go = _ffn_inputs(50, 64, 120, 64, torch.bfloat16, 6)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    S.gated_ffn_fn(*leaves, "gelu").backward(go)
    f = S.gated_ffn(x, wg, wu, wd, "gelu", need_backward=True)
    want = S.gated_ffn_backward(go, x, wg, wu, wd, f["gate"], f["up"], f["hidden"], "gelu")
    assert all(torch.equal(a.grad, b) for a, b in zip(leaves, want))
    with torch.no_grad():
        assert torch.equal(S.gated_ffn_fn(*leaves, "gelu"), S.gated_ffn(x, wg, wu, wd, "gelu")["out"])


def test_gated_ffn_refusals():
    x, wg, wu, wd, go = _ffn_inputs(4, 16, 24, 16, torch.bfloat16)
    with pytest.raises(ValueError, match="activation"):
        S.gated_ffn(x, wg, wu, wd, "swish")
    with pytest.raises(ValueError, match="do not fit"):
        S.gated_ffn(x, wg, wu[:8], wd)
    with pytest.raises(ValueError, match="w_up is"):
        S.gated_ffn(x, wg, wu.float(), wd)
    f = S.gated_ffn(x, wg, wu, wd, need_backward=True)
    with pytest.raises(ValueError, match="grad_out"):
        S.gated_ffn_backward(go[:2], x, wg, wu, wd, f["gate"], f["up"], f["hidden"])
    with pytest.raises(ValueError, match="hidden"):
        S.gated_ffn_backward(go, x, wg, wu, wd, f["gate"], f["up"], f["hidden"][:, :8])


# ---- dropout ---------------------------------------------------------------------

@pytest.mark.parametrize("n", [1, 7, 8, 9, 2047, 4096, 100003])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_dropout(n, dtype):
    g, dt = _gen(n), DT[dtype]
    x = _randn(g, n, dtype=dt)
    h = R.half_step(dt)
    for p, seed, off in ((0.1, 1, 0), (0.5, (1 << 63) + 77, (1 << 35) + 1), (0.0, 3, 3), (1.0, 3, 3)):
        y = S.dropout(x, p, seed, off)
        want = S.dropout_ref(torch.ones_like(x), p, seed, off).double()
        t = int(p * 65536 + 0.5)
        exact = torch.where(want != 0, x.double() * (65536.0 / max(1, 65536 - t)), 0.0)
        # the factor's and the product's fp32 roundings, then the type's: half a step, which below the
        # smallest normal number is that number's
        bound = h * exact.abs().clamp(min=torch.finfo(dt).tiny) + 2 * R.ULP32 * exact.abs()
        assert bool(((y.double() - exact).abs() <= bound * (exact != 0)).all())
        assert torch.equal(S.dropout_backward(x, p, seed, off), y)
    y = S.dropout(x, 1.0)
    assert not y.any()


def test_dropout_drops_infinities_and_repeats_over_views():
    x = torch.full((64, 96), float("inf"), device=DEV)
    y = S.dropout(x, 0.5, 11, 2)
    assert bool((y.isinf() | (y == 0)).all()) and 0 < int((y == 0).sum()) < y.numel()
    g = _gen(1)
    z = _randn(g, 96, 64).t()
    assert torch.equal(S.dropout(z, 0.5, 11, 2), S.dropout(z.contiguous(), 0.5, 11, 2))
    u = _randn(g, 1025)[1:]
    assert torch.equal(S.dropout(u, 0.5, 11, 2), S.dropout(u.clone(), 0.5, 11, 2))
    assert S.dropout(u[:0], 0.5).shape == (0,)


def test_dropout_share_and_offsets():
    """The share of kept elements is within six standard deviations of 1 - p, and
    two offsets, seeds or halves of a tensor do not share their masks."""
    n = 1 << 20
    x = torch.ones(n, device=DEV)
    for p in (0.02, 0.5, 0.9):
        kept = float((S.dropout(x, p, 5, 6) != 0).double().mean())
        assert abs(kept - (1 - p)) <= 6 * math.sqrt(p * (1 - p) / n) + 2.0 ** -17
    a, b, c = (S.dropout(x, 0.5, s, o) != 0 for s, o in ((5, 6), (5, 7), (6, 6)))
    for u, v in ((a, b), (a, c), (a[: n // 2], a[n // 2:])):
        assert abs(float((u == v).double().mean()) - 0.5) <= 6 * 0.5 / math.sqrt(u.numel())


def test_dropout_state_and_autograd():
    g = _gen(2)
    x = _randn(g, 33, 65).requires_grad_(True)
    state = torch.tensor([5, 1 << 40], device=DEV)
    y = S.dropout_fn(x, 0.3, state=state)
    state[1] += 1  # the program moves on before the backward
    gy = _randn(g, 33, 65)
    y.backward(gy)
    assert torch.equal(y, S.dropout(x, 0.3, 5, 1 << 40))
    assert torch.equal(x.grad, S.dropout(gy, 0.3, 5, 1 << 40))
    with pytest.raises(ValueError, match="state"):
        S.dropout(x, 0.3, state=state.int())
    with pytest.raises(ValueError, match="probability"):
        S.dropout(x, 1.5)
