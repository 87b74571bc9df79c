"""The sublayer operators without a GPU: C entry points' refusals, the Python
operators' checks, and the *_ref functions against 64-bit formulas."""

from __future__ import annotations

import ctypes

import pytest
import torch

import sublayer_ref as R
from FlagOS_mhc import _lib, sublayer as S
from FlagOS_mhc.dropout import philox_ref

P = ctypes.c_void_p(0x1000)
ODD = ctypes.c_void_p(0x1002)


def _err():
    return _lib.load().mhc_last_error()


def test_layer_norm_refusals():
    lib = _lib.load()
    f = lambda x=P, xt=1, wt=0, y=P, m=None, r=None, T=4, D=8: lib.mhc_layer_norm_fwd(
        x, xt, P, P, wt, 1e-5, y, m, r, T, D, None)
    assert f(x=None) == -1 and b"null" in _err()
    assert f(D=0) == -1 and f(T=-1) == -1
    assert f(xt=7) == -2 and b"dtype" in _err()
    assert f(xt=1, wt=2) == -2 and b"weight dtype" in _err()
    assert f(m=P) == -1 and b"together" in _err()
    assert f(T=1 << 32) == -2
    assert f(T=0) == 0
    b = lambda ws, n, T=4, D=8, gw=P: lib.mhc_layer_norm_bwd(P, P, 1, P, 0, P, P, P, gw, P, ws, n, T, D, None)
    need = lib.mhc_layer_norm_bwd_workspace_size(4, 8, 1)
    assert need >= 2 * 8 * 4
    assert b(None, 0) == -1 and b"workspace" in _err()
    assert b(P, need - 1) == -1 and b"workspace" in _err()
    assert b(P, need, T=0) == 0
    assert lib.mhc_layer_norm_bwd(None, P, 1, P, 0, P, P, P, P, P, P, need, 4, 8, None) == -1
    assert lib.mhc_layer_norm_bwd_workspace_size(0, 8, 1) == 0


def test_gated_ffn_refusals():
    lib = _lib.load()
    need = lib.mhc_gated_ffn_fwd_workspace_size(4, 16, 24, 16, 1)
    assert need > 0
    f = lambda x=P, dt=1, act=0, out=P, g=None, u=None, h=None, ws=P, n=need, T=4, D=16, F=24: lib.mhc_gated_ffn_fwd(
        x, P, P, P, dt, act, out, g, u, h, ws, n, T, D, F, 16, None)
    assert f(x=None) == -1 and b"null" in _err()
    assert f(x=ODD) == -1 and b"aligned" in _err()
    assert f(dt=3) == -2 and f(act=4) == -1 and f(act=-1) == -1
    assert f(D=0) == -1 and f(F=0) == -1 and f(T=-1) == -1
    assert f(g=P) == -1 and b"together" in _err()
    assert f(g=P, u=P) == -1 and b"together" in _err()
    assert f(n=need - 1) == -1 and b"workspace" in _err()
    assert f(ws=None) == -1 and b"workspace" in _err()
    assert f(T=0) == 0
    assert f(T=1 << 32) == -2
    need = lib.mhc_gated_ffn_bwd_workspace_size(4, 16, 24, 16, 1)
    assert need > 0
    b = lambda go=P, h=P, gx=P, ws=P, n=need, T=4: lib.mhc_gated_ffn_bwd(
        go, P, P, P, P, P, P, h, 1, 0, gx, P, P, P, ws, n, T, 16, 24, 16, None)
    assert b(go=None) == -1 and b(h=None) == -1 and b(gx=None) == -1
    assert b(h=ODD) == -1 and b"aligned" in _err()
    assert b(n=need - 1) == -1 and b"workspace" in _err()
    assert b(T=0) == 0


def test_dropout_refusals():
    lib = _lib.load()
    f = lambda x=P, n=8, dt=1, p=0.5: lib.mhc_dropout(x, P, n, dt, p, 0, 0, None, None)
    assert f(x=None) == -1 and b"null" in _err()
    assert f(n=-1) == -1 and f(p=-0.1) == -1 and f(p=1.5) == -1 and f(p=float("nan")) == -1
    assert f(dt=5) == -2
    assert f(n=0) == 0


def test_operators_refuse_cpu_tensors():
    x, w = torch.zeros(4, 16), torch.zeros(8, 16)
    for call in (lambda: S.layer_norm(x), lambda: S.layer_norm_backward(x, x, None, x[:, 0], x[:, 0]),
                 lambda: S.gated_ffn(x, w, w, w.t()), lambda: S.dropout(x, 0.5), lambda: S.dropout_backward(x, 0.5),
                 lambda: S.layer_norm_fn(x), lambda: S.gated_ffn_fn(x, w, w, w.t()), lambda: S.dropout_fn(x, 0.5)):
        with pytest.raises(RuntimeError, match="HIP"):
            call()


@pytest.mark.parametrize("shape", [(5, 7), (2, 3, 33), (1, 1)])
def test_layer_norm_ref(shape):
    g = torch.Generator().manual_seed(1)
    x, w, b = torch.randn(shape, generator=g), torch.randn(shape[-1], generator=g), torch.randn(shape[-1], generator=g)
    torch.testing.assert_close(S.layer_norm_ref(x, w, b), R.norm_fwd(x, w, b, 1e-5)[0].float())
    torch.testing.assert_close(S.layer_norm_ref(x), R.norm_fwd(x, None, None, 1e-5)[0].float())


@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh", "relu"])
def test_gated_ffn_formulas(kind):
    """The reference against the 64-bit formulas, and the formulas' gradients against differences."""
    g = torch.Generator().manual_seed(2)
    t = [torch.randn(s, generator=g) for s in ((6, 10), (14, 10), (14, 10), (9, 14))]
    torch.testing.assert_close(S.gated_ffn_ref(*t, kind), R.ffn_fwd(*t, kind)[0].float(), rtol=2e-5, atol=2e-5)
    go = torch.randn(6, 9, generator=g)
    for i, gr in enumerate(R.ffn_bwd(go, *t, kind)):
        v = torch.randn(t[i].shape, generator=g).double()
        f = lambda s: float((R.ffn_fwd(*[a.double() + s * v if j == i else a for j, a in enumerate(t)], kind)[0] * go).sum())
        num = (f(1e-6) - f(-1e-6)) / 2e-6
        assert abs(num - float((gr * v).sum())) <= 1e-6 * float(gr.norm() * v.norm())


def test_layer_norm_formula_gradients_against_differences():
    g = torch.Generator().manual_seed(3)
    x, w, gy = (torch.randn(s, generator=g).double() for s in ((4, 11), (11,), (4, 11)))
    gx, gw, gb, _, _ = R.norm_bwd(gy, x, w, 1e-5)
    for i, gr in ((0, gx), (1, gw)):
        v = torch.randn((x, w)[i].shape, generator=g).double()
        f = lambda s: float((R.norm_fwd(*[a + s * v if j == i else a for j, a in enumerate((x, w))], None, 1e-5)[0] * gy).sum())
        assert abs((f(1e-6) - f(-1e-6)) / 2e-6 - float((gr * v).sum())) <= 1e-6 * float(gr.norm() * v.norm())
    torch.testing.assert_close(gb, gy.sum(0))


def test_philox_known_answers():
    """The published known-answer vectors of Philox4x32-10."""
    assert R.philox(0, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = (1 << 64) - 1
    assert R.philox(ones, ones, ones) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    for seed, off in ((0, 0), ((1 << 63) + 5, (1 << 40) + 3)):
        got = philox_ref(300, seed, off)
        assert [[int(v) for v in r] for r in got[[0, 1, 299]]] == [R.philox(i, seed, off) for i in (0, 1, 299)]


def test_dropout_ref():
    x = torch.arange(1, 22, dtype=torch.float32).reshape(3, 7)
    for p in (0.0, 0.3, 1.0):
        t = int(p * 65536 + 0.5)
        want = []
        for i, v in enumerate(x.flatten().tolist()):
            w = R.philox(i // 8, 9, 4)[(i % 8) // 2]
            keep = (w >> (16 * (i % 2)) & 0xFFFF) >= t
            want.append(v * 65536.0 / (65536 - t) if keep else 0.0)
        torch.testing.assert_close(S.dropout_ref(x, p, 9, 4), torch.tensor(want).reshape(3, 7))
