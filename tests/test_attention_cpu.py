"""Rotary positions and attention without a GPU: C entry points' refusals, the
Python operators' checks, the *_ref functions and the formulas' gradients."""

from __future__ import annotations

import ctypes
import math
import sys

import pytest
import torch

import attention_ref as R
from FlagOS_mhc import _lib, sublayer as S
from FlagOS_mhc.attention import _ARGS, _STRIDES
from FlagOS_mhc.rotary import _ARGS as _ROTARY

P = 0x1000
ODD = 0x1002


def _err():
    return _lib.load().mhc_last_error()


def _args(q=P, k=P, v=P, qs=(0, 128, 64), ks=(0, 64, 64), vs=(0, 64, 64), cu_q=P, cu_k=P, lengths=0, rows_q=16,
          rows_k=16, B=2, H=2, Hk=1, d=64, dtype=1, causal=1, scale=0.125):
    return _ARGS.pack(q, k, v, *qs, *ks, *vs, cu_q, cu_k, lengths, rows_q, rows_k, B, H, Hk, d, dtype, causal, scale, 0)


@pytest.mark.parametrize("bad,code,text", [
    (dict(dtype=3), -2, b"dtype"), (dict(H=0), -1, b"heads"), (dict(H=3, Hk=2), -1, b"heads"), (dict(d=0), -1, b"d=0"),
    (dict(d=12), -2, b"whole 16"), (dict(d=264), -2, b"512"), (dict(dtype=0, d=132), -2, b"512"),
    (dict(rows_q=-1), -1, b"rows_q"), (dict(rows_q=(1 << 30) + 1), -2, b"above"), (dict(rows_k=(1 << 30) + 1), -2, b"above"),
    (dict(scale=0.0), -1, b"scale"), (dict(scale=-1.0), -1, b"scale"), (dict(scale=float("nan")), -1, b"scale"),
    (dict(scale=float("inf")), -1, b"scale"), (dict(q=0), -1, b"null"), (dict(v=0), -1, b"null"), (dict(k=ODD), -1, b"16 bytes"),
    (dict(qs=(0, 132, 64)), -1, b"16 bytes"), (dict(ks=(0, 56, 64)), -1, b"strides"), (dict(vs=(0, 64, -64)), -1, b"strides"),
    (dict(ks=(0, 1 << 24, 64)), -1, b"strides"), (dict(lengths=P), -1, b"lengths_k"),
    (dict(cu_q=0, rows_q=15), -1, b"sequences"), (dict(cu_k=0, rows_k=15), -1, b"sequences"),
    (dict(cu_q=0, B=0), -1, b"sequences"), (dict(B=-1), -1, b"sequences")])
def test_attention_refusals(bad, code, text):
    lib = _lib.load()
    a = _args(**bad)
    assert lib.mhc_attention_fwd(a, P, None, P, 1 << 40, None) == code and text in _err(), _err()
    st = _STRIDES.pack(0, 128, 64)
    assert lib.mhc_attention_bwd(a, P, st, P, P, P, P, P, P, 1 << 40, None) == code and text in _err(), _err()
    assert lib.mhc_attention_fwd_workspace_size(a) == lib.mhc_attention_bwd_workspace_size(a) == 0


def test_attention_buffers_refused():
    lib = _lib.load()
    assert lib.mhc_attention_fwd(None, P, None, P, 1, None) == -1
    a = _args()
    assert lib.mhc_attention_fwd(a, None, None, P, 1, None) == -1 and b"out" in _err()
    assert lib.mhc_attention_fwd(a, ODD, None, P, 1, None) == -1 and b"out" in _err()
    st = _STRIDES.pack(0, 128, 64)
    need = lib.mhc_attention_bwd_workspace_size(a)
    assert need >= 2 * 16 * 4
    ok = [a, P, st, P, P, P, P, P, P, need, None]
    for i in (1, 2, 3, 4, 5, 6, 7, 8):
        bad = list(ok)
        bad[i] = None
        assert lib.mhc_attention_bwd(*bad) == -1, i
    for i in (3, 5, 6, 7, 8):
        bad = list(ok)
        bad[i] = ODD
        assert lib.mhc_attention_bwd(*bad) == -1 and b"16-byte" in _err(), i
    ok[9] = need - 1
    assert lib.mhc_attention_bwd(*ok) == -1 and b"workspace" in _err()
    # one token over a long cache: parts of the keys need a workspace
    a = _args(cu_q=0, cu_k=0, rows_q=1, rows_k=32768, B=1)
    need = lib.mhc_attention_fwd_workspace_size(a)
    assert need > 0
    assert lib.mhc_attention_fwd(a, P, None, None, 0, None) == -1 and b"workspace" in _err()
    assert lib.mhc_attention_fwd(a, P, None, P, need - 1, None) == -1 and b"workspace" in _err()


def test_nothing_to_do():
    lib = _lib.load()
    assert lib.mhc_attention_fwd(_args(q=0, cu_q=0, cu_k=0, rows_q=0, B=1), None, None, None, 0, None) == 0
    a = _args(q=0, k=0, v=0, cu_q=0, cu_k=0, rows_q=0, rows_k=0, B=1)
    assert lib.mhc_attention_bwd(a, None, _STRIDES.pack(0, 128, 64), None, None, None, None, None, None, 0, None) == 0


def test_rotary_refusals():
    lib = _lib.load()
    f = lambda q=P, k=P, dt=1, freqs=P, pos=P, cu=0, seqs=0, length=4, layout=0, qo=P, ko=P, T=4, H=2, Hk=1, d=64, r=64, \
        row=128, flags=0: lib.mhc_rotary(_ROTARY.pack(q, k, qo, ko, freqs, pos, cu, row, 64, 64, 64, T, length, 1.0, seqs, dt, H,
                                                      Hk, d, r, layout, flags), None)
    assert f(T=-1) == -1 and f(H=0) == -1 and f(Hk=-1) == -1 and f(d=0) == -1 and f(r=66) == -1 and f(r=7) == -1
    assert f(layout=2) == -1 and f(row=-1) == -1 and f(flags=4) == -1
    assert f(dt=5) == -2 and b"dtype" in _err()
    assert f(d=8192, r=4098) == -2 and b"r=4098" in _err()
    assert f(H=1 << 20, d=1 << 12) == -2
    assert f(pos=0, length=0) == -1 and f(pos=0, cu=P, seqs=-1) == -1
    assert f(q=0) == -1 and f(qo=0) == -1 and f(k=0) == -1 and f(ko=0) == -1 and f(freqs=0) == -1
    assert f(T=0) == 0 and lib.mhc_rotary(None, None) == -1


# ---- Python checks ------------------------------------------------------------------

@pytest.fixture
def on_cpu(monkeypatch):
    """The operators' own checks, without a device."""
    monkeypatch.setattr(_lib, "require_device", lambda *a: None)
    monkeypatch.setattr(sys.modules["FlagOS_mhc.attention"], "_workspace_size", lambda *a: 0)
    monkeypatch.setattr(_lib, "call", lambda *a: None)


def t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


CU = torch.tensor([0, 3, 6], dtype=torch.int32)


@pytest.mark.parametrize("args,kw,error,text", [
    ((t(6, 4, 64), t(6, 2, 64), t(6, 2, 64).half()), {}, ValueError, "one type"),
    ((t(6, 4, 64).double(),) * 3, {}, NotImplementedError, "dtype"),
    ((t(6, 4, 64), t(6, 2, 32), t(6, 2, 32)), {}, ValueError, "do not fit"),
    ((t(6, 4, 64), t(6, 2, 64), t(5, 2, 64)), {}, ValueError, "do not fit"),
    ((t(4, 64), t(2, 64), t(2, 64)), {}, ValueError, "do not fit"),
    ((t(6, 3, 64), t(6, 2, 64), t(6, 2, 64)), {}, ValueError, "groups"),
    ((t(6, 0, 64), t(6, 2, 64), t(6, 2, 64)), {}, ValueError, "groups"),
    ((t(6, 4, 264), t(6, 2, 264), t(6, 2, 264)), {}, NotImplementedError, "width"),
    ((t(6, 4, 132, dtype=torch.float32),) * 3, {}, NotImplementedError, "width"),
    ((t(6, 4, 64), t(6, 2, 64), t(6, 2, 64)), dict(scale=0.0), ValueError, "scale"),
    ((t(6, 4, 64), t(6, 2, 64), t(6, 2, 64)), dict(scale=float("nan")), ValueError, "scale"),
    ((t(2, 3, 4, 64), t(2, 3, 2, 64), t(2, 3, 2, 64), CU), {}, ValueError, "packed rows"),
    ((t(6, 4, 64), t(7, 2, 64), t(7, 2, 64), CU), {}, ValueError, "cu_seqlens_k"),
    ((t(6, 4, 64), t(6, 2, 64), t(6, 2, 64), CU.float()), {}, ValueError, "int32"),
    ((t(6, 4, 64), t(6, 2, 64), t(6, 2, 64), CU[:0]), {}, ValueError, "int32"),
    ((t(6, 4, 64), t(6, 2, 64), t(6, 2, 64), CU), dict(cu_seqlens_k=CU[:2]), ValueError, "sequences"),
    ((t(6, 4, 64), t(6, 2, 64), t(6, 2, 64), CU), dict(cu_seqlens_k=CU, lengths_k=CU[:2]), ValueError, "lengths_k"),
    ((t(6, 4, 64), t(3, 5, 2, 64), t(3, 5, 2, 64), CU), {}, ValueError, "sequences"),
    ((t(2, 3, 4, 64), t(2, 5, 2, 64), t(2, 5, 2, 64)), dict(lengths_k=CU), ValueError, "lengths_k"),
    ((t(2, 3, 4, 64), t(2, 5, 2, 64), t(2, 5, 2, 64)), dict(lengths_k=CU[:2].float()), ValueError, "lengths_k"),
    ((t(2, 3, 4, 64), t(2, 5, 2, 64), t(2, 5, 2, 64)), dict(cu_seqlens_k=CU), ValueError, "cu_seqlens_k"),
])
def test_attention_checks(on_cpu, args, kw, error, text):
    with pytest.raises(error, match=text):
        S.attention(*args, **kw)
    cu = args[3] if len(args) > 3 else None
    with pytest.raises(error, match=text):
        S.attention_backward(args[0], *args[:3], args[0], t(4, 6, dtype=torch.float32), cu, **kw)


def test_attention_backward_checks(on_cpu):
    q, k = t(6, 4, 64), t(6, 2, 64)
    lse = t(4, 6, dtype=torch.float32)
    with pytest.raises(ValueError, match="grad_out"):
        S.attention_backward(q[:5], q, k, k, q, lse)
    with pytest.raises(ValueError, match="grad_out"):
        S.attention_backward(q, q, k, k, q.float(), lse)
    with pytest.raises(ValueError, match="lse"):
        S.attention_backward(q, q, k, k, q, lse.t())
    with pytest.raises(ValueError, match="lse"):
        S.attention_backward(q, q, k, k, q, lse.half())


def test_rotary_checks(on_cpu):
    f, _ = S.rotary_frequencies(64, device="cpu")
    q, k = t(6, 4, 64), t(6, 2, 64)
    for args, kw, text in (((q[0], None, f), {}, "dimension"), ((q, k[:5], f), {}, "k of shape"), ((q, k.half(), f), {}, "k of shape"),
                           ((q, k, f.float()), {}, "freqs"), ((q[..., :32], None, f), {}, "freqs"),
                           ((q, k, f), dict(layout="pairs"), "layout"), ((q, k, f, CU), {}, "positions"),
                           ((q, k, f, torch.zeros(6)), {}, "positions"), ((q, k, f, torch.arange(6)), dict(cu_seqlens=CU), "cu_seqlens"),
                           ((q[None], k[None], f), dict(cu_seqlens=CU), "packed rows"), ((q, k[:, :0], f), {}, "no heads"),
                           ((q[:, :0], None, f), {}, "no heads")):
        with pytest.raises(ValueError, match=text):
            S.rotary(*args, **kw)
    with pytest.raises(NotImplementedError, match="dtype"):
        S.rotary(q.double(), None, f)


def test_cpu_tensors_refused():
    q, k = t(6, 4, 64), t(6, 2, 64)
    f, _ = S.rotary_frequencies(64, device="cpu")
    for call in (lambda: S.attention(q, k, k), lambda: S.attention_fn(q, k, k), lambda: S.rotary(q, k, f),
                 lambda: S.rotary_fn(q, k, f), lambda: S.rotary_backward(q, k, f),
                 lambda: S.attention_backward(q, q, k, k, q, q[..., 0].t().float())):
        with pytest.raises(RuntimeError, match="HIP"):
            call()


# ---- frequencies -------------------------------------------------------------------

def test_rotary_frequencies():
    f, a = S.rotary_frequencies(8, 100.0, device="cpu")
    assert f.dtype == torch.float64 and a == 1.0
    torch.testing.assert_close(f, torch.tensor([1.0, 100 ** -0.25, 100 ** -0.5, 100 ** -0.75], dtype=torch.float64))
    g, a = S.rotary_frequencies(8, 100.0, scaling="linear", factor=4.0, device="cpu")
    assert a == 1.0 and torch.equal(g, f / 4)
    g, a = S.rotary_frequencies(8, 100.0, scaling="ntk", factor=4.0, device="cpu")
    assert a == 1.0 and float(g[0]) == 1.0
    torch.testing.assert_close(g[-1], f[-1] / 4)  # the slowest pair is stretched by factor
    g, a = S.rotary_frequencies(128, scaling="yarn", factor=16.0, original_length=4096, device="cpu")
    f, _ = S.rotary_frequencies(128, device="cpu")
    turns = 4096 * f / (2 * math.pi)
    assert a == 0.1 * math.log(16.0) + 1.0
    assert torch.equal(g[turns >= 32], f[turns >= 32])
    torch.testing.assert_close(g[turns <= 1], f[turns <= 1] / 16, rtol=1e-15, atol=0)
    mid = (turns > 1) & (turns < 32)
    assert bool(mid.any()) and bool(((g < f) & (g > f / 16))[mid].all())


@pytest.mark.parametrize("args,kw", [((7,), {}), ((0,), {}), ((8, 0.0), {}), ((8,), dict(scaling="cubic")),
                                     ((8,), dict(scaling="linear", factor=0.0)), ((8,), dict(scaling="yarn", factor=2.0)),
                                     ((8,), dict(scaling="yarn", factor=2.0, original_length=0)),
                                     ((8,), dict(scaling="yarn", factor=2.0, original_length=64, turns=(3.0, 2.0))),
                                     ((8, float("inf")), {})])
def test_rotary_frequencies_refused(args, kw):
    with pytest.raises(ValueError):
        S.rotary_frequencies(*args, device="cpu", **kw)


# ---- references -------------------------------------------------------------------

@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_ref(layout):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 2, 12, generator=g)
    f, a = S.rotary_frequencies(8, 50.0, scaling="yarn", factor=4.0, original_length=64, device="cpu")
    p = torch.tensor([0, 3, 100, -2, 7])
    got = S.rotary_ref(x, f, p, layout, a)
    z = torch.polar(torch.full((5, 4), a, dtype=torch.float64), p.double()[:, None] * f)[:, None]
    xd = x.double()
    pair = (xd[..., :4], xd[..., 4:8]) if layout == "half" else (xd[..., 0:8:2], xd[..., 1:8:2])
    w = torch.complex(*pair) * z
    want = xd.clone()
    if layout == "half":
        want[..., :4], want[..., 4:8] = w.real, w.imag
    else:
        want[..., 0:8:2], want[..., 1:8:2] = w.real, w.imag
    torch.testing.assert_close(got, want.float())


def test_attention_ref():
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g)
    q, k, v = r(13, 4, 8), r(13, 2, 8), r(13, 2, 8)
    cu = torch.tensor([0, 5, 5, 11], dtype=torch.int32)
    for causal in (True, False):
        want, _ = R.full(q, k, v, None, cu, cu, None, 3, causal, 8 ** -0.5)
        torch.testing.assert_close(S.attention_ref(q, k, v, cu, causal=causal), want[0][0].float())
    qb, kb, vb = r(2, 3, 4, 8), r(2, 7, 2, 8), r(2, 7, 2, 8)
    lengths = torch.tensor([7, 2], dtype=torch.int32)
    flat = lambda t: t.reshape(-1, *t.shape[-2:])
    want, _ = R.full(flat(qb), flat(kb), flat(vb), None, None, None, lengths, 2, True, 0.3)
    got = S.attention_ref(qb, kb, vb, lengths_k=lengths, scale=0.3)
    torch.testing.assert_close(got, want[0][0].view_as(got).float())
    assert not got[1, 0].any()  # the first of three queries over two keys sees none


@pytest.mark.parametrize("n,m,causal", [(6, 6, True), (3, 8, True), (7, 4, True), (5, 9, False)])
def test_attention_formula_gradients_against_differences(n, m, causal):
    g = torch.Generator().manual_seed(n * 10 + m)
    q, k, v, go = (torch.randn(s, 5, generator=g).double() for s in (n, m, m, n))
    _, _, grads = R.head(q, k, v, go, 0.4, causal, torch.float32)
    for i, (gr, _) in enumerate(grads):
        u = torch.randn(gr.shape, generator=g).double()
        f = lambda s: float((R.head(*[x + s * u if j == i else x for j, x in enumerate((q, k, v))], None, 0.4, causal,
                                    torch.float32)[0][0] * go).sum())
        assert abs((f(1e-5) - f(-1e-5)) / 2e-5 - float((gr * u).sum())) <= 1e-7 * float(1 + gr.norm() * u.norm())


def test_struct_is_the_headers():
    """The packed arguments have the C struct's layout."""
    class Args(ctypes.Structure):
        _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v")] + [(n, ctypes.c_int64 * 3) for n in ("qs", "ks", "vs")]
                    + [(n, ctypes.c_void_p) for n in ("cq", "ck", "len")] + [(n, ctypes.c_int64) for n in ("rq", "rk")]
                    + [(n, ctypes.c_int32) for n in ("seqs", "heads", "heads_k", "d", "dtype", "causal")]
                    + [("scale", ctypes.c_float), ("reserved", ctypes.c_int32)])
    assert ctypes.sizeof(Args) == _ARGS.size
    a = Args.from_buffer_copy(_args(B=7, H=6, Hk=3, d=40, scale=0.25, rows_k=99, vs=(1, 2, 3)))
    assert (a.seqs, a.heads, a.heads_k, a.d, a.scale, a.rk, list(a.vs), a.ck) == (7, 6, 3, 40, 0.25, 99, [1, 2, 3], P)


def test_rotary_struct_is_the_headers():
    class Args(ctypes.Structure):
        _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "qo", "ko", "freqs", "positions", "cu")]
                    + [(n, ctypes.c_int64) for n in ("q_row", "q_head", "k_row", "k_head", "rows", "length")]
                    + [("amplitude", ctypes.c_float)]
                    + [(n, ctypes.c_int32) for n in ("sequences", "dtype", "heads", "heads_k", "d", "r", "layout", "flags")])
    raw = _ROTARY.pack(*range(1, 8), *range(8, 14), 0.5, *range(14, 22))
    # (the C struct ends on a multiple of 8 bytes: its last one is four whole ones here)
    assert ctypes.sizeof(Args) - _ROTARY.size in (0, 4)
    a = Args.from_buffer_copy(raw + bytes(ctypes.sizeof(Args) - _ROTARY.size))
    assert (a.q, a.cu, a.q_row, a.length, a.amplitude, a.sequences, a.flags) == (1, 7, 8, 13, 0.5, 14, 21)
