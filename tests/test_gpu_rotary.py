"""Rotary positions on the GPU against 64-bit formulas."""

from __future__ import annotations

import pytest
import torch

import attention_ref as R
from FlagOS_mhc import sublayer as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


def _want(x, freqs, positions, layout, amplitude, sign=1):
    """(value, bound): the sine's and cosine's fp32 values (8 U), two products and a sum (3 U), the type."""
    w = positions.double()[..., None] * freqs * sign
    cos, sin = (f(w)[..., None, :] * amplitude for f in (torch.cos, torch.sin))
    r = 2 * freqs.numel()
    y, size = x.double().clone(), x.double().abs()
    i = torch.arange(r // 2, device=DEV)
    a, b = (i, i + r // 2) if layout == "half" else (2 * i, 2 * i + 1)
    xa, xb = x.double()[..., a], x.double()[..., b]
    y[..., a], y[..., b] = xa * cos - xb * sin, xa * sin + xb * cos
    size[..., a] = size[..., b] = (xa.abs() + xb.abs()) * amplitude
    bound = R.half_step(x.dtype) * y.abs() + 12 * R.U * size
    bound[..., r:] = 0.0
    # below the smallest normal number of fp16 half a step is that number's
    return y, bound + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)


# T, H, Hk, d, r: whole vectors, parts of the head, odd widths
SHAPES = [(1, 1, 1, 64, 64), (64, 32, 8, 128, 128), (5, 3, 1, 80, 40), (33, 4, 2, 96, 32), (130, 2, 2, 128, 16),
          (17, 5, 5, 33, 10), (1, 2, 1, 2, 2), (4100, 4, 1, 64, 32), (9, 2, 1, 256, 256), (3, 1, 1, 5000, 4096)]


@pytest.mark.parametrize("T,H,Hk,d,r", SHAPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_rotary(T, H, Hk, d, r, layout, dtype):
    print(f"[rotary] T={T} H={H} Hk={Hk} d={d} r={r} {layout} {dtype}", flush=True)
    g = _gen(T + d + r)
    q, k = _randn(g, T, H, d, dtype=DT[dtype]), _randn(g, T, Hk, d, dtype=DT[dtype])
    freqs, amp = S.rotary_frequencies(r, scaling="yarn", factor=4.0, original_length=2048)
    pos = torch.randint(-5, 1 << 20, (T,), device=DEV, generator=g)
    for p in (pos, pos.int()):
        for fn, sign in ((S.rotary, 1), (S.rotary_backward, -1)):
            out = fn(q, k, freqs, p, layout=layout, amplitude=amp)
            for name, x, y in zip("qk", (q, k), out):
                assert y.dtype == x.dtype
                R.within(y, _want(x, freqs, p, layout, amp, sign), f"{fn.__name__} {name}")
    alone, none = S.rotary(q, None, freqs, pos, layout=layout, amplitude=amp)
    assert none is None and torch.equal(alone, S.rotary(q, k, freqs, pos, layout=layout, amplitude=amp)[0])


def test_positions_of_packed_and_batched_rows():
    g = _gen(1)
    lengths = [3, 0, 70, 1, 0]
    T = sum(lengths) + 4
    q, k = _randn(g, T, 4, 64), _randn(g, T, 2, 64)
    freqs, _ = S.rotary_frequencies(64)
    cu = torch.tensor([0, 3, 3, 73, 74, 74], dtype=torch.int32, device=DEV)
    want = torch.tensor([i for n in lengths + [4] for i in range(n)], device=DEV)
    for a, b in zip(S.rotary(q, k, freqs, cu_seqlens=cu), S.rotary(q, k, freqs, want)):
        assert torch.equal(a, b)
    many = torch.arange(201, dtype=torch.int32, device=DEV)  # more sequences than lanes
    x = _randn(g, 230, 2, 64)
    want = torch.cat([torch.zeros(200, dtype=torch.int64), torch.arange(30)]).to(DEV)
    assert torch.equal(S.rotary(x, None, freqs, cu_seqlens=many)[0], S.rotary(x, None, freqs, want)[0])
    b = _randn(g, 3, 50, 2, 64)
    want = torch.arange(50, device=DEV).repeat(3)
    assert torch.equal(S.rotary(b, None, freqs)[0], S.rotary(b.view(150, 2, 64), None, freqs, want)[0].view_as(b))


def test_views_streams_and_empty():
    g = _gen(2)
    freqs, _ = S.rotary_frequencies(64)
    qkv = _randn(g, 2, 40, 8, 64, dtype=torch.bfloat16)
    q, k = qkv[:, :, :4], qkv[:, :, 4:6]
    want = S.rotary(q.contiguous(), k.contiguous(), freqs)
    for a, b in ((q, k), (q.transpose(2, 3).contiguous().transpose(2, 3), k), (q.transpose(0, 1).contiguous().transpose(0, 1), k)):
        assert all(torch.equal(x, y) for x, y in zip(S.rotary(a, b, freqs), want))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = S.rotary(q, k, freqs)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    a, b = S.rotary(q[:0], k[:0], freqs)
    assert a.shape == (0, 40, 4, 64) and b.shape == (0, 40, 2, 64)


def test_autograd():
    g = _gen(3)
    freqs, _ = S.rotary_frequencies(32)
    q, k = (_randn(g, 20, n, 64, dtype=torch.bfloat16).requires_grad_(True) for n in (4, 2))
    gq, gk = (_randn(g, 20, n, 64, dtype=torch.bfloat16) for n in (4, 2))
    a, b = S.rotary_fn(q, k, freqs, layout="interleaved")
    torch.autograd.backward((a, b), (gq, gk))
    want = S.rotary_backward(gq, gk, freqs, layout="interleaved")
    assert torch.equal(q.grad, want[0]) and torch.equal(k.grad, want[1])
    q.grad = k.grad = None
    S.rotary_fn(q, k, freqs)[1].backward(gk)  # k's alone
    assert q.grad is None and torch.equal(k.grad, S.rotary_backward(gk, None, freqs)[0])
    q.grad = None
    S.rotary_fn(q, None, freqs)[0].backward(gq)
    assert torch.equal(q.grad, S.rotary_backward(gq, None, freqs)[0])


def test_rotation_by_a_difference():
    """Products of rotated queries and keys depend on the difference of their positions."""
    g = _gen(4)
    freqs, _ = S.rotary_frequencies(128)
    q, k = _randn(g, 1, 1, 128).double(), _randn(g, 1, 1, 128).double()
    vals = []
    for p in (0, 1000, 500000):
        a = S.rotary(q.float(), None, freqs, torch.tensor([p + 7], device=DEV))[0]
        b = S.rotary(k.float(), None, freqs, torch.tensor([p], device=DEV))[0]
        vals.append(float((a.double() * b.double()).sum()))
    size = float(q.norm() * k.norm())
    assert max(vals) - min(vals) <= 2 * 24 * 2 ** -24 * size


@pytest.mark.parametrize("off,pad", [(1, 0), (0, 1), (3, 5), (4, 4)])
@pytest.mark.parametrize("d,r", [(80, 40), (64, 64), (48, 24), (36, 20)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_any_alignment_and_stride(off, pad, d, r, layout, dtype):
    """Views that begin and step at any element: the same bits as of copies."""
    g = _gen(off + pad)
    T, H = 37, 3
    buf = _randn(g, off + T * H * (d + pad) + 8, dtype=DT[dtype])
    q = buf[off:off + T * H * (d + pad)].view(T, H, d + pad)[..., :d]
    k = buf[off:off + T * (H * (d + pad))].view(T, H, d + pad)[:, :2, :d]
    freqs, _ = S.rotary_frequencies(r)
    pos = torch.randint(0, 1 << 17, (T,), device=DEV, generator=g)
    for got, want in zip(S.rotary(q, k, freqs, pos, layout=layout),
                         S.rotary(q.contiguous(), k.contiguous(), freqs, pos, layout=layout)):
        assert torch.equal(got, want)
    R.within(S.rotary(q, k, freqs, pos, layout=layout)[0], _want(q, freqs, pos, layout, 1.0), "q")


@pytest.mark.parametrize("d,r", [(36, 18), (38, 6), (46, 22), (40, 4), (44, 40), (20, 0)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_parts_of_every_width(d, r, layout, dtype):
    """Turned and copied parts that are whole accesses of 16 bytes, of 8, or of neither; r = 0 copies."""
    g = _gen(d + r)
    q, k = _randn(g, 1031, 3, d, dtype=DT[dtype]), _randn(g, 1031, 1, d, dtype=DT[dtype])
    freqs = S.rotary_frequencies(r)[0] if r else torch.empty(0, dtype=torch.float64, device=DEV)
    pos = torch.arange(1031, device=DEV)
    for x, y in zip((q, k), S.rotary(q, k, freqs, layout=layout)):
        R.within(y, _want(x, freqs, pos, layout, 1.0), f"{d} {r}")
        assert torch.equal(y[..., r:], x[..., r:])
