"""Starts and lengths that are no sequences: the results mean nothing, but no
row outside the outputs is written, and the calls after it are right."""

from __future__ import annotations

import pytest
import torch

import attention_ref as R
from FlagOS_mhc import attention as A
from FlagOS_mhc import sublayer as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
GUARD, MARK = 1 << 16, 7.0  # elements on either side

T = 1000
STARTS = {
    "down": [0, 1000, 0, 1000], "all_down": [0, 900, 700, 500, 300, 100], "below_zero": [0, -5, 400, -2147483648, 1000],
    "past_the_end": [0, 300, 2147483647, 500, 1000], "first_not_zero": [600, 700, 800, 1000], "back_and_forth": [0, 1000, 1, 999] * 40,
}


@pytest.mark.parametrize("H", [4, 64])  # waves that share keys; blocks of 128
@pytest.mark.parametrize("name", STARTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_row_outside(monkeypatch, name, H, dtype):
    guarded = []

    def empty(self, like):
        n = like.numel()
        buf = torch.full((n + 2 * GUARD,), MARK, dtype=like.dtype, device=like.device)
        guarded.append((buf, n))
        return buf[GUARD:GUARD + n].view(like.shape)

    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    q, go = (torch.randn(T, H, 64, device=DEV, generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(T, 2, 64, device=DEV, generator=g).to(dtype) for _ in range(2))
    cu = torch.tensor(STARTS[name], dtype=torch.int32, device=DEV)
    good = torch.arange(0, T + 1, T // (cu.numel() - 1), dtype=torch.int32, device=DEV)[:cu.numel()]
    lse = torch.zeros(H, T, device=DEV)
    out = torch.zeros_like(q)
    with monkeypatch.context() as m:
        m.setattr(A._Call, "empty", empty)
        for cq, ck in ((cu, None), (cu, good), (good, cu)):
            S.attention(q, k, v, cq, cu_seqlens_k=ck, need_backward=True)
            S.attention_backward(go, q, k, v, out, lse, cq, cu_seqlens_k=ck)
        torch.cuda.synchronize()
    for buf, n in guarded:
        assert bool((buf[:GUARD] == MARK).all()) and bool((buf[GUARD + n:] == MARK).all())
    whole = torch.tensor([0, T], dtype=torch.int32, device=DEV)
    got = S.attention(q, k, v, whole)["out"]
    want, _ = R.full(q, k, v, go, whole, whole, None, 1, True, 0.125)
    R.within(got, want[0], name)


def test_lengths_past_the_cache_and_below_zero():
    g = torch.Generator(device=DEV)
    g.manual_seed(4)
    q = torch.randn(5, 1, 8, 64, device=DEV, generator=g).bfloat16()
    k, v = (torch.randn(5, 96, 2, 64, device=DEV, generator=g).bfloat16() for _ in range(2))
    wrong = torch.tensor([97, -1, 2147483647, -2147483648, 40], dtype=torch.int32, device=DEV)
    got = S.attention(q, k, v, lengths_k=wrong)["out"]
    assert torch.equal(got, S.attention(q, k, v, lengths_k=wrong.clamp(0, 96))["out"])


@pytest.mark.parametrize("name", STARTS)
def test_rotary(name):
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    q = torch.randn(T, 4, 64, device=DEV, generator=g)
    freqs, amplitude = S.rotary_frequencies(64)
    cu = torch.tensor(STARTS[name], dtype=torch.int32, device=DEV)
    S.rotary(q, None, freqs, cu_seqlens=cu, amplitude=amplitude)
    got, _ = S.rotary(q, None, freqs, torch.arange(T, device=DEV))
    again, _ = S.rotary(q, None, freqs)
    torch.cuda.synchronize()
    assert torch.equal(got, again)
