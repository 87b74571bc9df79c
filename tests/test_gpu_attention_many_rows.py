"""More rows (queries times heads) than one dispatch has blocks for."""

from __future__ import annotations

import pytest
import torch

import attention_ref as R
from FlagOS_mhc import sublayer as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def test_short_sequences():
    """300000 packed sequences of two tokens, 32 heads of 8: 19.2 million rows, no parts of the keys."""
    B, H, Hk, d = 300_000, 32, 8, 8
    T, g = 2 * B, _gen(1)
    assert T * H > 1 << 24
    q, k, v = (torch.randn(T, n, d, device=DEV, generator=g).to(BF) for n in (H, Hk, Hk))
    cu = torch.arange(0, T + 1, 2, dtype=torch.int32, device=DEV)
    f = S.attention(q, k, v, cu, need_backward=True)
    grads = S.attention_backward(q, q, k, v, f["out"], f["lse"], cu)
    # a first token copies its value, in every sequence
    assert torch.equal(f["out"][::2], v[::2].repeat_interleave(H // Hk, 1))
    for lo in (0, T // 2, T - 80):
        rows = slice(lo, lo + 80)
        part = torch.arange(0, 81, 2, dtype=torch.int32, device=DEV)
        want, _ = R.full(q[rows], k[rows], v[rows], q[rows], part, part, None, 40, True, d ** -0.5)
        for name, got, w in zip(("out", "grad_q", "grad_k", "grad_v"), (f["out"], *grads), want):
            R.within(got[rows], w, f"{name} from {lo}")


def test_single_tokens_over_caches_in_parts():
    """262145 tokens of 64 heads over the same 2050 keys, in parts: 16.8 million rows are joined."""
    B, H, d, L = (1 << 18) + 1, 64, 8, 2050
    g = _gen(2)
    assert B * H > 1 << 24
    q = torch.randn(B, 1, H, d, device=DEV, generator=g).to(BF)
    k, v = (torch.randn(1, L, 1, d, device=DEV, generator=g).to(BF) for _ in range(2))
    f = S.attention(q, k.expand(B, L, 1, d), v.expand(B, L, 1, d), need_backward=True)
    for at in (slice(0, 64), slice(B // 2, B // 2 + 64), slice(B - 64, B)):
        want, lse = R.full(q[at, 0], k[0], v[0], None, None, None, None, 1, False, d ** -0.5)
        R.within(f["out"][at, 0], want[0], f"{at}")
        err = (f["lse"][:, at].double() - lse).abs()
        assert float(err.max()) <= 2.0 ** -12, float(err.max())
    assert bool(f["out"].isfinite().all())
