"""fp16 weights far below their row's largest: each keeps the precision of its own
size (64-bit results, every kernel of the forward)."""

from __future__ import annotations

import math

import pytest
import torch

import attention_ref as R
from FlagOS_mhc import sublayer as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16 = torch.float16


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


@pytest.mark.parametrize("S_,H,Hk", [(1, 4, 1), (40, 2, 1), (1100, 4, 4), (3500, 16, 16), (3500, 32, 8), (4200, 128, 8)])
@pytest.mark.parametrize("d", [64, 128])
def test_small_weights(S_, H, Hk, d):
    """Keys whose weights are 48.5 * 2^-24 of the row's largest, which lies in the same tile
    and has the value 0: each is off by no more than half a step of its own size.  Bounds:
    half a step (2^-11) for the weight and for the result, and the score's in fp32 (14
    times 8 U)."""
    print(f"[attention f16] weights {S_} {H} {d}", flush=True)
    L, g = 1024, _gen(S_)
    w = math.log(48.5 * 2.0 ** -24)
    k = torch.zeros(1, L, Hk, d, device=DEV, dtype=F16)
    k[..., 0] = w
    k[..., 1] = w - k[..., 0].float()
    k[:, ::32] = 0
    q = torch.zeros(1, S_, H, d, device=DEV, dtype=F16)
    q[..., :2] = 1
    v = (torch.rand(1, L, Hk, d, device=DEV, generator=g) * 100 + 100).to(F16)
    v[:, ::32] = 0
    out = S.attention(q, k, v, causal=False, scale=1.0)["out"]
    p = torch.softmax(k[0, :, 0, :2].double().sum(-1), 0)
    want = (p[:, None, None] * v[0].double()).sum(0).repeat_interleave(H // Hk, 0)
    assert float(want.min()) > 2.0 ** -10
    err = ((out[0].double() - want) / want).abs().max()
    assert float(err) <= 2 * R.half_step(F16) + 14 * 8 * R.U, float(err)
