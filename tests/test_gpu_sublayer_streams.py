"""Dropout over more elements than its grid has threads for, and the sublayer's
operators on two streams at one time."""

from __future__ import annotations

import pytest
import torch

import sublayer_ref as R
from FlagOS_mhc import sublayer as S
from test_gpu_sublayer import DEV, DT, _ffn_inputs, _gen, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_dropout_past_its_grid(dtype):
    """A thread takes every (16 blocks a CU x 256 threads)-th group of 8: 8.39 M
    elements on 256 CUs.  Forward and backward, values and mask."""
    n, dt, p, seed, off = 20_000_003, DT[dtype], 0.3, 21, 1 << 33
    print(f"[dropout] n={n} {dtype}", flush=True)
    x = _randn(_gen(n), n, dtype=dt)
    t = int(p * 65536 + 0.5)
    kept = S.dropout_ref(torch.ones(n), p, seed, off).ne(0).to(DEV)
    exact = torch.where(kept, x.double() * (65536.0 / (65536 - t)), 0.0)
    # the factor's and the product's fp32 roundings, then the type's: half a step, which below the
    # smallest normal number is that number's
    bound = R.half_step(dt) * exact.abs().clamp(min=torch.finfo(dt).tiny) + 2 * R.ULP32 * exact.abs()
    for y in (S.dropout(x, p, seed, off), S.dropout_backward(x, p, seed, off)):
        assert bool(((y.double() - exact).abs() <= bound * kept).all())


def _work(i, T, D, F):
    x, wg, wu, wd, go = _ffn_inputs(T, D, F, D, torch.bfloat16, 40 + i)
    w = _randn(_gen(50 + i), D)
    state = torch.tensor([i, 3], device=DEV)

    def step():
        n = S.layer_norm(x, w, None, need_backward=True)
        f = S.gated_ffn(n["y"], wg, wu, wd, need_backward=True)
        y = S.dropout(f["out"], 0.2, state=state)
        gn, *gw = S.gated_ffn_backward(S.dropout_backward(go, 0.2, state=state), n["y"], wg, wu, wd, f["gate"], f["up"],
                                       f["hidden"])
        return [y, *S.layer_norm_backward(gn, x, w, n["mean"], n["rstd"]), *gw]
    return step


# runs of k and tails (partial sums), padded copies, sums over the rows, few tokens
@pytest.mark.parametrize("T,D,F", [(2051, 1024, 2816), (300, 1003, 2677), (64, 2048, 5632), (3, 1024, 4096)])
def test_two_streams_at_one_time(T, D, F):
    """Nothing waits between the two: each has its own workspaces and results."""
    print(f"[streams] T={T} D={D} F={F}", flush=True)
    steps = [_work(i, T, D, F) for i in range(2)]
    want = [s() for s in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    got = [[], []]
    for _ in range(4):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(steps[i]())
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))
