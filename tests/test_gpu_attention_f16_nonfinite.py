"""fp16: infinities and NaNs of one query, or key, and the factors that dS is packed
with: they are a lane's own, so no other row's result moves."""

from __future__ import annotations

import pytest
import torch

from FlagOS_mhc import sublayer as S
from test_gpu_attention import DEV, _cu, _gen, _randn
from test_gpu_attention_norms import KERNELS

pytestmark = pytest.mark.gpu
F16 = torch.float16
CALLS = [(n, d) for n, (_, _, _, widths) in KERNELS.items() for d in widths]


def _inputs(kernel, d):
    lengths, H, Hk, _ = KERNELS[kernel]
    g, T = _gen(d), sum(lengths)
    return [_randn(g, T, n, d, dtype=F16) for n in (H, Hk, Hk, H)], _cu(lengths), lengths[0]


@pytest.mark.parametrize("kernel,d", CALLS)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_a_query_s_gradient(kernel, d, value):
    """Every key seen: dq of the other queries, and everything of the other sequences, keep their bits."""
    print(f"[attention f16 nonfinite] {kernel} {d} {value}", flush=True)
    (q, k, v, go), cu, n = _inputs(kernel, d)
    at = n // 2 + 3
    f = S.attention(q, k, v, cu, causal=False, need_backward=True)
    run = lambda: S.attention_backward(go, q, k, v, f["out"], f["lse"], cu, causal=False)
    want = run()
    go[at, 0, 5] = value
    got = run()
    rest = torch.ones(q.shape[0], dtype=torch.bool, device=DEV)
    rest[at] = False
    assert torch.equal(got[0][rest], want[0][rest]) and torch.equal(got[0][at, 1:], want[0][at, 1:])
    assert not bool(got[0][at, 0].isfinite().any())
    for a, b in zip(got[1:], want[1:]):
        assert torch.equal(a[n:], b[n:]) and torch.equal(a[:, 1:], b[:, 1:])
    assert not bool(got[1][:n, 0].isfinite().any()) and not bool(got[2][:n, 0, 5].isfinite().any())
    assert bool(got[2][:n, 0, :5].isfinite().all())


@pytest.mark.parametrize("kernel,d", CALLS)
def test_hidden_rows(kernel, d):
    """Causal, as test_gpu_attention_blocks.test_hidden_nans_in_blocks in bf16: a broken key or value
    reaches no query before it, a broken query or gradient no key behind it."""
    print(f"[attention f16 hidden] {kernel} {d}", flush=True)
    (q, k, v, go), cu, n = _inputs(kernel, d)
    at = n // 2 + 3

    def run():
        f = S.attention(q, k, v, cu, need_backward=True)
        return (f["out"], *S.attention_backward(go, q, k, v, f["out"], f["lse"], cu))

    def near(a, b, *rows):  # a tile with such a row is summed in another order: fp32 sums, one rounding
        for r in rows:
            x, y = a[r].double(), b[r].double()
            assert bool(x.isfinite().all()) and float((x - y).norm()) <= 2 ** -11 * float(y.norm())

    want = run()
    before, behind, other = slice(0, at), slice(at + 1, n), slice(n, None)
    for t, ok in ((k, 1), (v, 1), (q, 2), (go, 2)):
        for value in (float("nan"), float("inf")):
            old = t[at].clone()
            t[at, 0, 3] = value
            got = run()
            if ok == 1:
                near(got[0], want[0], before, other)
                near(got[1], want[1], before, other)
            else:
                for i in (2, 3):
                    near(got[i], want[i], behind, other)
                near(got[1], want[1], before, behind, other)
            t[at] = old
