"""Keys and values that need no gradient (a prefix's, a cache's): theirs are neither
computed nor allocated, through the function and the registered op, eager and
compiled."""

from __future__ import annotations

import sys

import pytest
import torch

from FlagOS_mhc import _lib, library as L, sublayer as S
from FlagOS_mhc.attention import _STRIDES
from test_attention_cpu import ODD, P, _args, _err
from test_attention_library import DEV, _gen

OPS = torch.ops.flagos_mhc


def test_meta_shapes_without_the_keys_gradients():
    with torch.device("meta"):
        q, k, lse = torch.empty(6, 4, 64, dtype=torch.bfloat16), torch.empty(6, 2, 64, dtype=torch.bfloat16), torch.empty(4, 6)
        got = OPS.attention_backward(q, q, k, k, q, lse, None, None, None, True, None, False)
        assert [(tuple(t.shape), t.dtype) for t in got] == [((6, 4, 64), q.dtype), ((0,), q.dtype), ((0,), q.dtype)]


def test_c_entry_takes_both_or_none():
    """.. and then only D's workspace (one float a row and head)."""
    lib, st = _lib.load(), _STRIDES.pack(0, 128, 64)
    a = _args(rows_q=600, rows_k=600)
    run = lambda gq, gk, gv, n, args=a: lib.mhc_attention_bwd(args, P, st, P, P, gq, gk, gv, P, n, None)
    full, own = lib.mhc_attention_bwd_workspace_size(a), 2 * 600 * 4
    assert full > -(-own // 256) * 256
    for gk, gv in ((P, None), (None, P), (ODD, P)):
        assert run(P, gk, gv, full) == -1 and b"grad_k" in _err()
    assert run(None, None, None, full) == -1 and b"grad_q" in _err()
    assert run(P, P, P, full - 1) == -1 and b"workspace" in _err()
    assert run(P, None, None, own - 1) == -1 and b"workspace" in _err()
    # no queries: nothing to do
    none = _args(q=0, rows_q=0, rows_k=600, cu_q=0, B=1, cu_k=0)
    assert lib.mhc_attention_bwd(none, None, st, None, None, None, None, None, None, 0, None) == 0


@pytest.mark.gpu
def test_opcheck_without_the_keys_gradients():
    g = _gen(1)
    r = lambda *s: torch.randn(*s, device=DEV, generator=g).to(torch.bfloat16)
    q, k, v = r(9, 4, 64), r(9, 2, 64), r(9, 2, 64)
    out, lse = OPS.attention(q, k, v)
    torch.library.opcheck(OPS.attention_backward.default, (r(9, 4, 64), q, k, v, out, lse, None, None, None, True, None, False))


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["fn", "op", "compiled"])
@pytest.mark.parametrize("trained", [(0,), (1,), (2,), (0, 1), (0, 1, 2)])
@pytest.mark.parametrize("T,d", [(70, 64), (1500, 128), (300, 33)])
def test_frozen(form, trained, T, d, monkeypatch):
    """The gradients that are wanted equal those of a call that wants them all; the keys' kernels run
    where one of theirs is wanted."""
    g = _gen(T)
    r = lambda n: torch.randn(T, n, d, device=DEV, generator=g).to(torch.bfloat16)
    args, go = (r(4), r(2), r(2)), r(4)
    cu = torch.tensor([0, T // 3, T], dtype=torch.int32, device=DEV)
    want = S.attention_backward(go, *args, *(lambda f: (f["out"], f["lse"]))(S.attention(*args, cu, need_backward=True)), cu)
    asked = []

    def spy(*a, _run=S.attention_backward, **k):
        out = _run(*a, **k)
        asked.append([t is not None for t in out])
        return out

    for m in ("attention", "library"):
        monkeypatch.setattr(sys.modules[f"FlagOS_mhc.{m}"], "attention_backward", spy)
    fn = S.attention_fn if form == "fn" else L.attention_op
    if form == "compiled":
        torch._dynamo.reset()
        fn = torch.compile(fn, backend="aot_eager", fullgraph=True)
    leaves = [t.clone().requires_grad_(i in trained) for i, t in enumerate(args)]
    fn(*leaves, cu).backward(go)
    assert asked == [[True] + [bool({1, 2} & set(trained))] * 2]
    for i, (t, w) in enumerate(zip(leaves, want)):
        assert torch.equal(t.grad, w) if i in trained else t.grad is None, i


@pytest.mark.gpu
def test_a_frozen_cache_takes_no_memory():
    """One trained query over a cache of 0.4 GB: the backward allocates the query's gradient and D alone."""
    g = _gen(5)
    cache = torch.randn(1, 100_000, 2, 8, 128, device=DEV, generator=g).to(torch.bfloat16)
    q = torch.randn(1, 4, 32, 128, device=DEV, generator=g).to(torch.bfloat16).requires_grad_(True)
    out = S.attention_fn(q, cache[:, :, 0], cache[:, :, 1])
    go = torch.ones_like(out)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out.backward(go)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < 1 << 20
