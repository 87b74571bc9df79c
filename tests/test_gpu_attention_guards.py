"""Starts that are no sequences, every buffer that the kernels write between
marked ones: outputs, lse, gradients, the workspaces (D, partial sums and their
maxima) and rotary's outputs.  Starts that become sequences within the buffer
give those sequences' results."""

from __future__ import annotations

import pytest
import torch

from FlagOS_mhc import _lib, sublayer as S
from FlagOS_mhc.attention import _Call, _STRIDES
from FlagOS_mhc.rotary import _ARGS as _ROTARY
from test_gpu_attention_starts import DEV, STARTS, T

pytestmark = pytest.mark.gpu
GUARD, MARK = 1 << 18, 0x5A  # bytes on either side


class Guarded:
    """Buffers with marked bytes before and behind them."""

    def __init__(self):
        self.all = []

    def __call__(self, shape, dtype):
        n = torch.Size(shape).numel() * dtype.itemsize
        buf = torch.full((n + 2 * GUARD,), MARK, dtype=torch.uint8, device=DEV)
        buf[GUARD:GUARD + n] = 0
        self.all.append((buf, n))
        return buf[GUARD:GUARD + n].view(dtype).view(shape)

    def check(self):
        torch.cuda.synchronize()
        for i, (buf, n) in enumerate(self.all):
            assert bool((buf[:GUARD] == MARK).all()) and bool((buf[GUARD + n:] == MARK).all()), i


def _attention(q, k, v, go, cu_q, cu_k):
    """Forward and backward through the C entry points."""
    lib, new = _lib.load(), Guarded()
    c = _Call("attention", q, k, v, cu_q, cu_k, None, True, None)
    out, lse = new(q.shape, q.dtype), new((c.H, c.rows_q), torch.float32)
    need = lib.mhc_attention_fwd_workspace_size(c.args)
    ws = new((need,), torch.uint8)
    _lib.call("attention", lib.mhc_attention_fwd, 0, c.args, out.data_ptr(), lse.data_ptr(), ws.data_ptr(), need)
    grads = [new(t.shape, t.dtype) for t in (q, k, v)]
    n = lib.mhc_attention_bwd_workspace_size(c.args)
    ws = new((n,), torch.uint8)
    row = q.shape[1] * q.shape[2]
    _lib.call("attention_backward", lib.mhc_attention_bwd, 0, c.args, go.data_ptr(), _STRIDES.pack(0, row, q.shape[2]), out.data_ptr(),
              lse.data_ptr(), *(t.data_ptr() for t in grads), ws.data_ptr(), n)
    new.check()
    return need, [out, lse, *grads]


# rows of q and of k, H: tiles of 32 rows; waves that share keys; blocks of 128; parts of the keys, which need a workspace
@pytest.mark.parametrize("rows,rows_k,H,parts", [(T, T, 4, False), (T, T, 32, False), (T, T, 64, False), (40, 16 * T, 4, True)])
@pytest.mark.parametrize("name", STARTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_attention(name, rows, rows_k, H, parts, dtype):
    print(f"[attention guards] {name} {rows} {H} {dtype}", flush=True)
    g = torch.Generator(device=DEV)
    g.manual_seed(rows + H)
    q, go = (torch.randn(rows, H, 64, device=DEV, generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(rows_k, 2, 64, device=DEV, generator=g).to(dtype) for _ in range(2))
    starts = torch.tensor(STARTS[name], dtype=torch.int64)
    bad = lambda n: (starts * n // T).clamp(-(1 << 31), (1 << 31) - 1).to(device=DEV, dtype=torch.int32)
    good = lambda n: torch.linspace(0, n, starts.numel()).int().to(DEV)
    for cq, ck in ((bad(rows), bad(rows_k)), (bad(rows), good(rows_k)), (good(rows), bad(rows_k))):
        need, _ = _attention(q, k, v, go, cq, ck)
    if starts.numel() < 8:  # (few sequences)
        assert (need > 0) == parts


# .. that are sequences once they are kept within the buffer (the first one is taken as 0)
INSIDE = {"first_not_zero": [600, 700, 800, 1000], "below_zero": [0, -5, 400, 1000], "past_the_end": [0, 300, 2147483647, 1001]}


@pytest.mark.parametrize("name", INSIDE)
@pytest.mark.parametrize("H", [4, 64])
def test_attention_within_the_buffer(name, H):
    g = torch.Generator(device=DEV)
    g.manual_seed(H)
    q, go = (torch.randn(T, H, 64, device=DEV, generator=g).bfloat16() for _ in range(2))
    k, v = (torch.randn(T, 2, 64, device=DEV, generator=g).bfloat16() for _ in range(2))
    cu = torch.tensor(INSIDE[name], dtype=torch.int32, device=DEV)
    kept = cu.clamp(0, T)
    kept[0] = 0
    _, got = _attention(q, k, v, go, cu, cu)
    _, want = _attention(q, k, v, go, kept, kept)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", [*STARTS, *(n + "_kept" for n in INSIDE)])
@pytest.mark.parametrize("dtype,code", [(torch.bfloat16, 1), (torch.float32, 0)])
def test_rotary(name, dtype, code):
    g = torch.Generator(device=DEV)
    g.manual_seed(7)
    q, k = (torch.randn(T, n, 64, device=DEV, generator=g).to(dtype) for n in (4, 2))
    freqs, _ = S.rotary_frequencies(64)
    kept = name.endswith("_kept")
    cu = torch.tensor(INSIDE[name[:-5]] if kept else STARTS[name], dtype=torch.int32, device=DEV)
    new = Guarded()
    qo, ko = new(q.shape, dtype), new(k.shape, dtype)
    _lib.call("rotary", _lib.load().mhc_rotary, 0,
              _ROTARY.pack(q.data_ptr(), k.data_ptr(), qo.data_ptr(), ko.data_ptr(), freqs.data_ptr(), 0, cu.data_ptr(), 256, 64, 128,
                           64, T, 1, 1.0, cu.numel() - 1, code, 4, 2, 64, 64, 0, 0))
    new.check()
    # every row is turned by some whole angle: lengths of pairs stay
    for x, y in ((q, qo), (k, ko)):
        size = lambda t: t.double().view(T, -1, 2, 32).square().sum(2).sqrt()
        assert float((size(y) - size(x)).abs().max()) <= 2 * torch.finfo(dtype).eps * float(size(x).max())
    if kept:
        c = cu.clamp(0, T).long()
        c[0] = 0
        at = torch.arange(T, device=DEV)
        first = c[torch.searchsorted(c, at, right=True) - 1]
        want = S.rotary(q, k, freqs, at - first)
        assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])
