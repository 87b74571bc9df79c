"""Layer norm over more rows than blocks: each block's walk, its columns' sums
and the sums of the blocks, for every width a thread's registers are cut for;
few rows take the backward's one-launch form.  Bounds: tests/test_gpu_sublayer.py."""

from __future__ import annotations

import pytest
import torch

from FlagOS_mhc import sublayer as S
from test_gpu_sublayer import DT, _check_norm, _gen, _randn

pytestmark = pytest.mark.gpu

MANY = [(9001, 256, "f32"), (9100, 512, "bf16"), (5003, 1003, "f16"), (2600, 1536, "bf16"), (1701, 4000, "bf16"),
        (1603, 7168, "bf16"), (1600, 4096, "f32"), (700, 12001, "bf16"), (300, 20003, "f16")]
FEW = [(1536, 256, "f32"), (1535, 513, "bf16"), (129, 4099, "f16"), (33, 9001, "bf16"), (1000, 9, "f32")]


@pytest.mark.parametrize("T,D,dtype", MANY + FEW)
def test_rows(T, D, dtype):
    print(f"[layer_norm rows] T={T} D={D} {dtype}", flush=True)
    g, dt = _gen(T + D), DT[dtype]
    x = (_randn(g, T, D) * 2 + 0.5).to(dt)
    w, b, gy = _randn(g, D) * 0.2 + 1, _randn(g, D), _randn(g, T, D, dtype=dt)
    first = _check_norm(x, w, b, gy)
    again = _check_norm(x, w, b, gy)
    assert all(torch.equal(p, q) for p, q in zip(first[1:], again[1:]))
    # without the weights' gradients: the same gradient of x
    gx, gw, gb = S.layer_norm_backward(gy, x, w, first[0]["mean"], first[0]["rstd"], need_params=False)
    assert torch.equal(gx, first[1]) and gw is None and gb is None
