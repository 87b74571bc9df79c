"""Arguments of attention and rotary positions that are refused, or taken, at
the edges of what is documented (no GPU: nothing is launched)."""

from __future__ import annotations

import pytest
import torch

from FlagOS_mhc import _lib, sublayer as S
from FlagOS_mhc.attention import _STRIDES
from test_attention_cpu import P, _args, _err, on_cpu, t  # noqa: F401 (on_cpu is a fixture)

LIMIT = 2.3586e38  # the largest fp32 number by log2(e)


def _c_calls(a):
    """Return codes of the C entry points."""
    lib, st = _lib.load(), _STRIDES.pack(0, 128, 64)
    yield lib.mhc_attention_fwd(a, P, None, P, 1 << 40, None)
    yield lib.mhc_attention_bwd(a, P, st, P, P, P, P, P, P, 1 << 40, None)


@pytest.mark.parametrize("scale", [LIMIT * 1.001, 2.4e38, 3e38])
def test_scale_times_log2e_is_a_number(on_cpu, scale):  # noqa: F811
    a = _args(scale=scale)
    for rc in _c_calls(a):
        assert rc == -1 and b"scale" in _err()
    assert _lib.load().mhc_attention_bwd_workspace_size(a) == 0
    q, k = t(6, 4, 64), t(6, 2, 64)
    with pytest.raises(ValueError, match="scale"):
        S.attention(q, k, k, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        S.attention_backward(q, q, k, k, q, t(4, 6, dtype=torch.float32), scale=scale)


@pytest.mark.parametrize("scale", [1e-38, 1.0, LIMIT * 0.999])
def test_scales_up_to_the_limit_are_taken(on_cpu, scale):  # noqa: F811
    assert _lib.load().mhc_attention_bwd_workspace_size(_args(scale=scale)) > 0
    q, k = t(6, 4, 64), t(6, 2, 64)
    assert S.attention(q, k, k, scale=scale)["out"].shape == q.shape


def test_reserved_is_zero():
    for word in (1, -1, 1 << 30):
        a = _args()[:-4] + word.to_bytes(4, "little", signed=True)
        assert _lib.load().mhc_attention_fwd_workspace_size(a) == _lib.load().mhc_attention_bwd_workspace_size(a) == 0
        for rc in _c_calls(a):
            assert rc == -1 and b"reserved" in _err()


def test_positions_have_the_rows_order(on_cpu):  # noqa: F811
    """One a row, flat or in the shape of the dimensions before the heads: another shape of as
    many (a transposed one) would be taken in its own order."""
    f, _ = S.rotary_frequencies(64, device="cpu")
    q, k = t(2, 3, 4, 64), t(2, 3, 1, 64)
    for shape in ((3, 2), (3, 1, 2), (1, 3, 2)):
        for call in (S.rotary, S.rotary_backward, S.rotary_fn):
            with pytest.raises(ValueError, match="positions"):
                call(q, k, f, torch.zeros(shape, dtype=torch.int64))
    for shape in ((6,), (6, 1), (2, 3), (1, 2, 3), (2, 3, 1)):
        assert S.rotary(q, k, f, torch.zeros(shape, dtype=torch.int32))[0].shape == q.shape
    assert S.rotary(t(6, 4, 64), None, f, torch.zeros(1, 6, dtype=torch.int32))[0].shape == (6, 4, 64)
    assert S.rotary(t(1, 1, 4, 64), None, f, torch.tensor(7))[0].shape == (1, 1, 4, 64)
