"""Sizes past which the sublayer kernels' 32-bit counts would wrap: refused at
the C entry points, before anything is launched (no GPU)."""

from __future__ import annotations

import ctypes

import pytest

from FlagOS_mhc import _lib

P = ctypes.c_void_p(0x1000)
MAX_ROW = (1 << 30) - 512


@pytest.mark.parametrize("D", [MAX_ROW + 1, 1 << 30, (1 << 31) - 1024, (1 << 31) - 1])
def test_layer_norm_rows_that_wrap_are_refused(D):
    """The loop over a row's 2 D sums goes on by 1024 after the last one below 2 D."""
    assert 2 * D + 1024 > 1 << 31
    lib = _lib.load()
    assert lib.mhc_layer_norm_fwd(P, 1, P, P, 0, 1e-5, P, None, None, 1, D, None) == -2
    assert b"above the supported" in lib.mhc_last_error()
    assert lib.mhc_layer_norm_bwd(P, P, 1, P, 0, P, P, P, P, P, P, 1 << 40, 1, D, None) == -2
    assert lib.mhc_layer_norm_bwd_workspace_size(1, D, 1) == 0


def test_layer_norm_longest_rows_are_taken():
    lib = _lib.load()
    assert 2 * MAX_ROW - 1 + 1024 < 1 << 31  # the last count of that loop, and its step past it
    assert lib.mhc_layer_norm_bwd_workspace_size(1, MAX_ROW, 1) == 8 * MAX_ROW
    # past the size checks: the workspace is what is missed
    assert lib.mhc_layer_norm_bwd(P, P, 1, P, 0, P, P, P, P, P, None, 0, 1, MAX_ROW, None) == -1
    assert b"workspace" in lib.mhc_last_error()


@pytest.mark.parametrize("which", ["T", "D", "F", "O"])
@pytest.mark.parametrize("size", [(1 << 31) - 255, (1 << 31) - 1])
def test_gated_ffn_sizes_that_wrap_are_refused(which, size):
    """A size is rounded up to a tile's 256 rows in 32 bits."""
    assert size + 255 > (1 << 31) - 1
    lib = _lib.load()
    n = {"T": 1, "D": 1, "F": 1, "O": 1, which: size}
    dims = [n[k] for k in "TDFO"]
    assert lib.mhc_gated_ffn_fwd(P, P, P, P, 1, 0, P, None, None, None, P, 1 << 60, *dims, None) == -2
    assert b"above the supported" in lib.mhc_last_error()
    assert lib.mhc_gated_ffn_bwd(P, P, P, P, P, P, P, P, 1, 0, P, P, P, P, P, 1 << 60, *dims, None) == -2
    assert b"above the supported" in lib.mhc_last_error()
    assert lib.mhc_gated_ffn_fwd_workspace_size(*dims, 1) == lib.mhc_gated_ffn_bwd_workspace_size(*dims, 1) == 0


def test_gated_ffn_largest_sizes_are_taken():
    lib = _lib.load()
    size = (1 << 31) - 256
    assert size + 255 == (1 << 31) - 1
    # past the size checks: the workspace is what is missed
    assert lib.mhc_gated_ffn_fwd(P, P, P, P, 1, 0, P, None, None, None, None, 0, 1, size, 1, 1, None) == -1
    assert b"workspace" in lib.mhc_last_error()
