"""A forward that is given hidden (what a training step keeps) needs no second
one in its workspace."""

from __future__ import annotations

import ctypes

import pytest
import torch

from FlagOS_mhc import _lib, sublayer as S
from FlagOS_mhc.gated_ffn import hidden_width

P = ctypes.c_void_p(0x1000)
SIZES = [(1, 64, 128, 64), (40, 333, 1001, 335), (300, 1003, 2677, 1001), (2051, 1024, 2816, 1024)]


@pytest.mark.parametrize("T,D,F,O", SIZES)
@pytest.mark.parametrize("code,size", [(0, 4), (1, 2), (2, 2)])
def test_workspace_is_less_by_hidden(T, D, F, O, code, size):
    lib = _lib.load()
    full = lib.mhc_gated_ffn_fwd_workspace_size(T, D, F, O, code)
    save = lib.mhc_gated_ffn_fwd_save_workspace_size(T, D, F, O, code)
    assert full - save == -(-T * hidden_width(F) * size // 256) * 256
    call = lambda n, h: lib.mhc_gated_ffn_fwd(P, P, P, P, code, 0, P, h, h, h, P, n, T, D, F, O, None)
    assert call(full - 1, None) == -1 and b"workspace" in lib.mhc_last_error()
    if save:
        assert call(save - 1, P) == -1 and b"workspace" in lib.mhc_last_error()
    assert lib.mhc_gated_ffn_fwd_save_workspace_size(0, D, F, O, code) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T,D,F,O", SIZES)
@pytest.mark.parametrize("dtype,code", [(torch.float32, 0), (torch.bfloat16, 1), (torch.float16, 2)])
def test_forward_stays_in_its_workspace(T, D, F, O, dtype, code):
    """Bytes beside the workspace keep their values, and the results are those of
    a forward that keeps nothing."""
    print(f"[gated_ffn workspace] T={T} D={D} F={F} O={O} {dtype}", flush=True)
    lib, dev = _lib.load(), torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(T + F)
    r = lambda *s, scale=1.0: (torch.randn(*s, device=dev, generator=g) * scale).to(dtype)
    x, wg, wu, wd = r(T, D), r(F, D, scale=D ** -0.5), r(F, D, scale=D ** -0.5), r(O, F, scale=F ** -0.5)
    n = lib.mhc_gated_ffn_fwd_save_workspace_size(T, D, F, O, code)
    ws = torch.full((256 + n + 4096,), 0x5A, dtype=torch.uint8, device=dev)
    out = torch.empty(T, O, dtype=dtype, device=dev)
    gate, up = (torch.empty(T, F, device=dev) for _ in range(2))
    hidden = torch.empty(T, hidden_width(F), dtype=dtype, device=dev)
    _lib.call("gated_ffn", lib.mhc_gated_ffn_fwd, dev.index, x.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(),
              code, 0, out.data_ptr(), gate.data_ptr(), up.data_ptr(), hidden.data_ptr(), ws.data_ptr() + 256, n, T, D, F, O)
    torch.cuda.synchronize()
    assert bool((ws[:256] == 0x5A).all()) and bool((ws[256 + n:] == 0x5A).all())
    f = S.gated_ffn(x, wg, wu, wd, need_backward=True)
    assert torch.equal(out, f["out"]) and torch.equal(gate, f["gate"]) and torch.equal(hidden, f["hidden"])
    assert torch.equal(out, S.gated_ffn(x, wg, wu, wd)["out"])


@pytest.mark.gpu
def test_training_forward_allocates_one_hidden():
    T, D, F = 4096, 512, 4096
    r = lambda *s: torch.randn(*s, device="cuda").to(torch.bfloat16)
    x, wg, wu, wd = r(T, D), r(F, D), r(F, D), r(D, F)
    S.gated_ffn(x, wg, wu, wd, need_backward=True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    f = S.gated_ffn(x, wg, wu, wd, need_backward=True)
    peak = torch.cuda.max_memory_allocated() - before
    kept = sum(t.numel() * t.element_size() for t in f.values())
    part = _lib.load().mhc_gated_ffn_fwd_save_workspace_size(T, D, F, D, 1)
    assert peak <= kept + part + 5 * 512  # blocks of 512 bytes
