"""ctypes binding of libmhc_amd.so, the gfx950 HIP kernels behind the ops.

The entry points and their arguments are declared in ``include/mhc_amd.h``.
There is deliberately no fallback: if the library is missing or the tensors
are not on a HIP device, the operators raise instead of computing on the CPU.
"""

from __future__ import annotations

import collections
import contextlib
import ctypes
import functools
import math
import os
import threading

import torch
from torch.autograd import forward_ad

_LIB_NAME = "libmhc_amd.so"
_LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), _LIB_NAME)

DTYPE_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
PRE_BWD_COMPENSATED = 1  # mhc_pre_bwd_ex flags (include/mhc_amd.h)
PRE_BWD_TWO_PASS = 2
PRE_BWD_SINGLE_PASS = 4

_c = ctypes
_vp, _i32, _i64, _f32, _sz = _c.c_void_p, _c.c_int32, _c.c_int64, _c.c_float, _c.c_size_t

_SIGNATURES = {
    "mhc_last_error": (_c.c_char_p, []),
    "mhc_version": (_i32, []),
    "mhc_post_fwd": (_c.c_int, [_vp, _vp, _vp, _vp, _vp, _i64, _i32, _i32, _i32, _vp]),
    "mhc_post_bwd": (_c.c_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
                                _i64, _i32, _i32, _i32, _vp]),
    "mhc_post_bwd_sum": (_c.c_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
                                    _i64, _i32, _i32, _i32, _vp]),
    "mhc_post_bwd_sum_fused": (_c.c_int, [_i64, _i32, _i32, _i32]),
    "mhc_pre_fwd_workspace_size": (_sz, [_i64, _i32, _i32, _i32]),
    "mhc_pre_fwd": (_c.c_int, [_vp, _i32, _vp, _i32, _vp, _vp, _f32, _f32, _f32, _f32, _i32,
                               _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz,
                               _i64, _i32, _i32, _vp]),
    "mhc_pre_fwd_ex": (_c.c_int, [_vp, _i32, _vp, _i32, _vp, _vp, _f32, _f32, _f32, _f32, _i32,
                                  _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _vp,
                                  _i64, _i32, _i32, _vp]),
    "mhc_debug_set_wait_limit": (None, [_i64]),
    "mhc_pre_fwd_noalloc": (_c.c_int, [_vp, _i32, _vp, _i32, _vp, _vp, _f32, _f32, _f32, _f32, _i32,
                                       _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i32, _i32, _vp]),
    "mhc_pre_bwd_acc": (_c.c_int, [_vp, _i32, _vp, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
                                   _f32, _f32, _f32, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _sz,
                                   _i64, _i32, _i32, _vp]),
    "mhc_pre_bwd_ex": (_c.c_int, [_vp, _i32, _vp, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
                                  _f32, _f32, _f32, _i32, _vp, _vp, _vp, _vp, _vp, _c.c_uint32, _vp,
                                  _vp, _sz, _i64, _i32, _i32, _vp]),
    "mhc_post_pre_fwd_workspace_size": (_sz, [_i64, _i32, _i32, _i32]),
    "mhc_post_pre_fwd": (_c.c_int, [_vp, _vp, _vp, _vp, _i32, _vp, _i32, _vp, _vp, _f32, _f32, _f32,
                                    _f32, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz,
                                    _i64, _i32, _i32, _vp]),
    "mhc_post_pre_fwd_ex": (_c.c_int, [_vp, _vp, _vp, _vp, _i32, _vp, _i32, _vp, _vp, _f32, _f32, _f32,
                                       _f32, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _vp,
                                       _i64, _i32, _i32, _vp]),
    "mhc_pre_bwd_workspace_size": (_sz, [_i64, _i32, _i32, _i32, _i32]),
    "mhc_pre_bwd": (_c.c_int, [_vp, _i32, _vp, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
                               _f32, _f32, _f32, _i32, _vp, _vp, _vp, _vp, _vp, _sz,
                               _i64, _i32, _i32, _vp]),
    "mhc_layer_norm_fwd": (_c.c_int, [_vp, _i32, _vp, _vp, _i32, _f32, _vp, _vp, _vp, _i64, _i32, _vp]),
    "mhc_layer_norm_bwd_workspace_size": (_sz, [_i64, _i32, _i32]),
    "mhc_layer_norm_bwd": (_c.c_int, [_vp, _vp, _i32, _vp, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _sz,
                                      _i64, _i32, _vp]),
    "mhc_gated_ffn_fwd_workspace_size": (_sz, [_i64, _i32, _i32, _i32, _i32]),
    "mhc_gated_ffn_fwd_save_workspace_size": (_sz, [_i64, _i32, _i32, _i32, _i32]),
    "mhc_gated_ffn_fwd": (_c.c_int, [_vp, _vp, _vp, _vp, _i32, _i32, _vp, _vp, _vp, _vp, _vp, _sz,
                                     _i64, _i32, _i32, _i32, _vp]),
    "mhc_gated_ffn_bwd_workspace_size": (_sz, [_i64, _i32, _i32, _i32, _i32]),
    "mhc_gated_ffn_bwd": (_c.c_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i32, _i32, _vp, _vp, _vp,
                                     _vp, _vp, _sz, _i64, _i32, _i32, _i32, _vp]),
    "mhc_dropout": (_c.c_int, [_vp, _vp, _i64, _i32, _c.c_double, _c.c_uint64, _c.c_uint64, _vp, _vp]),
}

EXPORTED = tuple(_SIGNATURES)

_lock = threading.Lock()
_lib = None


def lib_path() -> str:
    return _LIB_PATH


def load() -> ctypes.CDLL:
    """Load (once) and return the library; raise if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(_LIB_PATH):
                raise RuntimeError(
                    f"{_LIB_NAME} not found at {_LIB_PATH}; build it with "
                    "`python flagos-mhc_amd/build.py` (hipcc, gfx950). The mHC operators "
                    "have no CPU fallback.")
            lib = ctypes.CDLL(_LIB_PATH)
            for name, (res, args) in _SIGNATURES.items():
                fn = getattr(lib, name)
                fn.restype = res
                fn.argtypes = args
            _lib = lib
    return _lib


def check(rc: int, what: str) -> None:
    if rc != 0:
        msg = load().mhc_last_error().decode(errors="replace")
        if rc == -2:
            raise NotImplementedError(f"{what}: {msg}")
        raise RuntimeError(f"{what} failed ({rc}): {msg}")


def ptr(t):
    return None if t is None else t.data_ptr()


def stream_of(t: torch.Tensor):
    """The current HIP stream of t's device."""
    return torch._C._cuda_getCurrentRawStream(t.device.index)


_no_guard = contextlib.nullcontext()


def on_device(dev: torch.device):
    """A context in which `dev` is the current device (none is entered where it
    is already: switching costs a call more than a few microseconds)."""
    return _no_guard if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def call(what: str, fn, dev_index: int, *args) -> None:
    """fn(*args, current stream) on the device `dev_index`, checked.  (Host time
    is what small calls cost: nothing is done here that they do not need.)"""
    if torch._C._cuda_getDevice() == dev_index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev_index))
    else:
        with torch.cuda.device(dev_index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev_index))
    if rc:
        check(rc, what)


def operand(t: torch.Tensor, shape, dtype: torch.dtype) -> torch.Tensor:
    """t as a contiguous tensor of `dtype` with shape's elements in order (the
    kernels take its address only, so a tensor that already holds them is
    returned as it is, whatever its own shape)."""
    if t.dtype == dtype and t.is_contiguous() and t.numel() == math.prod(shape):
        return t
    return t.reshape(shape).to(dtype).contiguous()


@functools.lru_cache(maxsize=1024)
def workspace_size(name: str, dev_index: int, *args) -> int:
    """A *_workspace_size query: a function of the sizes and the device alone."""
    with torch.cuda.device(dev_index):
        return int(getattr(load(), name)(*args))


def workspace(name: str, dev: torch.device, *args):
    """(tensor, bytes) of scratch for a call on `dev`."""
    n = workspace_size(name, dev.index, *args)
    return torch.empty(n or 1, dtype=torch.uint8, device=dev), n


def pre_fwd_size_code(x_code: int, phi_code: int, addresses: int) -> int:
    """The phi dtype code to ask mhc_pre_fwd_workspace_size with: bf16 x and phi
    at 16-byte aligned addresses (or-ed together here) have kernels of their
    own, any other pair runs the general form, whose workspace is that of an
    fp32 phi (code 0)."""
    return phi_code if x_code == 1 and not addresses & 15 else 0


def require_device(what: str, *tensors) -> None:
    """Every tensor given is on one HIP device (kernels take addresses: one of
    another GPU would be read there)."""
    first = -1
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(
                f"{what}: expected tensors on a HIP (cuda) device, got {t.device}; "
                "the MI355X operators have no CPU path (use the *_ref functions on CPU)")
        index = t.get_device()
        if index != first:
            if first >= 0:
                raise ValueError(f"{what}: tensors on cuda:{first} and {t.device}, expected one device")
            first = index


def has_tangent(*tensors) -> bool:
    """Whether a tensor carries a forward-mode derivative (which requires_grad
    does not tell; the level is looked at first, as no program that runs none
    should pay for asking)."""
    return forward_ad._current_level >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def needs_autograd(*tensors) -> bool:
    """Whether an operator has to go through its autograd.Function: a gradient
    may be taken, or there is a tangent, which the Function refuses."""
    return (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)) or has_tangent(*tensors)


class _NoSecondDerivative(torch.autograd.Function):
    """Hands on the first n of its tensors; its own backward is an error."""

    @staticmethod
    def forward(ctx, what, n, *tensors):
        ctx.what = what
        return tuple(t.view_as(t) for t in tensors[:n])

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.what}: second derivatives are not implemented")


def first_order(what: str, grads, *inputs):
    """grads (None among them), computed from `inputs` by kernels: where a graph
    of the backward is asked for (create_graph), one that fails when it is
    differentiated, instead of none.  (torch's once_differentiable leaves it out
    where the output's gradient needs none, though the saved inputs do.)"""
    if not torch.is_grad_enabled():
        return grads
    have = [g for g in grads if g is not None]
    wrapped = iter(_NoSecondDerivative.apply(what, len(have), *have, *inputs))
    return tuple(None if g is None else next(wrapped) for g in grads)


def dtype_code(what: str, dt: torch.dtype) -> int:
    try:
        return DTYPE_CODE[dt]
    except KeyError:
        raise NotImplementedError(f"{what}: dtype {dt} not supported (float32, bfloat16, float16)")


class SinglePassStatus:
    """Where the single-pass pre forward and backward report their bounded waits.

    Those kernels wait for the other CUs of their group with a limit (0.25 s
    without progress); if a wait gives up, the call's outputs are NaN and the
    kernels write a failure code to the status word of ``mhc_pre_fwd_ex`` /
    ``mhc_pre_bwd_ex``.
    Each call gets a word in a ring of pinned host memory (written by the GPU
    with a system-scope store, read by the host once the call's event has
    completed), so no call waits for the GPU.  ``check`` raises for a failed
    call: without blocking at the start of every operator call (calls whose
    work has finished), blocking in the pre backward and in
    ``FlagOS_mhc.check_errors``."""

    # enough that a caller enqueueing far ahead of the GPU never waits for a
    # word (16 KB of pinned memory)
    SLOTS = 4096

    def __init__(self):
        self._lock = threading.RLock()
        self._words = None
        self._busy = [False] * self.SLOTS
        self._next = 0
        self._pending = collections.deque()  # (slot, event), oldest first

    def acquire(self):
        """A zeroed word for the next call: (slot, its address).  A word is
        reused only after the call that reported into it was checked."""
        with self._lock:
            if self._words is None:
                self._words = torch.zeros(self.SLOTS, dtype=torch.int32, pin_memory=True)
            while self._busy[self._next]:
                self.check(block=True)
            slot = self._next
            self._next = (slot + 1) % self.SLOTS
            self._words[slot] = 0
            return slot, self._words.data_ptr() + 4 * slot

    def commit(self, slot, stream) -> None:
        """The call that got `slot` was enqueued on `stream`."""
        ev = torch.cuda.Event()
        ev.record(stream)
        with self._lock:
            self._busy[slot] = True
            self._pending.append((slot, ev))

    def check(self, block: bool) -> None:
        if not self._pending:  # nothing reported since the last check
            return
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            return
        with self._lock:
            while self._pending:
                slot, ev = self._pending[0]
                if not block and not ev.query():
                    return
                ev.synchronize()
                self._pending.popleft()
                self._busy[slot] = False
                code = int(self._words[slot])
                if code:
                    raise RuntimeError(
                        f"mhc_pre_clamp_sinkhorn: an earlier single-pass forward or backward call gave "
                        f"up a bounded wait for the other CUs of its group (status {code}: the GPU "
                        "stalled longer than the wait limit); that call's outputs are NaN")


SINGLE_PASS = SinglePassStatus()


def check_errors(block: bool = True) -> None:
    """Raise RuntimeError if an earlier single-pass pre forward or backward
    gave up a bounded wait (its outputs are then NaN).  With ``block`` (the default)
    wait for every such call's work to finish first; without it, look only
    at calls that have finished."""
    SINGLE_PASS.check(block)
