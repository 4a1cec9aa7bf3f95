"""Glue between torch tensors and the exported C launchers of ``csrc``.

Every launcher takes raw device pointers, sizes and the CUDA stream and returns an int: 0 on
success, a positive ``cudaError_t`` if the launch failed, a negative code if it refused its
arguments.  Nothing here falls back to another implementation: a tensor that is not on a CUDA
device, a failed build or a refused size raises.
"""
from __future__ import annotations

import ctypes
import struct
import threading
from typing import Any

import torch

from ..csrc import build

_REFUSALS = {-1: "bad argument", -2: "unsupported size", -3: "scratch too small", -4: "set-up failed"}


class KernelError(RuntimeError):
    """A launcher refused its arguments or the launch failed."""


def ptr(tensor: torch.Tensor | None) -> ctypes.c_void_p:
    if tensor is None:
        return ctypes.c_void_p(0)
    return ctypes.c_void_p(tensor.data_ptr())


class _Bound(threading.local):
    stream = None  # the one that a step of this thread has bound for its launches


_bound = _Bound()


def stream_ptr() -> ctypes.c_void_p:
    """The stream launches go to: the one bound by ``stream_bound`` if any, else torch's current stream."""
    bound = _bound.stream
    return bound if bound is not None else ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


class stream_bound:
    """``with stream_bound():`` looks torch's current stream up once; the launches that this thread makes inside use it without asking again.
    Nesting rebinds (a graph capture inside a step launches on the capture's stream)."""

    def __enter__(self):
        self.previous = _bound.stream
        _bound.stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        return self

    def __exit__(self, *exc):
        _bound.stream = self.previous
        return False


def require_cuda(*tensors: torch.Tensor | None) -> None:
    for tensor in tensors:
        if tensor is not None and not tensor.is_cuda:
            raise KernelError("the kernels run on a CUDA device only; got a tensor on " + str(tensor.device))


_sm_counts: dict = {}


def sm_count(device=None) -> int:
    """Multiprocessors of the device (the current one by default), asked once per device: grids and split counts follow it."""
    index = None if device is None else (device if isinstance(device, torch.device) else torch.device(device)).index
    if index is None:
        index = torch.cuda.current_device()
    found = _sm_counts.get(index)
    if found is None:
        found = _sm_counts[index] = int(torch.cuda.get_device_properties(index).multi_processor_count)
    return found


LAUNCHES = [0]  # launcher calls that succeeded, for reports of how much of a step is this package's own code


def check(code: int, what: str) -> None:
    if code == 0:
        LAUNCHES[0] += 1
        return
    if code < 0:
        raise KernelError(f"{what}: launcher refused its arguments ({_REFUSALS.get(code, code)})")
    raise KernelError(f"{what}: CUDA error {code} at launch")


def is_bf16(tensor: torch.Tensor) -> int:
    if tensor.dtype == torch.bfloat16:
        return 1
    if tensor.dtype == torch.float32:
        return 0
    raise KernelError(f"unsupported element type {tensor.dtype} (float32 and bfloat16 only)")


_libraries: dict = {}


def library(module: str, **defines: Any) -> ctypes.CDLL:
    key = (module, tuple(sorted(defines.items()))) if defines else module
    found = _libraries.get(key)
    if found is None:
        found = _libraries[key] = build.load(module, defines)
    return found


_KINDS = {"p": ctypes.c_void_p, "i": ctypes.c_int, "l": ctypes.c_longlong, "f": ctypes.c_float}
_entries: dict = {}


def entry(module: str, name: str, arguments: str, head_dim: int = 0, result: str = "i", packed: bool = False):
    """An exported launcher with its arguments' and its result's kinds (p: address, i: int, l: long long, f: float), looked up once: plain Python numbers then go to it as they are,
    which costs a call of twenty arguments a few microseconds less than a ctypes object for each.  ``packed``: they go to ``name`` + "_packed" as one structure, which costs it 0.5 us in place of 2."""
    found = _entries.get((name, head_dim))
    if found is None:
        loaded, kinds = library(module, HB_HEAD_DIM=head_dim) if head_dim else library(module), [_KINDS[kind] for kind in arguments]
        if packed:
            found = _packed(getattr(loaded, name + "_packed"), struct.Struct("@" + "".join(_FORMATS[kind] for kind in arguments)).pack, name)
        else:
            found = getattr(loaded, name)
            found.restype = _KINDS[result]
        found.argtypes = kinds  # of a packed one, too: those of its launcher
        _entries[name, head_dim] = found
    return found


_FORMATS = {"p": "P", "i": "i", "l": "q", "f": "f"}


def _packed(function, pack, name: str):
    function.argtypes, function.restype = [ctypes.c_char_p], ctypes.c_int

    def call(*values):
        try:
            return function(pack(*values))
        except struct.error as error:
            raise KernelError(f"{name}: {error}") from None

    return call


def stream_address() -> int:
    """:func:`stream_ptr` as a number, without the objects on the way there."""
    bound = _bound.stream
    return (bound.value or 0) if bound is not None else torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


class _Scratch(threading.local):
    def __init__(self):
        self.kept: dict = {}


_scratch = _Scratch()
KEPT_SCRATCH = 16 << 20  # bytes; above it a tensor of its own costs nothing beside the work that wants it


def scratch(device: torch.device, stream: int, size: int):
    """(address, owner) of ``size`` bytes on a boundary of 512 for one call's launches on ``stream``: launches of one stream follow one another, so a thread keeps one piece of
    memory per stream for all of them (another thread's may come between two launches of one call).  The caller holds the owner until its launches are under way.  A graph
    that is being captured gets memory of its own (its replays may run beside other work of that stream), and so do large wishes."""
    if size > KEPT_SCRATCH or torch._C._cuda_isCurrentStreamCapturing():
        owner = torch.empty(max(1, size), dtype=torch.uint8, device=device)
        return owner.data_ptr(), owner
    kept = _scratch.kept
    found = kept.get((device.index, stream))
    if found is None or found[2] < size:
        room = max(1 << 16, 1 << (size - 1).bit_length()) if size else 1 << 16
        owner = torch.empty(room, dtype=torch.uint8, device=device)
        found = kept[device.index, stream] = (owner.data_ptr(), owner, room)
    return found[0], found[1]


i32 = int  # a Python int is passed as a C int by ctypes itself; the name marks which arguments are 32-bit


def f32(value: float) -> ctypes.c_float:
    return ctypes.c_float(float(value))
