"""Per-device native engine handles (side stream, workspace, staging ring).

One `helm_engine` per HIP device, created on first use and destroyed at
interpreter exit.  The engine's side stream is what HELM's per-device
``_get_kv_copy_stream`` (helm/runtime/kv_cache.py:383-391) memoizes.
"""
from __future__ import annotations

import atexit
import ctypes
import os
from typing import Dict

import torch
from torch.autograd import forward_ad as _forward_ad

from helm_amd import _native

_engines: Dict[int, ctypes.c_void_p] = {}
_copy_streams: Dict[int, torch.cuda.ExternalStream] = {}


def device_index(device: torch.device) -> int:
    if device.type != "cuda":
        raise ValueError(f"expected a HIP device, got {device}")
    return device.index if device.index is not None else torch.cuda.current_device()


def get_engine(device: torch.device) -> ctypes.c_void_p:
    idx = device.index if device.index is not None else device_index(device)
    eng = _engines.get(idx)
    if eng is None:
        _native.load()
        chunk = int(os.environ.get("HELM_AMD_CHUNK_MB", "64")) << 20
        slots = int(os.environ.get("HELM_AMD_RING_SLOTS", "2"))
        handle = ctypes.c_void_p()
        with torch.cuda.device(idx):
            _native.call("helm_engine_create", idx, chunk, slots, ctypes.byref(handle))
        _engines[idx] = eng = handle
    return eng


def copy_stream(device: torch.device) -> torch.cuda.ExternalStream:
    """The engine's side stream as a torch stream object (memoized per device)."""
    idx = device_index(device)
    s = _copy_streams.get(idx)
    if s is None:
        ptr = _native.load().helm_engine_copy_stream(get_engine(device))
        s = torch.cuda.ExternalStream(ptr, device=torch.device("cuda", idx))
        _copy_streams[idx] = s
    return s


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_ptr(device: torch.device) -> int:
    """hipStream_t of torch's current stream on `device` (torch's raw-stream
    query where this torch has it: no Stream object per call)."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    if _raw_stream is not None:
        return _raw_stream(idx)
    return torch.cuda.current_stream(idx).cuda_stream


_get_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def launch_on(idx: int, fn: str, *args) -> int:
    """One native call that launches on HIP device `idx`, on torch's current stream
    there (its last argument, returned): the device is current for it (and the one before
    is again afterwards); raises as ``_native.call`` does."""
    f = _native.entry(fn)
    stream = _raw_stream(idx) if _raw_stream is not None else \
        torch.cuda.current_stream(idx).cuda_stream
    if idx == _get_device():
        rc = f(*args, stream)
    else:
        with torch.cuda.device(idx):
            rc = f(*args, stream)
    if rc:
        _native.check(fn, rc)
    return stream


def common_device(what: str, *tensors: torch.Tensor) -> int:
    """The index of the one HIP device that a call's operands sit on."""
    idx = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != idx:
            raise ValueError(f"{what}: operands on {tensors[0].device} and {t.device}")
    if idx < 0:
        raise RuntimeError(f"{what} needs HIP tensors")
    return idx


def refuse_overlap(what: str, out: torch.Tensor, *inputs: torch.Tensor) -> None:
    """Refuses a contiguous `out` that shares memory with an operand (other workgroups
    may still be reading it).  The first of them may be `out` itself: a workgroup
    reads its own rows of it and then writes them."""
    lo = out.data_ptr()
    hi = lo + out.numel() * out.element_size()
    for i, t in enumerate(inputs):
        at = t.data_ptr()
        if at >= hi or lo == hi or not t.numel() or (i == 0 and at == lo and t.is_contiguous()):
            continue
        span = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1
        if at + span * t.element_size() > lo:
            raise ValueError(f"{what}: out lies over another operand (only q itself may be out)")


def refuse_grad(what: str, *tensors: torch.Tensor) -> None:
    """The package serves models: its attention records nothing for a backward pass, and
    has no tangent to give (which no_grad does not drop)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise RuntimeError(f"{what} records no gradient: call it under torch.no_grad()")
    if _forward_ad._current_level >= 0:
        for t in tensors:
            if _forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what} gives no forward-mode tangent: unpack its operands")


@atexit.register
def _destroy_engines() -> None:
    if not _engines:
        return
    lib = _native.load()
    for eng in _engines.values():
        lib.helm_engine_destroy(eng)
    _engines.clear()
    _copy_streams.clear()
