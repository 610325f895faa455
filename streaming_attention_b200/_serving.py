"""What the serving entry points share: argument checks, strides, the launch
and the device's error word."""

from __future__ import annotations

import ctypes
import functools
from typing import Optional, Tuple

import torch

from . import _lib
from . import fast as _fast

Tensor = torch.Tensor

DTYPES = {torch.float32: _lib.REP_DTYPES["float32"], torch.float16: _lib.REP_DTYPES["float16"],
          torch.bfloat16: _lib.REP_DTYPES["bfloat16"]}
MAX_DIM = 256


def dtype_code(*ts: Tensor) -> int:
    """The SA_REP_* code of the tensors' one element type."""
    dt = ts[0].dtype
    code = DTYPES.get(dt)
    if code is None:
        raise ValueError(f"unsupported dtype {dt}: float32, float16 and bfloat16 are accepted")
    for t in ts[1:]:
        if t.dtype != dt:
            raise ValueError(f"all inputs must have one dtype, got {dt} and {t.dtype}")
    return code


def device_of(first: Tensor, *others: Tensor) -> torch.device:
    """The CUDA device that all tensors are on."""
    dev = first.device
    index = first.get_device()
    for t in others:
        if t.get_device() != index:
            for x in (first, *others):
                if not x.is_cuda:
                    raise ValueError("the B200 kernels require CUDA tensors")
            raise ValueError("all tensors must be on the same device")
    if dev.type != "cuda":
        raise ValueError("the B200 kernels require CUDA tensors")
    return dev


def int32(t: Tensor, shape: Tuple[int, ...], what: str) -> Tensor:
    """Checks a contiguous int32 index tensor of the given shape."""
    if t.dtype != torch.int32:
        raise ValueError(f"{what} must be int32, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{what} must have shape {list(shape)}, got {list(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def below_2_31(**sizes: int) -> None:
    """Refuses sizes that the C ABI's 32-bit arguments would cut off."""
    for what, n in sizes.items():
        if n >= 1 << 31:
            raise ValueError(f"{what} must be below 2^31, got {n}")


def rows(t: Tensor) -> Tensor:
    """t, or a copy of it, with a contiguous last dimension."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.detach().contiguous()


def repeats(t: Tensor) -> bool:
    """Whether entries of t share memory along an axis (an expanded tensor), so that
    a kernel cannot write them."""
    return any(st == 0 and n > 1 for n, st in zip(t.shape, t.stride()))


_ARRAYS = {n: ctypes.c_int64 * n for n in (3, 4, 8, 12)}


def strides(*values: int):
    return _ARRAYS[len(values)](*values)


def ptr(t: Optional[Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def whole(x, what: str) -> int:
    if type(x) is int:
        return x
    try:
        i = int(x)
    except (TypeError, ValueError, OverflowError):
        i = None
    if i is None or i != x:
        raise ValueError(f"{what} must be a whole number, got {x!r}")
    return i


def check_window(window: Optional[int], sinks: int) -> Tuple[int, int]:
    """Window (0: without end) and first tokens as the C ABI takes them; what lies
    beyond every position (2^31) hides and shows no more than that does."""
    w, s = 0, whole(sinks, "sinks")
    if window is not None:
        w = whole(window, "window")
        if w <= 0:
            raise ValueError("window must be positive, or None for no end")
    if s < 0:
        raise ValueError("sinks must be non-negative")
    return min(w, 1 << 40), min(s, 1 << 40)


@functools.lru_cache(maxsize=1024)
def _workspace_size(name: str, *sizes: int) -> int:
    nbytes = ctypes.c_size_t(0)
    rc = getattr(_lib.load(), name)(*sizes, ctypes.byref(nbytes))
    if rc:
        _lib.check(rc, name)
    return nbytes.value


def workspace(dev: torch.device, name: str, *sizes: int) -> Tensor:
    """Device memory of the size that the entry point `name` asks for."""
    return torch.empty(_workspace_size(name, *sizes), device=dev, dtype=torch.uint8)


def _raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# the current stream's handle without a Stream object around it (2 us a call), where torch has it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)


def launch(dev: torch.device, name: str, *args) -> None:
    """Calls a serving entry point on the current stream of `dev`."""
    index = dev.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return launch(dev, name, *args)
    rc = getattr(_lib.load(), name)(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)
    if _fast._CHECK_STATUS and not torch.cuda.is_current_stream_capturing():
        check_serving_status(dev)


def check_serving_status(device: Optional[torch.device] = None) -> None:
    """Raises for what the serving kernels recorded on `device` since the last
    such call: offsets, slots, page ids or lengths out of range (ValueError; the
    kernels skip what they point at) or a bounded wait that gave up (SAError).
    Synchronises the current stream.  With SA_CHECK_STATUS=1 every serving call
    does this itself."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with torch.cuda.device(dev):
        rc = _lib.load().sa_serving_status(torch.cuda.current_stream(dev).cuda_stream)
    _lib.check(rc, "serving status")
