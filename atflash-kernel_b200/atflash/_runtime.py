"""Per-device runtime state of the Python layer: the device error flag that the
kernels' bounded waits report into, and the current stream handle."""
import ctypes
import threading

import torch

from . import _ffi

_flags = {}
_lock = threading.Lock()


def error_flag(device: torch.device) -> torch.Tensor:
    """int32[1] on `device`, zero-initialised once per device."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    with _lock:
        t = _flags.get(idx)
        if t is None:
            t = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", idx))
            # kernels on any stream read it from now on (a capture cannot wait: its fill
            # is the graph's first node)
            if not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream(idx).synchronize()
            _flags[idx] = t
    return t


def error_flag_ptr(device: torch.device) -> int:
    """Address of error_flag(device); of a flag that is there, without the lock."""
    t = _flags.get(device.index)
    return (error_flag(device) if t is None else t).data_ptr()


def check_device_errors(device=None) -> int:
    """Synchronise `device`, return (and clear) its kernel error flag.

    2 is an index report: a call left out lengths, pages, rows or items that do not fit
    (its documentation says which); later calls run as ever. Any other non-zero
    value means that a bounded device wait expired and a kernel returned early: its
    outputs are not valid, nor are those of attention calls since, which return
    without computing until this function clears the flag."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    flag = error_flag(dev)
    out = ctypes.c_int(0)
    with torch.cuda.device(dev):
        _ffi.check("atf_read_error_flag", _ffi.load().atf_read_error_flag(flag.data_ptr(), ctypes.byref(out)))
    return out.value


def stream_handle(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def launch(name: str, fn, device: torch.device, *args) -> None:
    """fn(*args, current stream) with `device` current; raises on a non-zero status.
    (The device guard and a Stream object cost more than the call itself: both are
    left out where `device` is current already.)"""
    idx = device.index
    if idx == torch.cuda.current_device():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(idx))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(idx))
    if rc:
        _ffi.check(name, rc)


def narrow_i32(t: torch.Tensor, device: torch.device, top: int = 0x7fffffff) -> torch.Tensor:
    """An index tensor as contiguous int32 on `device`. 64-bit values that do not fit
    become -1 or `top`, which the kernels report, instead of another valid index."""
    if t.dtype == torch.int64:
        t = t.clamp(-1, top)
    return t.to(device=device, dtype=torch.int32).contiguous()


class PlanTensors:
    """The device tensors of a plan. Runs use them on their own current stream, which
    need not be the one they were allocated on: each stream is recorded with the
    allocator, so that tensors dropped by a new plan are not handed out again before the
    runs that read them have ended."""

    def __init__(self, device: torch.device, *tensors: torch.Tensor):
        self._idx, self._tensors, self._streams = device.index, tensors, set()

    def use(self) -> None:
        """Before a launch that reads the tensors on the current stream."""
        raw = torch._C._cuda_getCurrentRawStream(self._idx)
        if raw not in self._streams:
            stream = torch.cuda.current_stream(self._idx)
            for t in self._tensors:
                t.record_stream(stream)
            self._streams.add(raw)


def require_cuda(*tensors: torch.Tensor) -> torch.device:
    dev = None
    for t in tensors:
        if not t.is_cuda:
            raise ValueError("atflash kernels take CUDA tensors (there is no CPU path)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError("all tensors must be on the same device")
    return dev


def selftest_wait_timeout(device=None) -> int:
    """Run the bounded-wait self-test on `device` (about 2 s): a kernel waits on
    a barrier nothing arrives on, gives up after the wait limit and reports
    through the error flag. Returns the flag value (1 = wait timed out)."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    flag = error_flag(dev)
    with torch.cuda.device(dev):
        _ffi.check("atf_selftest_wait_timeout",
                   _ffi.load().atf_selftest_wait_timeout(flag.data_ptr(), stream_handle(dev)))
    return check_device_errors(dev)
