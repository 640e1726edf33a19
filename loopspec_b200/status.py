"""The device status word of the stream-ordered operators (slots, qk_norm,
prefix_attention).

Their calls enqueue kernels and return. What only the GPU sees -- a length,
position, block or slot out of range, exhausted blocks -- is skipped and
recorded in a status word. A caller that keeps a `DeviceStatus` passes it to
every call of a stream and checks it when it synchronises anyway; a call
without one waits for its kernels and raises at once.
"""

from __future__ import annotations

from contextlib import nullcontext

import torch

from . import _lib


class DeviceStatus:
    """A status word on one GPU, for calls on tensors of that GPU: kernels write it by its address."""

    def __init__(self, device="cuda"):
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"the status word must be on a GPU, not on {device}")
        self.word = torch.zeros(1, dtype=torch.int32, device=device)
        self.gpu = self.word.get_device()
        self.ptr = self.word.data_ptr()

    def check(self, stream=None):
        """Wait for the stream (default: the current one); raise EngineError
        with LS_ECAPACITY or LS_EDEVICE, and clear the word, if a call on it
        recorded a fault."""
        device = self.word.device
        if stream is None:
            stream = torch.cuda.current_stream(device).cuda_stream
        with torch.cuda.device(device):
            _lib.check(_lib.lib().ls_check_status(self.ptr, stream))


# The current stream's handle without the Stream object around it, which costs
# 2 of the ~8 microseconds that a small call takes on the host; the current
# device without the initialisation check, as there are tensors on one.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def enqueue(call, pack, before, after, gpu, status, stream):
    """Run `call(struct, stream)` on the tensors' GPU (its index), where the struct
    is pack(*before, status word, *after); with no status, wait and raise."""
    if stream is None:
        stream = _raw_stream(gpu)
    if status is None:
        with torch.cuda.device(gpu), torch.cuda.stream(torch.cuda.ExternalStream(stream, gpu)):
            own = DeviceStatus(torch.device("cuda", gpu))
            _lib.check(call(pack(*before, own.ptr, *after), stream))
            own.check(stream)
        return
    if status.gpu != gpu:
        raise ValueError(f"the status word is on GPU {status.gpu}, the tensors on GPU {gpu}")
    if gpu == _current_device():
        code = call(pack(*before, status.ptr, *after), stream)
    else:
        with torch.cuda.device(gpu):
            code = call(pack(*before, status.ptr, *after), stream)
    if code:
        _lib.check(code)


def on_stream(device, stream):
    """A context whose allocations belong to `stream` (a handle, or None for the current one)."""
    return nullcontext() if stream is None else torch.cuda.stream(torch.cuda.ExternalStream(stream, device))
