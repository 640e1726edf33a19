"""The device status word of the stream-ordered operators (slots, qk_norm,
prefix_attention).

Their calls enqueue kernels and return. What only the GPU sees -- a length,
position, block or slot out of range, exhausted blocks -- is skipped and
recorded in a status word. A caller that keeps a `DeviceStatus` passes it to
every call of a stream and checks it when it synchronises anyway; a call
without one waits for its kernels and raises at once.
"""

from __future__ import annotations

from . import _lib


class DeviceStatus:
    def __init__(self, device="cuda"):
        import torch
        self.word = torch.zeros(1, dtype=torch.int32, device=device)
        self.ptr = self.word.data_ptr()

    def check(self, stream=None):
        """Wait for the stream (default: the current one); raise EngineError
        with LS_ECAPACITY or LS_EDEVICE, and clear the word, if a call on it
        recorded a fault."""
        import torch
        device = self.word.device
        if stream is None:
            stream = torch.cuda.current_stream(device).cuda_stream
        with torch.cuda.device(device):
            _lib.check(_lib.lib().ls_check_status(self.ptr, stream))


def enqueue(call, pack, before, after, device, status, stream):
    """Run `call(struct, stream)` on the tensors' device, where the struct is
    pack(*before, status word, *after); with no status, wait and raise."""
    import torch
    if stream is None:
        stream = torch.cuda.current_stream(device).cuda_stream
    if status is None:
        with torch.cuda.device(device), torch.cuda.stream(torch.cuda.ExternalStream(stream, device)):
            own = DeviceStatus(device)
            _lib.check(call(pack(*before, own.ptr, *after), stream))
            own.check(stream)
    elif device.index == torch.cuda.current_device():
        _lib.check(call(pack(*before, status.ptr, *after), stream))
    else:
        with torch.cuda.device(device):
            _lib.check(call(pack(*before, status.ptr, *after), stream))


def require(ok, message):
    if not ok:
        raise ValueError(message)
