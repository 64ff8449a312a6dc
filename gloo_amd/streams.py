"""Torch's streams for calls that enqueue kernels of their own."""
from . import _lib

torch = _lib.torch

# the current stream's handle without making a Stream object (0.1 instead of
# 1.8 us on the host), where this torch has it
_raw = getattr(getattr(torch, "_C", None), "_cuda_getCurrentRawStream", None)


def current_stream_ptr(device):
    """hipStream_t of torch's current stream on `device` (a torch.device with
    an index)."""
    if _raw is not None:
        return _raw(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def as_torch_stream(stream, device):
    """A torch.cuda.Stream of `device`, or a raw hipStream_t of it as one."""
    if isinstance(stream, int):
        return torch.cuda.ExternalStream(stream, device)
    if stream.device != device:
        raise ValueError("the stream is on %s, the tensors on %s" % (stream.device, device))
    return stream
