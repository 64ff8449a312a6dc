"""Microscaled 4-bit (MXFP4, OCP MX v1.0) messages: gradients squeezed to 17/32
byte per element for the exchange, and the fold of what arrives.

    q = gloo_amd.mx.quantize(grad, residual=err, residual_out=err)
    ...                                     # exchange the payloads (uint8 tensors)
    gloo_amd.mx.reduce_n(grad, payloads, scale=1 / len(payloads))

A payload of n elements is one uint8 tensor of payload_bytes(n): ceil(n / 32)
blocks of 16 bytes (32 E2M1 codes, two to a byte, the even element in the low
half), one scale byte per block (2^(byte - 127); 255: the whole block is
NaN), zero bytes up to a multiple of 16.  Rules of rounding: glx.h
glx_mx_quantize.

Calls enqueue on `stream` (torch.cuda.Stream or raw hipStream_t; default:
torch's current stream) without synchronising and can be captured in a HIP
graph.  Tensors are contiguous and share one device; payloads start at a
16-byte boundary and may be longer than payload_bytes(n), the rest is neither
read nor written.
"""
import ctypes

from . import _lib
from .algorithms import _stream_ptr, torch_dtype_code
from .errors import check

lib = _lib.lib


def payload_bytes(n):
    """Bytes of the payload of n elements."""
    if not 0 <= n <= 1 << 60:
        raise ValueError("payload_bytes: %d elements" % n)
    return int(lib.glx_mx_payload_bytes(n))


def _check(t, what, device, dtype=None):
    if not t.is_cuda or (device is not None and t.device != device):
        raise ValueError("mx: %s is on %s" % (what, t.device))
    if not t.is_contiguous():
        raise ValueError("mx: %s is not contiguous" % what)
    if dtype is not None and t.dtype != dtype:
        raise TypeError("mx: %s is %s, not %s" % (what, t.dtype, dtype))


def _check_payload(t, n, what, device):
    import torch
    _check(t, what, device, torch.uint8)
    if t.numel() < payload_bytes(n):
        raise ValueError("mx: %s has %d bytes, %d elements need %d"
                         % (what, t.numel(), n, payload_bytes(n)))


def _stream(stream, device):
    if stream is None:
        import torch
        stream = torch.cuda.current_stream(device)
    return _stream_ptr(stream)


def _new_payload(n, device, stream):
    import torch
    if stream is None:
        return torch.empty(payload_bytes(n), dtype=torch.uint8, device=device)
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device)
    with torch.cuda.stream(stream):  # the memory belongs to the stream that uses it
        return torch.empty(payload_bytes(n), dtype=torch.uint8, device=device)


def quantize(x, payload=None, residual=None, residual_out=None, stream=None):
    """The payload of x (float32, float16 or bfloat16), or with `residual`
    (float32, as many elements) of x + residual.  residual_out receives what
    the payload leaves out, to be added to the next message; it may be
    `residual` itself.  Returns the payload (allocated unless given)."""
    import torch
    _check(x, "x", None)
    n = x.numel()
    for t, what in ((residual, "residual"), (residual_out, "residual_out")):
        if t is not None:
            _check(t, what, x.device, torch.float32)
            if t.numel() != n:
                raise ValueError("mx: %s has %d elements, x %d" % (what, t.numel(), n))
    code = torch_dtype_code(x)
    if payload is None:
        payload = _new_payload(n, x.device, stream)
    _check_payload(payload, n, "payload", x.device)
    check(lib.glx_mx_quantize(code, payload.data_ptr(), x.data_ptr(),
                              None if residual is None else residual.data_ptr(),
                              None if residual_out is None else residual_out.data_ptr(),
                              n, _stream(stream, x.device)), "mx.quantize")
    return payload


def _sources(payloads, n, device):
    payloads = list(payloads)
    for j, t in enumerate(payloads):
        _check_payload(t, n, "payload %d" % j, device)
    return (ctypes.c_void_p * len(payloads))(*[t.data_ptr() for t in payloads]), len(payloads)


def reduce_n(dst, payloads, scale=1.0, stream=None):
    """dst = scale * the left fold of 1..16 payloads of dst.numel() elements,
    in float32, rounded once to dst's type (float32, float16, bfloat16)."""
    _check(dst, "dst", None)
    arr, k = _sources(payloads, dst.numel(), dst.device)
    check(lib.glx_mx_reduce_n(torch_dtype_code(dst), dst.data_ptr(), arr, k, dst.numel(),
                              float(scale), _stream(stream, dst.device)), "mx.reduce_n")
    return dst


def dequantize(dst, payload, stream=None):
    """dst = the values of a payload of dst.numel() elements."""
    return reduce_n(dst, [payload], stream=stream)


def requantize_n(payload, payloads, n, scale=1.0, stream=None):
    """payload = the payload of scale * the left fold of 1..16 payloads of n
    elements (in float32): one hop of a compressed exchange.  payload may be
    one of the sources."""
    if payload is None:
        raise ValueError("mx: requantize_n needs a payload to write")
    _check_payload(payload, n, "payload", None)
    arr, k = _sources(payloads, n, payload.device)
    check(lib.glx_mx_requantize_n(payload.data_ptr(), arr, k, int(n), float(scale),
                                  _stream(stream, payload.device)), "mx.requantize_n")
    return payload
