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
from .algorithms import BFLOAT16, FLOAT16, FLOAT32
from .errors import check
from .streams import as_torch_stream, current_stream_ptr

lib = _lib.lib
torch = _lib.torch
_CODES = {} if torch is None else {
    torch.float32: FLOAT32, torch.float16: FLOAT16, torch.bfloat16: BFLOAT16}


def payload_bytes(n):
    """Bytes of the payload of n elements (glx_mx_payload_bytes)."""
    if not 0 <= n <= 1 << 60:
        raise ValueError("payload_bytes: %d elements" % n)
    return ((n + 31) // 32 * 17 + 15) // 16 * 16


def _check(t, what, device=None):
    if not t.is_cuda or (device is not None and t.device != device):
        raise ValueError("mx: %s is on %s" % (what, t.device))
    if not t.is_contiguous() or t.is_neg():
        raise ValueError("mx: %s is not contiguous, or a negated view" % what)


def _code(t, what):
    code = _CODES.get(t.dtype)
    if code is None:
        raise TypeError("mx: %s is %s, not float32, float16 or bfloat16" % (what, t.dtype))
    return code


def _payload_ptr(t, need, device, j=None):
    """Address of a payload (the j-th source) of at least `need` bytes."""
    if t.dtype != torch.uint8 or t.device != device or not t.is_contiguous() or t.is_neg() or \
            t.numel() < need or not t.is_cuda:
        what = "payload" if j is None else "payload %d" % j
        _check(t, what, device)
        if t.dtype != torch.uint8:
            raise TypeError("mx: %s is %s, not uint8" % (what, t.dtype))
        raise ValueError("mx: %s has %d bytes of the %d needed" % (what, t.numel(), need))
    return t.data_ptr()


def _residual_ptr(t, n, device, what):
    if t is None:
        return None
    _check(t, what, device)
    if t.dtype != torch.float32:
        raise TypeError("mx: %s is %s, not float32" % (what, t.dtype))
    if t.numel() != n:
        raise ValueError("mx: %s has %d elements, x %d" % (what, t.numel(), n))
    return t.data_ptr()


def quantize(x, payload=None, residual=None, residual_out=None, stream=None):
    """The payload of x (float32, float16 or bfloat16), or with `residual`
    (float32, as many elements) of x + residual.  residual_out receives what
    the payload leaves out, to be added to the next message; it may be
    `residual` itself.  Returns the payload (allocated unless given)."""
    if stream is not None:
        with torch.cuda.stream(as_torch_stream(stream, x.device)):
            return quantize(x, payload, residual, residual_out)
    _check(x, "x")
    code, n, device = _code(x, "x"), x.numel(), x.device
    need = payload_bytes(n)
    if payload is None:
        payload = torch.empty(need, dtype=torch.uint8, device=device)
    check(lib.glx_mx_quantize_on(device.index, code, _payload_ptr(payload, need, device),
                                 x.data_ptr(), _residual_ptr(residual, n, device, "residual"),
                                 _residual_ptr(residual_out, n, device, "residual_out"),
                                 n, current_stream_ptr(device)), "mx.quantize")
    return payload


def _sources(payloads, need, device):
    ptrs = [_payload_ptr(t, need, device, j) for j, t in enumerate(payloads)]
    return (ctypes.c_void_p * len(ptrs))(*ptrs), len(ptrs)


def reduce_n(dst, payloads, scale=1.0, stream=None):
    """dst = scale * the left fold of 1..16 payloads of dst.numel() elements,
    in float32, rounded once to dst's type (float32, float16, bfloat16)."""
    if stream is not None:
        with torch.cuda.stream(as_torch_stream(stream, dst.device)):
            return reduce_n(dst, payloads, scale)
    _check(dst, "dst")
    code, n, device = _code(dst, "dst"), dst.numel(), dst.device
    arr, k = _sources(payloads, payload_bytes(n), device)
    check(lib.glx_mx_reduce_n_on(device.index, code, dst.data_ptr(), arr, k, n, scale,
                                 current_stream_ptr(device)), "mx.reduce_n")
    return dst


def dequantize(dst, payload, stream=None):
    """dst = the values of a payload of dst.numel() elements."""
    return reduce_n(dst, (payload,), 1.0, stream)


def requantize_n(payload, payloads, n, scale=1.0, stream=None):
    """payload = the payload of scale * the left fold of 1..16 payloads of n
    elements (in float32): one hop of a compressed exchange.  payload may be
    one of the sources."""
    if stream is not None:
        with torch.cuda.stream(as_torch_stream(stream, payload.device)):
            return requantize_n(payload, payloads, n, scale)
    need, device = payload_bytes(n), payload.device
    out = _payload_ptr(payload, need, device)
    arr, k = _sources(payloads, need, device)
    check(lib.glx_mx_requantize_n_on(device.index, out, arr, k, n, scale,
                                     current_stream_ptr(device)), "mx.requantize_n")
    return payload
