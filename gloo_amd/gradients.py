"""The global norm of a list of gradients, and clipping by it: what a
data-parallel program does with the buffers its allreduce returns.

    g = gloo_amd.Gradients(grads)          # the tensors' memory, laid out once
    total = g.clip_norm(1.0)               # in place; the norm, on the device
"""
import ctypes

from . import _lib
from .algorithms import BFLOAT16, FLOAT16, FLOAT32, FLOAT64
from .errors import check, check_handle
from .streams import as_torch_stream, current_stream_ptr

lib = _lib.lib
torch = _lib.torch
_CODES = {} if torch is None else {
    torch.float32: FLOAT32, torch.float64: FLOAT64, torch.float16: FLOAT16,
    torch.bfloat16: BFLOAT16}


def _dense(t):
    """Whether the elements of t fill one stretch of memory, in any order."""
    expect = 1
    for stride, size in sorted(zip(t.stride(), t.shape)):
        if size == 1:
            continue
        if stride != expect:
            return False
        expect *= size
    return True


def _same_order(a, b):
    """Whether the strides of two tensors of one shape agree where they matter."""
    return a.numel() == 0 or all(
        x == y for x, y, n in zip(a.stride(), b.stride(), a.shape) if n > 1)


class Gradients:
    """Gradient tensors of one device (float32, float64, float16 or bfloat16,
    mixed as they come; empty ones too).  A tensor may start at any element of
    its storage and have its dimensions in any order, but its elements fill
    one stretch of memory.  With `outs`, tensors of the same types, shapes and
    strides, clip_norm writes there and leaves the gradients as they are
    (outs[i] may be grads[i]).  Tensors that share memory are refused.

    The object keeps the memory that the tensors have when it is made, as the
    allreduce classes do: after giving a parameter another gradient tensor,
    make another one.  Calls enqueue on `stream` (torch.cuda.Stream or raw
    hipStream_t; default: torch's current stream) without synchronising, and
    can be captured in a HIP graph; each has a workspace of its own, so they
    may run at once on several streams.  The caller orders them after whatever
    wrote the gradients, and keeps the object alive while a graph holding it is
    replayed.  Make it outside of a capture, and once, not once a step: dropping
    it waits for the device's work (and may happen during a capture, of a graph
    that does not hold it)."""

    def __init__(self, grads, outs=None):
        grads = list(grads)
        outs = None if outs is None else list(outs)
        if outs is not None and len(outs) != len(grads):
            raise ValueError("%d gradients, %d outs" % (len(grads), len(outs)))
        self._h = None
        device = grads[0].device if grads else None
        codes = []
        for i, t in enumerate(grads):
            code = _CODES.get(t.dtype)
            if code is None:
                raise TypeError("gradient %d is %s" % (i, t.dtype))
            codes.append(code)
            if not t.is_cuda or t.device != device:
                raise ValueError("gradient %d is on %s" % (i, t.device))
            if t.is_neg():
                raise ValueError("gradient %d is a negated view" % i)
            if not t.is_contiguous() and not _dense(t):
                raise ValueError("gradient %d has gaps or overlaps in its memory (strides %s)"
                                 % (i, t.stride()))
            if outs is None:
                continue
            o = outs[i]
            if o.dtype != t.dtype:
                raise TypeError("out %d is %s, its gradient %s" % (i, o.dtype, t.dtype))
            if o.is_neg():
                raise ValueError("out %d is a negated view" % i)
            if o.device != device or o.shape != t.shape or (
                    o.stride() != t.stride() and not _same_order(o, t)):
                raise ValueError("out %d does not have its gradient's device, shape and strides"
                                 % i)
        n = len(grads)
        self.device = device or torch.device("cuda", torch.cuda.current_device())
        wide = FLOAT64 in codes
        self.dtype = torch.float64 if wide else torch.float32  # of the norm
        self._code = FLOAT64 if wide else FLOAT32
        # aliases hold the memory, also if a tensor is given another later
        self._keep = [t.detach() for t in grads] + [t.detach() for t in outs or ()]
        ptrs = (ctypes.c_void_p * n)(*[t.data_ptr() for t in grads])
        optr = None if outs is None else (ctypes.c_void_p * n)(*[t.data_ptr() for t in outs])
        self._h = check_handle(
            lib.glx_gradients_create(ptrs, optr, (ctypes.c_size_t * n)(*[t.numel() for t in grads]),
                                     (ctypes.c_int * n)(*codes), n), "Gradients")
        self._ws = lib.glx_gradients_workspace_bytes(self._h) // 8

    def _scalar(self, t, dtype, what):
        if t.dtype != dtype or t.numel() != 1 or t.device != self.device:
            raise ValueError("%s: one %s on %s" % (what, dtype, self.device))
        if t.is_neg():
            raise ValueError("%s is a negated view" % what)
        return t.data_ptr()

    def _begin(self, dtype, out):
        """(handle, result tensor, workspace, its pointer or None, stream) of
        one call on the current stream, which what is allocated here belongs to."""
        if self._h is None:
            raise ValueError("Gradients: closed")
        if out is None:
            out = torch.empty_strided((), (), dtype=dtype, device=self.device)
        else:
            self._scalar(out, dtype, "out")
        ws = torch.empty(self._ws, dtype=torch.float64, device=self.device) if self._ws else None
        return (self._h, out, ws, None if ws is None else ws.data_ptr(),
                current_stream_ptr(self.device))

    def power_sum(self, p=2.0, out=None, stream=None):
        """The sum of |x|^p over all gradients (the maximum of |x| for
        p = inf; p is 1, 2 or inf), accumulated in and returned as float64.
        Ranks holding shards allreduce it (SUM; MAX for inf) and give it to
        clip_norm.  For p = 2, float64 values beyond about 1.3e154 make it
        infinite, and it is 0 if all are below 1.5e-162."""
        if stream is not None:
            with torch.cuda.stream(as_torch_stream(stream, self.device)):
                return self.power_sum(p, out)
        h, out, ws, wp, s = self._begin(torch.float64, out)
        check(lib.glx_gradients_power_sum(h, p, out.data_ptr(), wp, s), "Gradients")
        return out

    def norm(self, p=2.0, out=None, stream=None):
        """The p-norm of all gradients together: float32, or float64 if one
        of them is."""
        if stream is not None:
            with torch.cuda.stream(as_torch_stream(stream, self.device)):
                return self.norm(p, out)
        h, out, ws, wp, s = self._begin(self.dtype, out)
        check(lib.glx_gradients_norm(h, p, out.data_ptr(), self._code, wp, s), "Gradients")
        return out

    def clip_norm(self, max_norm, p=2.0, power_sum=None, out=None, stream=None):
        """Scale every gradient by min(1, max_norm / (norm + 1e-6)), in place
        or into outs, and return the norm (as norm() does): the list's own,
        or that of power_sum (a float64 on the device).  A NaN norm makes
        every gradient NaN, an infinite one 0 (NaN where it was infinite), or
        NaN if max_norm is infinite too (inf / inf)."""
        if stream is not None:
            with torch.cuda.stream(as_torch_stream(stream, self.device)):
                return self.clip_norm(max_norm, p, power_sum, out)
        total = None if power_sum is None else self._scalar(power_sum, torch.float64, "power_sum")
        h, out, ws, wp, s = self._begin(self.dtype, out)
        check(lib.glx_gradients_clip(h, max_norm, p, total, out.data_ptr(), self._code, wp, s),
              "Gradients")
        return out

    def close(self):
        """Free the handle, after the work in flight on its device (no graph
        holding it may be replayed afterwards)."""
        h, self._h = getattr(self, "_h", None), None
        if h:
            lib.glx_gradients_destroy(h)

    def __del__(self):
        self.close()
