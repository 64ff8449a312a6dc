"""CPU: what the gradient and MXFP4 entry points decide on the host, run against
two imagined GPUs (tests/cpp/gradients_host_test.cc)."""
import os
import subprocess
import types

import pytest

import gloo_amd
from gloo_amd import mx

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("cpp") / "gradients_host_test")
    lib = os.path.join(ROOT, "gloo_amd")
    subprocess.check_call(
        ["g++", "-std=c++17", "-O1", "-Wall", "-rdynamic", "-D__HIP_PLATFORM_AMD__",
         "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "include"),
         os.path.join(ROOT, "tests", "cpp", "gradients_host_test.cc"), "-o", exe, "-L" + lib,
         "-lgloo_amd", "-L/opt/rocm/lib", "-lamdhip64", "-Wl,-rpath," + lib])
    return exe


@pytest.mark.parametrize("case", ["mx_pointers", "mx_on", "workspace", "devices", "destroy", "cached"])
def test_host(program, case):
    p = subprocess.run([program, case], capture_output=True, text=True, timeout=60)
    assert p.returncode == 0, p.stdout + p.stderr


class Recorder:
    """The library's entry points, writing down the stream of each call."""

    def __init__(self):
        self.streams = []

    def __getattr__(self, name):
        def call(*args):
            self.streams.append(args[-1])
            return 0
        return call


def cuda_tensor(dtype, n, device):
    """What the bindings ask of a tensor, without a GPU."""
    size = torch.empty(0, dtype=dtype).element_size()
    return types.SimpleNamespace(
        dtype=dtype, device=torch.device(device), is_cuda=True, data_ptr=lambda: 1 << 20,
        numel=lambda: n, is_contiguous=lambda: True, is_neg=lambda: False, element_size=lambda: size)


def test_negated_scalars_are_refused():
    """A negated view (z.conj().imag) holds its values' opposites in memory."""
    z = torch.zeros(1, dtype=torch.complex128).conj().imag
    assert z.is_neg()
    g = gloo_amd.Gradients.__new__(gloo_amd.Gradients)
    g._h, g._ws, g._code, g.device, g.dtype = 1, 0, 6, z.device, torch.float64
    try:
        for call in (lambda: g.norm(out=z), lambda: g.power_sum(out=z),
                     lambda: g.clip_norm(1.0, power_sum=z)):
            with pytest.raises(ValueError, match="negated"):
                call()
    finally:
        g._h = None  # not a handle


def test_stream_of_another_device_is_refused(monkeypatch):
    """torch.cuda.stream() of a stream on another device leaves the tensors'
    device's current stream as it is: the call would go there unnoticed."""
    rec = Recorder()
    monkeypatch.setattr(mx, "lib", rec)
    monkeypatch.setattr(gloo_amd.gradients, "lib", rec)
    monkeypatch.setattr(mx, "current_stream_ptr", lambda d: "current of %s" % d)
    monkeypatch.setattr(gloo_amd.gradients, "current_stream_ptr", lambda d: "current of %s" % d)

    class With:
        def __init__(self, stream):
            pass

        def __enter__(self):
            pass

        def __exit__(self, *a):
            pass
    monkeypatch.setattr(torch.cuda, "stream", With)
    x = cuda_tensor(torch.float32, 64, "cuda:0")
    p = cuda_tensor(torch.uint8, 48, "cuda:0")
    g = gloo_amd.Gradients.__new__(gloo_amd.Gradients)
    g._h, g._ws, g._code, g.device, g.dtype = 1, 0, 5, x.device, torch.float32
    one = cuda_tensor(torch.float32, 1, "cuda:0")
    wide = cuda_tensor(torch.float64, 1, "cuda:0")
    calls = [lambda s: mx.quantize(x, p, stream=s), lambda s: mx.reduce_n(x, [p], stream=s),
             lambda s: mx.dequantize(x, p, stream=s),
             lambda s: mx.requantize_n(p, [p], 64, stream=s),
             lambda s: g.norm(out=one, stream=s), lambda s: g.power_sum(out=wide, stream=s),
             lambda s: g.clip_norm(1.0, out=one, stream=s)]
    here, there = (types.SimpleNamespace(device=torch.device(d)) for d in ("cuda:0", "cuda:1"))
    try:
        for call in calls:
            with pytest.raises(ValueError, match="stream is on cuda:1"):
                call(there)
            assert not rec.streams
            call(here)
            assert rec.streams.pop() == "current of cuda:0"
    finally:
        g._h = None  # not a handle
