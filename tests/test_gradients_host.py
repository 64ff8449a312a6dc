"""CPU: what the gradient and MXFP4 entry points decide on the host, run against
two imagined GPUs (tests/cpp/gradients_host_test.cc)."""
import os
import subprocess

import pytest

import gloo_amd  # noqa: F401  (the library the program links)

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


@pytest.mark.parametrize("case", ["mx_pointers", "mx_on", "workspace", "devices"])
def test_host(program, case):
    p = subprocess.run([program, case], capture_output=True, text=True, timeout=60)
    assert p.returncode == 0, p.stdout + p.stderr
