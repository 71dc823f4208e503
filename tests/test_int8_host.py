"""The host code of the 8-bit tables without a device: hip_stub.cpp stands in for the HIP runtime (two devices, memory that is
addresses only, kernels that end at once), in a process of its own for each test."""
import os
import subprocess
import sys
import textwrap

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STUB = os.path.join(ROOT, "tests", "hip_stub.cpp")

pytestmark = pytest.mark.skipif(not os.path.exists("/opt/rocm/include/hip/hip_runtime_api.h"), reason="needs the HIP headers")

HEAD = """
import ctypes as C, sys
sys.modules["torch"] = None                 # (its own runtime stays out)
stub = C.CDLL(sys.argv[1], C.RTLD_GLOBAL)
for f in (stub.stub_mallocs, stub.stub_frees, stub.stub_launches):
    f.restype = C.c_long
for f in (stub.stub_in_use, stub.stub_most):
    f.restype = C.c_size_t
stub.stub_set_room.argtypes = [C.c_size_t]
from neurondb_amd import _lib
L = _lib.lib()
P = 4096                                    # a device pointer: nothing follows it here
def device():
    d = C.c_int(-1)
    stub.hipGetDevice(C.byref(d))
    return d.value
def table(dim, n=0):
    h = C.c_void_p()
    _lib.check(L.ndbhip_i8_create(dim, C.byref(h)))
    if n:
        _lib.check(L.ndbhip_i8_load_device(h, P, 3, n, dim, P))
    return h
def workspace(t, nq, k):
    b = C.c_size_t()
    _lib.check(L.ndbhip_i8_workspace(t, nq, k, C.byref(b)))
    return b.value
assert L.ndbhip_init(0) == 0
"""


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("stub") / "hip_stub.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", STUB, "-o", so], check=True)
    return so


def run(stub, code):
    r = subprocess.run([sys.executable, "-c", HEAD + textwrap.dedent(code) + "\nprint('done')", stub], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.endswith("done\n"), r.stdout + r.stderr


def test_calls_leave_the_current_device_as_it_was(stub):
    """kernels go to the library's device, and the caller's own is current again afterwards, whatever the call came to"""
    run(stub, """
        import numpy as np
        f = np.ones((300, 16), np.float32).ctypes.data
        def calls(t):
            w = workspace(t, 4, 5) or 1
            return [
                lambda: L.ndbhip_i8_quantize_device(P, 0, 3, 16, 16, P, 16, P), lambda: L.ndbhip_i8_dequantize_device(P, 16, P, 3, 16, P, 0, 16),
                lambda: L.ndbhip_i8_export_device(t, P, 16, P), lambda: L.ndbhip_i8_product_device(t, P, 0, None, 4, 16, None, P, 0, 300, P, w),
                lambda: L.ndbhip_i8_search_device(t, P, 0, None, 4, 16, None, None, 0, 5, P, P, P, w), lambda: L.ndbhip_i8_search(t, f, 4, None, None, 0, 5, f, f),
                lambda: L.ndbhip_scores_adjust_device(P, 0, 4, 70, 70, None, None, 0, None, P, 0, None, 0, 2 * P, 70),
                lambda: L.ndbhip_i8_load(t, f, 300), lambda: L.ndbhip_i8_load_device(t, P, 0, 300, 16, None), lambda: L.ndbhip_i8_load(t, f, 0)]
        stub.hipSetDevice(1)
        for n in (0, 300):
            t = table(16)
            if n:
                _lib.check(L.ndbhip_i8_load(t, f, n))
            for i, c in enumerate(calls(t)):
                stub.hipSetDevice(1)
                before = stub.stub_launches()
                assert c() == 0, i
                assert device() == 1, (n, i)
                assert stub.stub_launches() == before or stub.stub_launch_device() == 0
            _lib.check(L.ndbhip_i8_load(t, f, 300))
            stub.hipSetDevice(1)
            stub.stub_set_room(stub.stub_in_use())
            assert L.ndbhip_i8_search(t, f, 4, None, None, 0, 5, f, f) in (0, _lib.ERR_NOMEM) and device() == 1
            stub.stub_set_room(1 << 60)
            assert L.ndbhip_i8_destroy(t) == 0 and device() == 1
    """)
