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


def test_workspace_of_long_tables_stays_in_bounds(stub):
    """a search's passes are cut so that the workspace is about a gigabyte; a tile's 256 queries may take 16"""
    run(stub, """
        G = 1 << 30
        for n, dim in ((1_000, 64), (1_000_000, 768), (27_000_000, 64), (100_000_000, 64), (100_000_000, 768), (500_000_000, 64), (0x7FFFFF00, 64), (0x7FFFFF00, 90)):
            t = table(dim, n)
            bound = max(1.02 * G, min(16 * G, 41 * n)) + (64 << 20)
            for k in (1, 10, 128, 129, 1024):
                last = 0
                for nq in (1, 31, 33, 255, 256, 257, 1024, 5000, 2**31 - 1):
                    w = workspace(t, nq, k)
                    assert w >= last and w <= bound and w < stub.stub_in_use() * 5 // 8 + G, (n, dim, k, nq, w)
                    last = w
            assert workspace(t, 2**31 - 1, 0) <= 4096 * (dim + 64 + 4) + 4096
            _lib.check(L.ndbhip_i8_destroy(t))
        assert stub.stub_in_use() < G
    """)


def test_passes(stub):
    """launches of a call: the queries, then the product, then what picks the best; the table is read no more often than needed"""
    run(stub, """
        def product(t, nq, dim, n):
            before = stub.stub_launches()
            _lib.check(L.ndbhip_i8_product_device(t, P, 3, P, nq, dim, None, P, 0, n, P, workspace(t, nq, 0)))
            return stub.stub_launches() - before
        def search(t, nq, dim, k):
            before = stub.stub_launches()
            _lib.check(L.ndbhip_i8_search_device(t, P, 3, P, nq, dim, None, None, 0, k, P, P, P, workspace(t, nq, k)))
            return stub.stub_launches() - before
        t = table(768, 10_000_000)
        assert product(t, 1024, 768, 10_000_000) == 2 and product(t, 4096, 768, 10_000_000) == 2 and product(t, 4097, 768, 10_000_000) == 4
        t = table(32, 300)
        assert search(t, 4096, 32, 5) == 3 and search(t, 9001, 32, 5) == 9
        t = table(64, 100_000_000)              # 256 queries: 3.7 GB
        assert search(t, 256, 64, 10) == 3 and search(t, 257, 64, 10) == 6
        t = table(64, 500_000_000)              # 16 GiB: 192 queries a pass
        assert search(t, 192, 64, 10) == 3 and search(t, 193, 64, 10) == 6
    """)


def test_searches_of_host_arrays_keep_their_workspace(stub):
    """hipMalloc and hipFree, which waits for everything on the device, are for the first search and for larger ones only; searches
    at the same time have a workspace each; all of it goes with the table's rows"""
    run(stub, """
        import numpy as np, threading
        a = np.ones((300, 16), np.float32).ctypes.data
        def search(t, nq, k=5):
            return L.ndbhip_i8_search(t, a, nq, None, None, 0, k, a, a)
        empty = stub.stub_in_use()
        t = table(16, 100_000)
        rows = stub.stub_in_use()
        _lib.check(search(t, 4))
        m, f, kept = stub.stub_mallocs(), stub.stub_frees(), stub.stub_in_use()
        assert kept > rows
        for _ in range(5):
            _lib.check(search(t, 4))
            _lib.check(search(t, 1))
        assert (stub.stub_mallocs(), stub.stub_frees(), stub.stub_in_use()) == (m, f, kept)
        _lib.check(search(t, 200))                      # a larger one: in place of the first
        assert stub.stub_mallocs() == m + 1 and stub.stub_frees() == f + 1
        # two at the same time
        stub.stub_set_sync_ms(300)
        got = []
        th = [threading.Thread(target=lambda: got.append(search(t, 4))) for _ in range(2)]
        [x.start() for x in th]
        [x.join() for x in th]
        stub.stub_set_sync_ms(0)
        assert got == [0, 0] and stub.stub_mallocs() == m + 2
        _lib.check(search(t, 4)), _lib.check(search(t, 200))
        assert stub.stub_mallocs() == m + 2
        # no room: an error, and the next search has its workspace again
        stub.stub_set_room(stub.stub_in_use())
        assert search(t, 250, 1000) == _lib.ERR_NOMEM and "room" in _lib.last_error()
        stub.stub_set_room(1 << 62)
        _lib.check(search(t, 250, 1000)), _lib.check(search(t, 4))
        # a workspace of more than a gigabyte is not kept
        before = stub.stub_in_use()
        big = table(64, 100_000_000)
        rows = stub.stub_in_use()
        _lib.check(L.ndbhip_i8_search(big, a, 256, None, None, 0, 5, a, a))
        assert stub.stub_in_use() == rows and stub.stub_most() > rows + 3 * 10**9
        _lib.check(L.ndbhip_i8_destroy(big))
        assert stub.stub_in_use() == before
        _lib.check(L.ndbhip_i8_load_device(t, P, 3, 1000, 16, P))
        _lib.check(L.ndbhip_i8_destroy(t))
        assert stub.stub_in_use() == empty
    """)
