"""8-bit tables and scores without a device: arguments are refused before the device is asked for, good ones end in
ERR_NODEVICE (there is no CPU fallback), and the cases of perf/operators.py agree with their own 64-bit values."""
import ctypes as C
import importlib.util
import os
import random
import re
import subprocess

import numpy as np
import pytest
import torch

from neurondb_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
L = _lib.lib()
P = 4096            # a pointer that is never followed
INVALID, NODEVICE, OK = _lib.ERR_INVALID, _lib.ERR_NODEVICE, _lib.OK

no_gpu = pytest.mark.skipif(L.ndbhip_device_count() > 0, reason="a GPU is present: fake pointers must not reach it")


def table(dim=16):
    h = C.c_void_p()
    assert L.ndbhip_i8_create(dim, C.byref(h)) == OK
    return h


def test_handles():
    h = C.c_void_p()
    for dim in (0, -1, 32768):
        assert L.ndbhip_i8_create(dim, C.byref(h)) == INVALID
    assert L.ndbhip_i8_create(4, None) == INVALID
    t = table(33)
    assert (L.ndbhip_i8_dim(t), L.ndbhip_i8_nrows(t)) == (33, 0)
    assert (L.ndbhip_i8_dim(None), L.ndbhip_i8_nrows(None)) == (-1, -1)
    b = C.c_size_t(7)
    assert L.ndbhip_i8_workspace(t, 10, 5, C.byref(b)) == OK and b.value == 0      # an empty table needs none
    for args in ((None, 1, 0, C.byref(b)), (t, -1, 0, C.byref(b)), (t, 1, -1, C.byref(b)), (t, 1, 1025, C.byref(b)), (t, 1, 0, None)):
        assert L.ndbhip_i8_workspace(*args) == INVALID
    assert L.ndbhip_i8_destroy(t) == OK and L.ndbhip_i8_destroy(None) == OK


@no_gpu
@pytest.mark.parametrize("change,want", [
    ({}, NODEVICE), ({"dtype": 3}, INVALID), ({"dtype": -1}, INVALID), ({"n": -1}, INVALID), ({"n": 1 << 31}, INVALID), ({"dim": 0}, INVALID),
    ({"dim": 32768, "xs": 32768, "cs": 32768}, INVALID), ({"xs": 15}, INVALID), ({"cs": 15}, INVALID), ({"x": None}, INVALID),
    ({"c": None}, INVALID), ({"s": None}, INVALID), ({"dtype": 2, "xs": 17, "cs": 99}, NODEVICE)])
def test_quantise_and_dequantise_arguments(change, want):
    a = dict(dtype=0, n=3, dim=16, xs=16, cs=16, x=P, c=P, s=P)
    a.update(change)
    assert L.ndbhip_i8_quantize_device(a["x"], a["dtype"], a["n"], a["dim"], a["xs"], a["c"], a["cs"], a["s"]) == want
    assert L.ndbhip_i8_dequantize_device(a["c"], a["cs"], a["s"], a["n"], a["dim"], a["x"], a["dtype"], a["xs"]) == want


@no_gpu
def test_table_arguments():
    t = table()
    assert L.ndbhip_i8_load(t, P, 3) == NODEVICE
    for args in ((None, P, 3), (t, None, 3), (t, P, -1), (t, P, 1 << 31)):
        assert L.ndbhip_i8_load(*args) == INVALID
    assert L.ndbhip_i8_load_device(t, P, 1, 3, 16, None) == NODEVICE
    assert L.ndbhip_i8_load_device(t, P, 3, 3, 16, P) == NODEVICE
    for args in ((None, P, 0, 3, 16, None), (t, None, 0, 3, 16, None), (t, P, 4, 3, 16, None), (t, P, 0, -1, 16, None), (t, P, 0, 3, 15, None),
                 (t, P, 0, 3, 16, P), (t, P, 3, 3, 16, None)):
        assert L.ndbhip_i8_load_device(*args) == INVALID, args
    assert L.ndbhip_i8_export_device(None, P, 16, P) == INVALID
    assert L.ndbhip_i8_export_device(t, P, 16, P) == NODEVICE
    assert L.ndbhip_i8_destroy(t) == OK


@no_gpu
def test_product_and_search_arguments():
    t = table()
    good = [t, P, 0, None, 4, 16, None, P, 0, 0, P, 0]
    assert L.ndbhip_i8_product_device(*good) == NODEVICE
    for at, v in ((0, None), (1, None), (2, 4), (2, 3), (3, P), (4, -1), (5, 15), (8, 3), (9, -1)):
        a = list(good)
        a[at] = v
        assert L.ndbhip_i8_product_device(*a) == INVALID, (at, v)
    good = [t, P, 0, None, 4, 16, None, None, 0, 5, P, P, P, 0]
    assert L.ndbhip_i8_search_device(*good) == NODEVICE
    for at, v in ((0, None), (1, None), (2, 7), (2, 3), (3, P), (4, -1), (5, 15), (9, 0), (9, 1025), (10, None), (11, None)):
        a = list(good)
        a[at] = v
        assert L.ndbhip_i8_search_device(*a) == INVALID, (at, v)
    assert L.ndbhip_i8_search_device(t, P, 0, None, 4, 16, None, P, -1, 5, P, P, P, 0) == INVALID
    good = [t, P, 4, None, None, 0, 5, P, P]
    assert L.ndbhip_i8_search(*good) == NODEVICE
    for at, v in ((0, None), (1, None), (2, -1), (6, 0), (6, 1025), (7, None), (8, None)):
        a = list(good)
        a[at] = v
        assert L.ndbhip_i8_search(*a) == INVALID, (at, v)
    assert L.ndbhip_i8_destroy(t) == OK


@no_gpu
def test_adjust_arguments():
    good = [P, 0, 4, 70, 70, P, P, 5, P, P, 0, P, 3, 2 * P, 70]
    assert L.ndbhip_scores_adjust_device(*good) == NODEVICE
    for at, v in ((0, None), (1, 3), (2, -1), (3, -1), (4, 69), (6, None), (7, -1), (8, None), (10, 69), (10, -1), (12, 2),
                  (12, -1), (13, None), (14, 69)):
        a = list(good)
        a[at] = v
        assert L.ndbhip_scores_adjust_device(*a) == INVALID, (at, v)
    assert L.ndbhip_scores_adjust_device(P, 0, 4, 70, 70, None, None, 0, None, None, 0, None, 0, P, 71) == INVALID     # in place, another stride
    assert L.ndbhip_scores_adjust_device(P, 0, 4, 70, 70, None, None, 0, None, None, 0, None, 0, P, 70) == NODEVICE


def test_errors_have_a_text():
    h = C.c_void_p()
    assert L.ndbhip_i8_create(0, C.byref(h)) == INVALID
    assert "dim" in _lib.last_error()
    with pytest.raises(_lib.NdbHipError):
        _lib.check(INVALID)


# ------------------------------------------------------------------ the generated code

@pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")
def test_generated_code_of_the_8_bit_kernels(tmp_path):
    """M0, which the LDS copies write in inline assembly, is nobody else's; nothing spills to scratch; no packed fp32"""
    src = os.path.join(ROOT, "neurondb_amd", "csrc", "ndbhip_int8.hip")
    make = open(os.path.join(os.path.dirname(src), "Makefile")).read()
    flags = re.search(r"^CXXFLAGS \?= (.*?[^\\])$", make, re.S | re.M).group(1).replace("\\\n", " ").replace("$(ARCH)", "gfx950").split()
    flags += re.search(r"ndbhip_int8.o: CXXFLAGS \+= (.*)", make).group(1).split()
    out = str(tmp_path / "i8.s")
    subprocess.run(["/opt/rocm/bin/hipcc", *flags, "--cuda-device-only", "-S", src, "-o", out], check=True, stderr=subprocess.DEVNULL)
    s = open(out).read()
    lines = s.splitlines()
    m0 = [i for i, l in enumerate(lines) if re.search(r"\bm0\b", l.split(";")[0])]
    assert len(m0) > 50
    for i in m0:
        assert re.match(r"\ts_mov_b32 m0, s\d+", lines[i]) and "s_nop 4" in lines[i + 1] and "global_load_lds_dword" in lines[i + 2], lines[i]
    assert len([l for l in lines if "global_load_lds" in l]) == len(m0)
    assert set(re.findall(r"\.amdhsa_private_segment_fixed_size (\d+)", s)) == {"0"}
    assert not re.search(r"v_pk_\w+_f32", s)
    tiles = [k for k in re.findall(r"\.amdhsa_kernel (\S+)", s) if "k_i8_tile" in k]
    assert len(tiles) == 2 * (4 + 2 * 2 * 3)
    assert s.count("v_mfma_i32_32x32x32_i8") >= 32 * len(tiles)


# ------------------------------------------------------------------ the plain forms of perf/operators.py, on the CPU

def cases():
    spec = importlib.util.spec_from_file_location("operators_cases", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_listed_and_drawn_cases_are_of_known_shape():
    m = cases()
    listed = m.listed()
    assert 4 <= len(listed) <= 12 and len({c["name"] for c in listed}) == len(listed)
    keys = {c["op"]: set(c) - {"name"} for c in listed}
    assert all(sum(c["op"] == op for c in listed) >= 2 for op in keys)
    rng = random.Random(5)
    top = max(max(m.work(c)["bytes"], m.work(c)["flops"] / 50) for c in listed)
    for _ in range(300):
        c = m.draw(rng)
        assert set(c) == keys[c["op"]]
        assert max(m.work(c)["bytes"], m.work(c)["flops"] / 50) <= top


def test_plain_bytes_against_integers():
    """byte = the integer nearest to x * inv, the product exact: Fractions decide"""
    from fractions import Fraction
    m = cases()
    x = torch.from_numpy(np.random.default_rng(3).standard_normal((6, 40)).astype(np.float32))
    x[0] = torch.linspace(-63.5, 63.5, 40)
    x[0, 0] = 127.0
    codes, scales = m._quantise(x)
    for r in range(6):
        top = max(abs(float(v)) for v in x[r])
        inv = Fraction(float(np.float32(np.float64(127.0) / np.float64(top))))
        for c in range(40):
            p = Fraction(float(x[r, c])) * inv
            assert int(codes[r, c]) == round(p)         # Fraction's round: halves to even
        assert float(scales[r]) == float(np.float32(np.float64(top) / 127.0))


def test_plain_selection_puts_equal_scores_in_the_order_of_their_ids():
    m = cases()
    s = torch.tensor([[1.0, 3.0, 3.0, -0.0, 0.0, float("nan"), float("-inf"), 2.0]])
    ids, v = m._best(s, 8)
    assert ids.tolist() == [[1, 2, 7, 0, 3, 4, -1, -1]]
    assert v[0, :6].tolist() == [3, 3, 2, 1, 0, 0] and torch.isinf(v[0, 6:]).all()
