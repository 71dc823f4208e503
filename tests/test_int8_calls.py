"""The way from Python and C to the 8-bit kernels, without a device: what the calls on torch tensors refuse."""
import os
import re

import pytest
import torch

from neurondb_amd import _lib, int8
from neurondb_amd._lib import NdbHipError

L = _lib.lib()
no_gpu = pytest.mark.skipif(L.ndbhip_device_count() > 0, reason="a GPU is present: the module serves its tensors")


@pytest.fixture
def adjust():
    """csrc/ndb_torch.cpp told that the library is on the CPU: its checks run, and a good call ends where the device is asked for"""
    m = int8._native("cpu")

    def call(scores, seen=None, penalties=None, bias=None, mask=None, out=None):
        return m.adjust(1, scores, seen, penalties, bias, mask, out)
    return call


def code_of(call):
    with pytest.raises(NdbHipError) as e:
        call()
    return e.value.code


@no_gpu
def test_adjust_refuses_what_it_cannot_read(adjust):
    s, w = torch.ones(4, 70), torch.zeros(4, 3, dtype=torch.int32)
    off, ids, pen = torch.zeros(5, dtype=torch.int64), torch.zeros(2, dtype=torch.int32), torch.ones(4, 3)
    bad = [
        lambda: adjust(None), lambda: adjust([1.0]), lambda: adjust(s[0]), lambda: adjust(s.double()), lambda: adjust(s.int()),
        lambda: adjust(s.to_sparse()), lambda: adjust(torch.ones(4, 70, device="meta")),
        lambda: adjust(s, seen=(off, ids)), lambda: adjust(s, penalties=pen), lambda: adjust(s, (off[:4], ids), pen),
        lambda: adjust(s, (off, ids, ids), pen), lambda: adjust(s, (off.int(), ids), pen), lambda: adjust(s, (off, ids.long()), pen),
        lambda: adjust(s, (off, ids[None]), pen), lambda: adjust(s, (off, ids), pen[:, :2]), lambda: adjust(s, (off, ids), pen[:3]),
        lambda: adjust(s, bias=torch.ones(69)), lambda: adjust(s, bias=torch.ones(3, 70)), lambda: adjust(s, bias=torch.ones(70).half()),
        lambda: adjust(s, bias=torch.ones(1, 1, 70)), lambda: adjust(s, mask=w[:, :2]), lambda: adjust(s, mask=w[:3]), lambda: adjust(s, mask=w.float()),
        lambda: adjust(s, out=s.half()), lambda: adjust(s, out=torch.ones(4, 71)), lambda: adjust(s, out=torch.ones(70, 4).t()),
        lambda: adjust(s, out=torch.ones(1, 70).expand(4, 70)),
    ]
    for i, c in enumerate(bad):
        assert code_of(c) == _lib.ERR_INVALID, i
    with pytest.raises(TypeError):
        adjust(s, seen=3, penalties=pen)


@no_gpu
def test_adjust_takes_what_it_can_read(adjust):
    s, w = torch.ones(4, 70), torch.zeros(4, 3, dtype=torch.int32)
    off, ids, pen = torch.zeros(5, dtype=torch.int64), torch.zeros(2, dtype=torch.int32), torch.ones(4, 3)
    good = [
        lambda: adjust(s), lambda: adjust(s.half()), lambda: adjust(s.bfloat16()), lambda: adjust(s.t().contiguous().t()), lambda: adjust(s[:, ::2]),
        lambda: adjust(s, (off, ids), pen), lambda: adjust(s, [off, ids], pen), lambda: adjust(s, (off, ids[:0]), pen),
        lambda: adjust(s, bias=torch.ones(70)), lambda: adjust(s, bias=torch.ones(1, 70)), lambda: adjust(s, bias=torch.ones(70, 4).t()),
        lambda: adjust(s, bias=torch.ones(1).expand(70)), lambda: adjust(s, mask=w[0]), lambda: adjust(s, mask=w),
        lambda: adjust(s, mask=w.view(torch.uint32)), lambda: adjust(s, out=s), lambda: adjust(s, out=torch.ones(4, 99)[:, 7:77]), lambda: adjust(s[:0]),
    ]
    for i, c in enumerate(good):
        assert code_of(c) == _lib.ERR_NODEVICE, i


@pytest.mark.parametrize("taken_up,want", [(True, 1), (False, None)])
def test_a_table_is_on_the_device_of_the_tensors_it_will_meet(monkeypatch, taken_up, want):
    """as the first call of a process: torch's current device, as the calls on tensors take, or, without one, the process's own"""
    asked = []
    monkeypatch.setattr(_lib, "_inited", False)
    monkeypatch.setattr(int8, "ensure_init", asked.append)
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: taken_up)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    int8.Int8Table(8).close()
    int8.Int8Table(8, device=0).close()
    assert asked == [want, 0]


@pytest.fixture
def on_cpu(monkeypatch):
    """the module as after its first call, told that the library is on the CPU: a good call ends where the device is asked for"""
    monkeypatch.setattr(int8, "ensure_init", lambda device=None: None)
    monkeypatch.setattr(_lib, "_inited", True)
    monkeypatch.setattr(_lib, "_device", 0)
    T = int8._Torch()
    T.device, T.stream, T.adjust = torch.device("cpu"), lambda: 1, int8._native("cpu").adjust
    monkeypatch.setattr(int8, "_state", T)


@no_gpu
def test_tensors_whose_gradients_would_be_lost_are_refused(on_cpu):
    """the results carry no graph: an argument that autograd follows is refused while it does"""
    x, b, s = torch.ones(4, 16), torch.ones(70), torch.ones(4, 70)
    c, sc, pen = torch.ones(4, 16, dtype=torch.int8), torch.ones(4), torch.ones(4, 3)
    off, ids = torch.zeros(5, dtype=torch.int64), torch.zeros(2, dtype=torch.int32)
    g = lambda t: t.clone().requires_grad_()        # noqa: E731
    t = int8.Int8Table(16)
    t._n = 70
    calls = [
        lambda f: int8.quantize_rows(f(x)), lambda f: int8.quantize_rows(f(x) * 2), lambda f: int8.quantize_rows(x, scales=f(sc)),
        lambda f: int8.dequantize_rows(c, f(sc)), lambda f: int8.dequantize_rows(c, sc, out=f(x)),
        lambda f: int8.adjust_scores(f(s)), lambda f: int8.adjust_scores(s, out=f(s)), lambda f: int8.adjust_scores(s, bias=f(b)),
        lambda f: int8.adjust_scores(s, (off, ids), f(pen)),
        lambda f: t.scores(f(x)), lambda f: t.scores(x, bias=f(b)), lambda f: t.scores((c, f(sc))), lambda f: t.scores(x, out=f(s)),
        lambda f: t.search(f(x), 3), lambda f: t.search(x, 3, bias=f(b)), lambda f: t.search((c, f(sc)), 3),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(NdbHipError, match="gradient") as e:
            call(g)
        assert e.value.code == _lib.ERR_INVALID, i
        assert code_of(lambda: call(lambda v: v)) == _lib.ERR_NODEVICE, i
        with torch.no_grad():
            assert code_of(lambda: call(g)) == _lib.ERR_NODEVICE, i
        assert code_of(lambda: call(lambda v: g(v).detach())) == _lib.ERR_NODEVICE, i
    # a table is a copy: its rows may come from a model that is being trained
    assert code_of(lambda: t.load(g(x))) == _lib.ERR_NODEVICE
    t.close()


@no_gpu
def test_what_is_written_into_is_a_new_version(on_cpu, monkeypatch):
    """a tensor that a call writes into, saved for some backward, is seen to have changed there"""
    monkeypatch.setattr(int8, "_call", lambda *a: None)
    x, s, sc = torch.ones(4, 16), torch.ones(4, 70), torch.ones(4)
    c = torch.ones(4, 16, dtype=torch.int8)
    t = int8.Int8Table(16)
    monkeypatch.setattr(t, "_n", 70)
    for call, outs in ((lambda: int8.quantize_rows(x, c, sc), (c, sc)), (lambda: int8.dequantize_rows(c, sc, out=x), (x,)), (lambda: t.scores(x, out=s), (s,))):
        before = [o._version for o in outs]
        call()
        assert [o._version for o in outs] == [v + 1 for v in before]
    with torch.inference_mode():
        still = torch.ones(4, 70)
    t.scores(x, out=still)                  # (these have no versions)
    t.close()


def test_assembly_that_writes_m0_says_so():
    """M0 is the compiler's too (LDS, relative moves, barriers' messages): inline assembly that writes it has to name it"""
    src = open(os.path.join(os.path.dirname(int8.__file__), "csrc", "ndbhip_int8.hip")).read()
    asm = [a for a in re.findall(r"asm volatile\((.*?)\);", src, re.S) if "m0" in a]
    assert len(asm) == 3
    for a in asm:
        assert re.search(r':\s*"m0"\s*$', a), a


@no_gpu
def test_adjust_refuses_a_result_that_overlaps_the_scores():
    """blocks of threads read and write at the same time: a shared element would be read before or after it is written.  Rows
    of one buffer that lie between each other are apart."""
    def call(nq, n, stride, at, ostride, dtype=0):
        s = 4 if dtype == 0 else 2
        return L.ndbhip_scores_adjust_device(1 << 20, dtype, nq, n, stride, None, None, 0, None, None, 0, None, 0, (1 << 20) + at * s, ostride)
    for dtype in (0, 1, 2):
        for args in ((4, 70, 70, 1, 70), (4, 70, 70, -1, 70), (4, 70, 70, 70, 70), (4, 70, 70, -210, 70), (4, 70, 140, 69, 140), (4, 70, 140, -69, 140),
                     (4, 70, 140, 70, 70), (4, 70, 70, 0, 71), (2, 70, 1000, 999, 70), (3, 70, 1000, 70, 965), (3, 70, 1000, 70, 900), (1, 70, 70, 69, 70), (1, 70, 70, -69, 70)):
            assert call(*args, dtype) == _lib.ERR_INVALID, args
            assert "overlap" in _lib.last_error() or "in place" in _lib.last_error()
        for args in ((4, 70, 70, 0, 70), (1, 70, 70, 0, 99), (4, 70, 70, 280, 70), (4, 70, 70, -280, 70), (4, 70, 140, 70, 140), (4, 70, 140, -70, 140),
                     (4, 70, 210, 140, 210), (2, 70, 1000, 70, 70), (3, 70, 1000, 70, 1100), (1, 70, 70, 70, 70), (1, 70, 70, -70, 70)):
            assert call(*args, dtype) == _lib.ERR_NODEVICE, args
    # (2^31 rows: neither a long search nor an overflow)
    assert call(2**31 - 1, 1, 2, 1, 2) == _lib.ERR_NODEVICE and call(2**31 - 1, 2, 2, 1, 2) == _lib.ERR_INVALID


@no_gpu
def test_counts_that_no_int_holds_are_refused(on_cpu):
    """a C int takes the low 32 bits of a number: 2^32 + 5 would be 5"""
    assert code_of(lambda: int8.Int8Table(2**32 + 16)) == _lib.ERR_INVALID
    t = int8.Int8Table(1)
    t._n = 70
    few, many = torch.ones(4, 1), torch.empty(2**32 + 4, 1, dtype=torch.float16)
    for k in (2**32 + 5, -2**32 + 5):
        assert code_of(lambda: t.search(few, k)) == _lib.ERR_INVALID
        assert code_of(lambda: t.search(few.numpy(), k)) == _lib.ERR_INVALID
    assert code_of(lambda: t.search(few, 5)) == _lib.ERR_NODEVICE
    assert code_of(lambda: t.search(many, 5)) == _lib.ERR_INVALID
    assert code_of(lambda: t.scores(many)) == _lib.ERR_INVALID
    t.close()


@no_gpu
def test_a_closed_table_refuses_and_stays_empty(on_cpu):
    import numpy as np
    t = int8.Int8Table(4)
    t._n = 70
    t.close()
    t.close()
    assert t.nrows == 0
    x = torch.ones(3, 4)
    for call in (lambda: t.load(x), lambda: t.load(np.ones((3, 4), np.float32)), lambda: t.search(x, 3), lambda: t.search(x.numpy(), 3),
                 lambda: t.scores(x), lambda: t.export()):
        assert code_of(call) in (_lib.ERR_INVALID, _lib.ERR_NODEVICE)       # (the calls on tensors ask for the device first)
        assert t.nrows == 0
