"""The way from Python and C to the 8-bit kernels, without a device: what the calls on torch tensors refuse."""
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
