"""8-bit tables and scores over the C ABI (include/ndbhip.h, "8-bit tables and scores"): rows as signed bytes with one
scale each, the int8 product of a batch of queries with a table, penalties / biases / masks over scores, and the k best
rows of a table.

Everything here takes and returns torch tensors on the device the library runs on, is ordered on torch's current stream
and can be captured into a graph (the workspace of a call comes from torch's allocator; a graph owns its own).

No call has a gradient.  A tensor that requires one is refused while autograd follows it, so that none is lost unseen
(detach() it, or call under no_grad()); the rows a table is loaded with are copied, and may be such tensors.
"""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
import os
import sys
import threading

import numpy as np

from . import _lib
from ._lib import ERR_INVALID, ERR_NODEVICE, NdbHipError, check, ensure_init, lib

STREAM_LEGACY = 1           # NDBHIP_STREAM_LEGACY: the default stream, whose own handle is 0


def _bad(msg):
    return NdbHipError(ERR_INVALID, msg)


def _native(device):
    """csrc/ndb_torch.cpp: the calls whose host time is what they cost, in one crossing; tensors are to be on `device`"""
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "_ndb_torch.so")
    if not os.path.exists(path):
        raise NdbHipError(ERR_NODEVICE, f"{path} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'`")
    loader = importlib.machinery.ExtensionFileLoader("_ndb_torch", path)
    m = importlib.util.module_from_spec(importlib.util.spec_from_loader("_ndb_torch", loader))
    loader.exec_module(m)
    L = lib()
    m.setup(NdbHipError, str(device), *(C.cast(f, C.c_void_p).value for f in
                                        (L.ndbhip_swap_thread_stream, L.ndbhip_last_error, L.ndbhip_scores_adjust_device)))
    return m


class _Torch:
    """torch and what is asked of it at every call, looked up once (the package itself loads without torch)"""

    def __init__(self):
        import torch
        if not _lib._inited:
            ensure_init(torch.cuda.current_device())
        self.torch, self.Tensor = torch, torch.Tensor
        self.types = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.int8: 3}
        self.floats = (torch.float32, torch.float16, torch.bfloat16)
        self.f32, self.i8, self.i32, self.i64 = (torch.float32,), (torch.int8,), (torch.int32,), (torch.int64,)
        self.words = (torch.int32, torch.uint32) if hasattr(torch, "uint32") else (torch.int32,)
        self.increment_version = torch.autograd.graph.increment_version
        self.device = torch.device("cuda", _lib._device)
        self.lib = lib()
        # torch's own short cut to the current stream's handle (0.1 us, against 1.7 us through a Stream object)
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        index = _lib._device
        self.stream = (lambda: raw(index)) if raw else (lambda: torch.cuda.current_stream(index).cuda_stream)
        self.adjust = _native(self.device).adjust


_state = None


def _torch():
    global _state
    if _state is None:
        _state = _Torch()
    return _state


class _Previous(threading.local):
    def __init__(self):
        self.p = C.c_void_p()
        self.ref = C.byref(self.p)


_previous = _Previous()


def _call(fn, *args):
    """One call of the library on torch's current stream of the library's device; the thread's stream is as before afterwards."""
    T = _state
    swap = T.lib.ndbhip_swap_thread_stream
    ref = _previous.ref
    check(swap(T.stream() or STREAM_LEGACY, ref))
    prev = _previous.p.value
    try:
        rc = fn(*args)
        if rc:
            raise NdbHipError(rc, _lib.last_error())
    finally:
        swap(prev, ref)


def _tensor(t, name, dtypes, ndim, followed=False):
    """checks what every tensor argument has to be; followed: it may be one whose gradients autograd is to find"""
    T = _state
    if not isinstance(t, T.Tensor):
        raise _bad(f"{name} must be a torch tensor")
    if t.device != T.device:
        raise _bad(f"{name} is on {t.device}, the library on {T.device}")
    if t.dtype not in dtypes:
        raise _bad(f"{name} must be one of {[str(d) for d in dtypes]}, not {t.dtype}")
    if t.dim() != ndim and (type(ndim) is int or t.dim() not in ndim):
        raise _bad(f"{name} has {t.dim()} dimensions")
    if t.requires_grad and not followed and T.torch.is_grad_enabled():
        raise _bad(f"{name} requires a gradient, which this call has none of: detach() it, or call under no_grad()")
    return t


def _written(out):
    """the caller's own tensors that a call has written into: what autograd has saved of them is another version now"""
    for t in out:
        if not t.is_inference():
            _state.increment_version(t)


def _rows(t):
    """(tensor with neighbouring elements in a row and rows that do not overlap, elements from a row to the next)"""
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t, max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else t.shape[1]


def _out_rows(t, name):
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise _bad(f"{name} must have neighbouring elements in a row and rows that do not overlap")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _int(v, name):
    """a number for a C int, which would silently take the low 32 bits of a larger one"""
    v = int(v)
    if not -1 << 31 <= v < 1 << 31:
        raise _bad(f"{name} is {v}")
    return v


def _p(t):
    return None if t is None else t.data_ptr()


def quantize_rows(x, codes=None, scales=None):
    """Rows [n, dim] (float32, float16, bfloat16) -> (codes int8 [n, dim], scales float32 [n]); ndbhip_i8_quantize_device."""
    T = _torch()
    x, stride = _rows(_tensor(x, "x", T.floats, 2))
    n, dim = x.shape
    given = None
    if codes is not None or scales is not None:
        given = [t for t in (codes, scales) if t is not None]
    if codes is None:
        codes = T.torch.empty((n, dim), dtype=T.torch.int8, device=T.device)
        cstride = dim
    else:
        cstride = _out_rows(_tensor(codes, "codes", T.i8, 2), "codes")
    if scales is None:
        scales = T.torch.empty(n, dtype=T.torch.float32, device=T.device)
    else:
        _tensor(scales, "scales", T.f32, 1)
    if codes.shape != x.shape or scales.shape[0] != n or not scales.is_contiguous():
        raise _bad("codes must be [n, dim] and scales [n], contiguous")
    _call(T.lib.ndbhip_i8_quantize_device, _p(x), T.types[x.dtype], n, dim, stride, _p(codes), cstride, _p(scales))
    if given is not None:
        _written(given)
    return codes, scales


def dequantize_rows(codes, scales, dtype=None, out=None):
    """The values (codes int8 [n, dim], scales float32 [n]) stand for, as float32 (or `dtype`); ndbhip_i8_dequantize_device."""
    T = _torch()
    codes, stride = _rows(_tensor(codes, "codes", T.i8, 2))
    scales = _tensor(scales, "scales", T.f32, 1).contiguous()
    n, dim = codes.shape
    if scales.shape[0] != n:
        raise _bad("a scale for every row")
    given = out
    if out is None:
        out = T.torch.empty((n, dim), dtype=dtype or T.torch.float32, device=T.device)
    _tensor(out, "out", T.floats, 2)
    if out.shape != codes.shape or dtype not in (None, out.dtype):
        raise _bad("out must have the codes' shape and the dtype asked for")
    _call(T.lib.ndbhip_i8_dequantize_device, _p(codes), stride, _p(scales), n, dim, _p(out), T.types[out.dtype], _out_rows(out, "out"))
    if given is not None:
        _written((given,))
    return out


def _mask_arg(mask, nq, n):
    """(tensor, words from one query's mask to the next)"""
    if mask is None:
        return None, 0
    _tensor(mask, "mask", _state.words, (1, 2))
    m = mask[None] if mask.dim() == 1 else mask
    if m.shape[0] not in (1, nq) or m.shape[1] < (n + 31) // 32:
        raise _bad(f"mask must be [words] or [1 or {nq}, words] with at least {(n + 31) // 32} words of 32 rows")
    m, stride = _rows(m)
    return m, 0 if m.shape[0] == 1 else stride


def _bias_arg(bias, n):
    if bias is None:
        return None
    if _tensor(bias, "bias", _state.f32, 1).shape[0] != n:
        raise _bad(f"bias must be [{n}]")
    return bias.contiguous()


def adjust_scores(scores, seen=None, penalties=None, bias=None, mask=None, out=None):
    """Penalties, biases and masks over scores [nq, n] (float32, float16, bfloat16); ndbhip_scores_adjust_device.

    seen       (offsets int64 [nq + 1], ids int32 [...]): the ids query q has been given before, an id once for every time
    penalties  float32 [nq, 3] = repeat, presence, frequency of each query (with `seen`)
    bias       float32 [n] or [nq, n]
    mask       int32 words [ceil(n / 32)] or [nq, ceil(n / 32)], bit i % 32 of word i / 32: 0 = -inf
    out        another tensor of the scores' shape and type that shares no element with them, or `scores` itself (in place);
               None: a new one
    """
    T = _state or _torch()
    return T.adjust(T.stream() or STREAM_LEGACY, scores, seen, penalties, bias, mask, out)


class Int8Table:
    """A table of rows held as signed bytes with one fp32 scale each, resident in HBM (ndbhip_i8).

    Scores are inner products; rows and queries of norm 1 make them cosines, and a bias of -|x|^2 / 2 a row turns the
    order into the L2 one."""

    def __init__(self, dim: int, device: int | None = None):
        if device is None and not _lib._inited:
            # the device of the tensors it is going to meet, where the program has taken one up; else the process's own
            cuda = getattr(sys.modules.get("torch"), "cuda", None)
            if cuda is not None and cuda.is_initialized():
                device = cuda.current_device()
        ensure_init(device)
        self.dim = _int(dim, "dim")
        h = C.c_void_p()
        check(lib().ndbhip_i8_create(self.dim, C.byref(h)))
        self._h = h
        self._n = 0
        self._ws = {}            # (queries, k) -> bytes of workspace, for the rows there are

    def close(self):
        if getattr(self, "_h", None):
            check(lib().ndbhip_i8_destroy(self._h))
            self._h = None
            self._loaded()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def nrows(self) -> int:
        return self._n

    def _loaded(self):
        self._n = max(int(lib().ndbhip_i8_nrows(self._h)), 0)        # (-1: closed)
        self._ws.clear()

    def load(self, rows, scales=None):
        """The table's rows, in place of what it held: a numpy float32 array or a tensor [n, dim] of float32, float16,
        bfloat16 — quantised on the way — or of int8 with their scales [n]."""
        if isinstance(rows, np.ndarray):
            if scales is not None:
                raise _bad("scales go with int8 tensors")
            r = np.ascontiguousarray(rows, dtype=np.float32)
            if r.ndim != 2 or r.shape[1] != self.dim:
                raise _bad(f"rows must be [n, {self.dim}]")
            try:
                check(lib().ndbhip_i8_load(self._h, r.ctypes.data, r.shape[0]))
            finally:
                self._loaded()
            return
        T = _torch()
        r, stride = _rows(_tensor(rows, "rows", tuple(T.types), 2, followed=True))
        if r.shape[1] != self.dim:
            raise _bad(f"rows must be [n, {self.dim}]")
        if (r.dtype == T.torch.int8) != (scales is not None):
            raise _bad("scales go with int8 rows, and only with them")
        if scales is not None:
            scales = _tensor(scales, "scales", T.f32, 1, followed=True).contiguous()
            if scales.shape[0] != r.shape[0]:
                raise _bad("a scale for every row")
        try:
            _call(T.lib.ndbhip_i8_load_device, self._h, _p(r), T.types[r.dtype], r.shape[0], stride, _p(scales))
        finally:
            self._loaded()

    def export(self):
        """(codes int8 [n, dim], scales float32 [n])"""
        T = _torch()
        codes = T.torch.empty((self._n, self.dim), dtype=T.torch.int8, device=T.device)
        scales = T.torch.empty(self._n, dtype=T.torch.float32, device=T.device)
        _call(T.lib.ndbhip_i8_export_device, self._h, _p(codes), self.dim, _p(scales))
        return codes, scales

    def _queries(self, queries):
        T = _torch()
        scales = None
        if isinstance(queries, (tuple, list)):
            queries, scales = queries
            scales = _tensor(scales, "query scales", T.f32, 1).contiguous()
        q, stride = _rows(_tensor(queries, "queries", T.types, 2))
        if q.shape[1] != self.dim:
            raise _bad(f"queries must be [nq, {self.dim}]")
        if (q.dtype == T.torch.int8) != (scales is not None) or scales is not None and scales.shape[0] != q.shape[0]:
            raise _bad("int8 queries come as (codes [nq, dim], scales [nq]), others alone")
        if q.shape[0] >= 1 << 31:
            _int(q.shape[0], "the number of queries")
        return T, q, stride, scales

    def _workspace(self, T, nq, k):
        b = self._ws.get((nq, k))
        if b is None:
            if len(self._ws) >= 4096:
                self._ws.clear()
            out = C.c_size_t(0)
            check(lib().ndbhip_i8_workspace(self._h, nq, k, C.byref(out)))
            b = self._ws[(nq, k)] = out.value
        return T.torch.empty(b, dtype=T.torch.uint8, device=T.device), b

    def scores(self, queries, bias=None, dtype=None, out=None):
        """Every score: [nq, nrows] of float32 (or `dtype`, or into `out`); ndbhip_i8_product_device.  queries: [nq, dim] of
        float32, float16, bfloat16, or (codes, scales)."""
        T, q, stride, qs = self._queries(queries)
        nq, n = q.shape[0], self._n
        bias = _bias_arg(bias, n)
        given = out
        if out is None:
            out = T.torch.empty((nq, n), dtype=dtype or T.torch.float32, device=T.device)
        _tensor(out, "out", T.floats, 2)
        if out.shape != (nq, n) or dtype not in (None, out.dtype):
            raise _bad(f"out must be [{nq}, {n}] and of the dtype asked for")
        ostride = _out_rows(out, "out")
        ws, wsb = self._workspace(T, nq, 0)
        _call(T.lib.ndbhip_i8_product_device, self._h, _p(q), T.types[q.dtype], _p(qs), nq, stride, _p(bias), _p(out), T.types[out.dtype],
              ostride, _p(ws), wsb)
        if given is not None:
            _written((given,))
        return out

    def search(self, queries, k, bias=None, mask=None):
        """The k best rows of each query: (ids int64 [nq, k], scores float32 [nq, k]), higher scores first, equal ones by id; places
        no row fills hold -1 and -inf.  ndbhip_i8_search_device.  bias: float32 [nrows]; mask: as in adjust_scores.  numpy float32
        queries (and numpy bias, mask uint32 / int32) take the host form and return numpy arrays."""
        if isinstance(queries, np.ndarray):
            return self._search_host(queries, _int(k, "k"), bias, mask)
        T, q, stride, qs = self._queries(queries)
        nq, n, k = q.shape[0], self._n, int(k)
        if not 0 < k < 1 << 31:
            raise _bad(f"k is {k}")
        bias = _bias_arg(bias, n)
        mask, mstride = _mask_arg(mask, nq, n)
        ws, wsb = self._workspace(T, nq, k)
        ids = T.torch.empty((nq, k), dtype=T.torch.int64, device=T.device)
        scores = T.torch.empty((nq, k), dtype=T.torch.float32, device=T.device)
        _call(T.lib.ndbhip_i8_search_device, self._h, _p(q), T.types[q.dtype], _p(qs), nq, stride, _p(bias), _p(mask), mstride, k, _p(ids),
              _p(scores), _p(ws), wsb)
        return ids, scores

    def _search_host(self, queries, k, bias, mask):
        q = np.ascontiguousarray(queries, dtype=np.float32)
        n = self._n
        if q.ndim != 2 or q.shape[1] != self.dim:
            raise _bad(f"queries must be [nq, {self.dim}]")
        _int(q.shape[0], "the number of queries")
        p = lambda a: None if a is None else a.ctypes.data_as(C.c_void_p)     # noqa: E731
        if bias is not None:
            bias = np.ascontiguousarray(bias, dtype=np.float32)
            if bias.shape != (n,):
                raise _bad(f"bias must be [{n}]")
        mstride = 0
        if mask is not None:
            mask = np.ascontiguousarray(mask)
            if mask.dtype not in (np.uint32, np.int32):
                raise _bad("mask must be uint32 or int32 words")
            m = mask[None] if mask.ndim == 1 else mask
            if m.ndim != 2 or m.shape[0] not in (1, q.shape[0]) or m.shape[1] < (n + 31) // 32:
                raise _bad(f"mask must be [words] or [1 or {q.shape[0]}, words] with at least {(n + 31) // 32} words of 32 rows")
            mstride = 0 if m.shape[0] == 1 else m.shape[1]
        ids = np.empty((q.shape[0], max(k, 0)), dtype=np.int64)
        scores = np.empty((q.shape[0], max(k, 0)), dtype=np.float32)
        check(lib().ndbhip_i8_search(self._h, p(q), q.shape[0], p(bias), p(mask), mstride, k, p(ids), p(scores)))
        return ids, scores
