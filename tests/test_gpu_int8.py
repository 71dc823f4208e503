"""8-bit tables and scores on the device (include/ndbhip.h) against a plain statement of the definitions.

The reference below runs on the CPU: integer sums in 64 bits, and the fp32 roundings the definition names one by one —
so bytes, scales, scores and ids are compared bit for bit, with no tolerance.  Where a value is compared with 64-bit
arithmetic instead, the tolerance counts the roundings (half a step each, finfo.eps / 2 relative)."""
import math

import numpy as np
import pytest
import torch

import neurondb_amd as nd
from neurondb_amd import _lib
from neurondb_amd._lib import NdbHipError

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TINY = 2.0 ** -100


# ------------------------------------------------------------------ the plain form

def quantise(x):
    x = x.detach().cpu().float()
    top = x.abs().amax(1) if x.shape[0] else torch.empty(0)
    finite = torch.isfinite(top)
    live = finite & (top >= TINY)
    t64 = torch.where(live, top, torch.ones_like(top)).double()
    scale, inv = (t64 / 127.0).float(), (127.0 / t64).float()
    codes = (torch.nan_to_num(x.double(), nan=0.0, posinf=0.0, neginf=0.0) * inv.double()[:, None]).round()
    codes = torch.where(live[:, None], codes, torch.zeros_like(codes)).to(torch.int8)
    scale = torch.where(live, scale, torch.where(finite, torch.zeros_like(scale), torch.full_like(scale, math.nan)))
    return codes, scale


def scores_of(qc, qs, rc, rs, bias=None):
    dot = (qc.double() @ rc.double().t()).float()       # exact: the sums stay far below 2^53
    s = (dot * rs[None]) * qs[:, None]
    return s if bias is None else s + bias.cpu()[None]


def unpack(mask, n):
    b = np.unpackbits(np.ascontiguousarray(mask.cpu().numpy()).view(np.uint8), axis=1, bitorder="little")
    return torch.from_numpy(b[:, :n].astype(bool))


def pack(bits):
    nq, n = bits.shape
    w = (n + 31) // 32
    full = np.zeros((nq, w * 32), dtype=np.uint8)
    full[:, :n] = bits
    return torch.from_numpy(np.packbits(full, axis=1, bitorder="little").view(np.int32).copy())


def best(s, k, mask=None):
    s = s.numpy().copy()
    if mask is not None:
        s[~np.broadcast_to(unpack(mask, s.shape[1]).numpy(), s.shape)] = -np.inf
    s[np.isnan(s)] = -np.inf
    s = s + np.float32(0)
    ids = np.argsort(-s, axis=1, kind="stable")[:, :k]
    v = np.take_along_axis(s, ids, 1)
    ids = np.where(v == -np.inf, -1, ids)
    pad = k - ids.shape[1]
    if pad > 0:
        ids = np.pad(ids, ((0, 0), (0, pad)), constant_values=-1)
        v = np.pad(v, ((0, 0), (0, pad)), constant_values=-np.inf)
    return torch.from_numpy(ids.astype(np.int64)), torch.from_numpy(v)


def same(a, b):
    """equal bit for bit, NaN with NaN"""
    a, b = a.detach().cpu(), b.detach().cpu()
    assert a.dtype == b.dtype and a.shape == b.shape, (a.dtype, b.dtype, a.shape, b.shape)
    if a.is_floating_point():
        w = torch.int32 if a.dtype == F32 else torch.int16
        x, y = (a + 0.0).view(w), (b + 0.0).view(w)
        ok = (x == y) | (a.isnan() & b.isnan())
    else:
        ok = a == b
    assert bool(ok.all()), (int((~ok).sum()), (~ok).nonzero()[:5], a[~ok][:5], b[~ok][:5])


def rand(seed, *shape, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ------------------------------------------------------------------ bytes and scales

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [1, 3, 4, 5, 8, 15, 17, 63, 64, 65, 128, 257, 300, 768, 1023, 1025, 2049, 4100, 32767])
def test_quantise(dim, dtype):
    n = 5 if dim > 5000 else 70
    x = rand(dim, n, dim, dtype=dtype)
    x[1] = 0
    x[2, dim // 2] = math.nan
    x[3, 0] = -math.inf
    codes, scales = nd.quantize_rows(x.cuda())
    c, s = quantise(x)
    same(codes, c)
    same(scales, s)
    same(nd.dequantize_rows(codes, scales), c.float() * s[:, None])
    assert bool(scales[2:4].isnan().all()) and not codes[1:4].any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [1, 3, 5, 8, 9, 31, 100, 128, 255, 256, 257, 300, 505, 512, 513, 1000, 1024, 1025, 1100])
def test_many_rows_there_and_back(dim, dtype):
    """as many rows as several are quantised a lane at, in a matrix with a border that stays as it is"""
    n = 6 * 256 * 256 // min(64, 1 << max(0, (dim * (4 if dtype == F32 else 2) - 1) // 16).bit_length()) + 3
    x = rand(dim, n, dim, dtype=dtype)
    x[n // 2] = 0
    x[n - 1, dim // 2] = math.nan
    c = torch.full((n + 9, dim + 5), 77, dtype=torch.int8, device="cuda")
    s = torch.full((n + 9,), 77.0, device="cuda")
    nd.quantize_rows(x.cuda(), c[:n, 2:dim + 2], s[:n])
    rc, rs = quantise(x)
    same(c[:n, 2:dim + 2], rc)
    same(s[:n], rs)
    out = torch.full((n + 9, dim + 3), 77.0, dtype=dtype, device="cuda")
    nd.dequantize_rows(c[:n, 2:dim + 2], s[:n], out=out[:n, 1:dim + 1])
    same(out[:n, 1:dim + 1], (rc.float() * rs[:, None]).to(dtype))
    assert bool((c[n:] == 77).all()) and bool((c[:, :2] == 77).all()) and bool((c[:, dim + 2:] == 77).all())
    assert bool((s[n:] == 77).all())
    assert bool((out[n:] == 77).all()) and bool((out[:, :1] == 77).all()) and bool((out[:, dim + 1:] == 77).all())


def test_quantise_halves_tiny_and_huge_values():
    half = torch.arange(-127, 128, dtype=F32)[None].repeat(2, 1)
    half[0, 1:-1] += 0.5                    # top = 127, inv = 1: every product is a half, ties to even
    half[1, 1:-1] += 0.49999997
    x = torch.zeros(8, 255)
    x[:2] = half
    x[2] = half[0] * 2.0 ** -90
    x[3] = 2.0 ** -101                      # below the smallest row that is not zeros
    x[4] = 2.0 ** -100
    x[5, 7] = torch.finfo(F32).max
    x[6] = torch.finfo(F32).tiny / 8        # denormal
    x[7] = half[0] * 2.0 ** 100
    codes, scales = nd.quantize_rows(x.cuda())
    c, s = quantise(x)
    same(codes, c)
    same(scales, s)
    assert float(s[3]) == 0.0 and float(s[4]) > 0.0


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_quantise_strides_and_alignment(dtype):
    wide = rand(5, 40, 400, dtype=dtype)
    d = wide.cuda()
    for lo, dim, step in [(0, 256, 1), (1, 255, 1), (3, 128, 2), (0, 399, 3)]:
        c, s = quantise(wide[::step, lo:lo + dim])
        codes = torch.full((c.shape[0], 411), 99, dtype=torch.int8, device="cuda")
        got, scales = nd.quantize_rows(d[::step, lo:lo + dim], codes=codes[:, 5:5 + dim])
        same(got, c)
        same(scales, s)
        assert bool((codes[:, :5] == 99).all()) and bool((codes[:, 5 + dim:] == 99).all())
        for out_t in (F32, F16, BF16):
            out = torch.full((c.shape[0], 411), 7.0, dtype=out_t, device="cuda")
            same(nd.dequantize_rows(got, scales, out=out[:, 3:3 + dim]), (c.float() * s[:, None]).to(out_t))
            assert bool((out[:, :3] == 7).all()) and bool((out[:, 3 + dim:] == 7).all())
    same(nd.quantize_rows(d.t())[0], quantise(wide.t())[0])     # columns as rows


def test_values_are_within_half_a_step():
    """|x - byte * scale|: half a byte's step for the rounding, and half a step of fp32 for each of inv, scale and the
    product (relative to at most 127.5 scale)"""
    x = rand(11, 64, 768)
    codes, scales = nd.quantize_rows(x.cuda())
    v = nd.dequantize_rows(codes, scales).cpu().double()
    s = scales.cpu().double()[:, None]
    e = 2.0 ** -24
    assert bool(((x.double() - v).abs() <= 0.5 * s + 127.5 * s * 3 * e).all())


@pytest.mark.parametrize("n,dim", [(1, 1), (31, 5), (32, 64), (33, 65), (257, 100), (1000, 768)])
def test_table_holds_the_bytes_it_was_given(n, dim):
    x = rand(n + dim, n, dim)
    c, s = quantise(x)
    for load in (lambda t: t.load(x.numpy()), lambda t: t.load(x.cuda()), lambda t: t.load(c.cuda(), s.cuda()),
                 lambda t: t.load(torch.cat([c, c], 1)[:, dim:].cuda(), s.cuda())):
        t = nd.Int8Table(dim)
        load(t)
        assert t.nrows == n
        codes, scales = t.export()
        same(codes, c)
        same(scales, s)
    t.load(x[:0].cuda())
    assert t.nrows == 0


# ------------------------------------------------------------------ the product

@pytest.mark.parametrize("nq,n,dim", [(1, 1, 1), (1, 33, 17), (2, 1000, 128), (5, 31, 64), (31, 257, 300), (32, 96, 65), (33, 4097, 100),
                                      (64, 512, 768), (65, 300, 1536), (100, 5000, 96), (130, 777, 63), (200, 1025, 320), (257, 2000, 129),
                                      (300, 255, 2048), (600, 513, 40)])
@pytest.mark.parametrize("out_t", [F32, F16, BF16])
def test_product(nq, n, dim, out_t):
    rows, q = rand(n, n, dim), rand(nq + 7, nq, dim)
    t = nd.Int8Table(dim)
    t.load(rows.cuda())
    bias = rand(3, n)
    ref = scores_of(*quantise(q), *quantise(rows))
    same(t.scores(q.cuda(), dtype=out_t), ref.to(out_t))
    same(t.scores(q.cuda(), dtype=out_t, bias=bias.cuda()), (ref + bias).to(out_t))


@pytest.mark.parametrize("nq", [3, 70, 300])
@pytest.mark.parametrize("q_t", [F32, F16, BF16, torch.int8])
def test_product_query_types_strides_and_what_lies_beside_the_scores(nq, q_t):
    n, dim = 611, 200
    rows, q = rand(1, n, dim), rand(2, nq, dim + 9, dtype=F32 if q_t == torch.int8 else q_t)
    t = nd.Int8Table(dim)
    t.load(rows.cuda())
    qv = q[:, 3:3 + dim]
    c, s = quantise(qv)
    given = (c.cuda(), s.cuda()) if q_t == torch.int8 else q.cuda()[:, 3:3 + dim]
    ref = scores_of(c, s, *quantise(rows))
    for off, width in [(0, 611), (1, 640), (4, 616), (0, 700)]:
        for out_t in (F32, BF16):
            out = torch.full((nq, width + off), 55.0, dtype=out_t, device="cuda")
            same(t.scores(given, out=out[:, off:off + n]), ref.to(out_t))
            assert bool((out[:, :off] == 55).all()) and bool((out[:, off + n:] == 55).all())


def test_product_against_64_bits():
    """three roundings to fp32 (the sum, and two products), half a step each"""
    rows, q = rand(1, 500, 1000), rand(2, 90, 1000)
    t = nd.Int8Table(1000)
    t.load(rows.cuda())
    (qc, qs), (rc, rs) = quantise(q), quantise(rows)
    exact = (qc.double() @ rc.double().t()) * rs.double()[None] * qs.double()[:, None]
    got = t.scores(q.cuda()).cpu().double()
    e = 2.0 ** -24
    assert bool(((got - exact).abs() <= exact.abs() * ((1 + e) ** 3 - 1)).all())


@pytest.mark.parametrize("nq", [2, 80])
def test_product_largest_sums(nq):
    """bytes of +-127 throughout: the longest rows' sums, past the integers fp32 holds"""
    dim = 32767
    c = torch.full((40, dim), 127, dtype=torch.int8)
    c[1] = -127
    c[2, ::2] = -127
    s = torch.linspace(0.5, 2, 40)
    qc = torch.full((nq, dim), 127, dtype=torch.int8)
    qc[1] = -128                            # (not a byte the quantiser makes, but a caller's bytes are the caller's)
    qs = torch.linspace(1, 3, nq)
    t = nd.Int8Table(dim)
    t.load(c.cuda(), s.cuda())
    same(t.scores((qc.cuda(), qs.cuda())), scores_of(qc, qs, c, s))


def test_non_finite_rows_and_queries():
    rows, q = rand(1, 100, 64), rand(2, 70, 64)
    rows[5, 1] = math.nan
    rows[40, 2] = math.inf
    q[1, 0] = -math.inf
    q[2] = 0
    t = nd.Int8Table(64)
    t.load(rows.cuda())
    ref = scores_of(*quantise(q), *quantise(rows))
    got = t.scores(q.cuda())
    same(got, ref)
    assert bool(got[:, [5, 40]].isnan().all()) and bool(got[1].isnan().all())
    ids, sc = t.search(q.cuda(), 100)
    same(ids, best(ref, 100)[0])
    same(sc, best(ref, 100)[1])
    assert bool((ids[1] == -1).all()) and int((ids[0] == -1).sum()) == 2


@pytest.mark.parametrize("nq,n,dim", [(130, 400_003, 520), (31, 1_700_001, 513), (280, 400_003, 520), (1000, 60_001, 1000)])
@pytest.mark.parametrize("out_t", [F32, BF16])
def test_scores_that_no_cache_holds(nq, n, dim, out_t):
    """large matrices are stored another way: the same scores as in pieces, and nothing beside them"""
    t = nd.Int8Table(dim)
    t.load(torch.randn(n, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(n)))
    q, bias = rand(nq, nq, dim).cuda(), rand(3, n).cuda()
    out = torch.full((nq, n + 5), 9.0, dtype=out_t, device="cuda")
    t.scores(q, bias=bias, out=out[:, 2:2 + n])
    for at in range(0, nq, 13):
        same(out[at:at + 13, 2:2 + n], t.scores(q[at:at + 13], bias=bias, dtype=out_t))
    assert bool((out[:, :2] == 9).all()) and bool((out[:, 2 + n:] == 9).all())
    codes, scales = t.export()
    rows = torch.tensor([0, 77, n // 2, n - 1])
    ref = scores_of(*quantise(q), codes[rows.cuda()].cpu(), scales[rows.cuda()].cpu(), bias[rows.cuda()].cpu())
    same(out[:, 2:2 + n][:, rows.cuda()], ref.to(out_t))


def test_more_scores_than_32_bits_count():
    n, nq, dim = 1_000_000, 2200, 16
    rows, q = torch.randn(n, dim, device="cuda"), torch.randn(nq, dim, device="cuda")
    t = nd.Int8Table(dim)
    t.load(rows)
    out = t.scores(q, dtype=F16)
    assert out.numel() > 2 ** 31
    for i in (0, 1, 1099, 2147, 2148, nq - 1):
        at = torch.tensor([0, 5, 483_648, n // 2, n - 1])
        ref = scores_of(*quantise(q[i:i + 1]), *quantise(rows[at.cuda()])).half()
        same(out[i:i + 1, at.cuda()], ref)


# ------------------------------------------------------------------ the k best

@pytest.mark.parametrize("nq,n,dim,k", [(1, 1, 1, 1), (1, 5, 3, 9), (1, 1000, 128, 10), (1, 40_000, 64, 1), (3, 31, 64, 31), (7, 33, 65, 40),
                                        (32, 5000, 100, 10), (33, 5000, 100, 64), (64, 20_000, 48, 100), (65, 3000, 768, 10), (90, 9000, 33, 1024),
                                        (129, 2049, 200, 7), (260, 10_000, 96, 33), (520, 4100, 64, 128), (5, 100_000, 32, 300)])
@pytest.mark.parametrize("what", ["plain", "bias", "mask1", "mask", "all"])
def test_search(nq, n, dim, k, what):
    rows, q = rand(n + k, n, dim), rand(nq, nq, dim)
    rows[:: max(1, n // 7)] = rows[n // 2].clone()      # equal scores
    t = nd.Int8Table(dim)
    t.load(rows.cuda())
    bias = rand(9, n) if what in ("bias", "all") else None
    if bias is not None:
        bias[n // 3] = math.nan
        bias[n // 4] = -math.inf
    mask = None
    if what in ("mask", "mask1", "all"):
        g = np.random.default_rng(n)
        bits = g.random((1 if what == "mask1" else nq, n)) < 0.3
        if what != "mask1":
            bits[nq // 2] = False                       # nothing left
        mask = pack(bits)
    ref = best(scores_of(*quantise(q), *quantise(rows), bias=bias), k, mask)
    ids, sc = t.search(q.cuda(), k, bias=None if bias is None else bias.cuda(), mask=None if mask is None else mask.cuda())
    same(ids, ref[0])
    same(sc, ref[1])


@pytest.mark.parametrize("nq,n,dim,k", [(130, 60_001, 33, 10), (65, 100_003, 64, 3), (200, 70_001, 40, 129), (384, 40_007, 130, 20), (700, 33_000, 8, 5),
                                        (257, 9000, 2049, 12)])
@pytest.mark.parametrize("what", ["plain", "bias", "mask1", "mask", "all"])
def test_search_and_product_in_many_tiles(nq, n, dim, k, what):
    """batches whose product takes LDS tiles, narrow and wide ones, with rows, queries and dimensions that fill none"""
    rows, q = rand(n + k, n, dim), rand(nq, nq, dim)
    rows[:: n // 9] = rows[n // 2].clone()
    t = nd.Int8Table(dim)
    t.load(rows.cuda())
    bias = rand(9, n) if what in ("bias", "all") else None
    mask = None
    if what in ("mask", "mask1", "all"):
        bits = np.random.default_rng(n).random((1 if what == "mask1" else nq, n)) < 0.05
        bits[-1, : n // 2] = False
        if what != "mask1":
            bits[nq // 2] = False
        mask = pack(bits)
    s = scores_of(*quantise(q), *quantise(rows), bias=bias)
    if mask is None:
        for out_t in (F32, F16):
            same(t.scores(q.cuda(), bias=None if bias is None else bias.cuda(), dtype=out_t), s.to(out_t))
    at = [0, 1, nq // 2, nq - 2, nq - 1]
    ref = best(s[at], k, mask if what in ("plain", "bias", "mask1") else mask[at])
    ids, sc = t.search(q.cuda(), k, bias=None if bias is None else bias.cuda(), mask=None if mask is None else mask.cuda())
    same(ids[at], ref[0])
    same(sc[at], ref[1])
    # every query: the k best, recomputed from the scores on the device
    if mask is not None:
        s = s.masked_fill(~unpack(mask, n), -math.inf)
    same(sc, s.cuda().topk(k, 1).values)


@pytest.mark.parametrize("nq,n,k", [(1, 70_000, 10), (4, 3000, 1024), (70, 9000, 50), (300, 3000, 200)])
def test_search_where_every_score_is_equal(nq, n, k):
    for rows in (torch.ones(n, 32), torch.zeros(n, 32), torch.ones(n, 32) * (torch.arange(n) % 2 * 2 - 1)[:, None]):
        t = nd.Int8Table(32)
        t.load(rows.cuda())
        q = torch.ones(nq, 32)
        q[nq // 2] = 0
        ids, sc = t.search(q.cuda(), k)
        ref = best(scores_of(*quantise(q), *quantise(rows)), k)
        same(ids, ref[0])
        same(sc, ref[1])


def test_search_scales_of_zero_and_infinite_products():
    """row scales that overflow a product, query scales of 0, below 0 and NaN: what the definition's roundings say"""
    n = 200
    rc = torch.randint(-127, 128, (n, 64), dtype=torch.int8, generator=torch.Generator().manual_seed(1))
    rs = torch.ones(n)
    rs[::3] = 3e38
    rs[1::7] = 0.0
    rs[2::11] = -2.0
    qc = torch.randint(-127, 128, (80, 64), dtype=torch.int8, generator=torch.Generator().manual_seed(2))
    qs = torch.rand(80, generator=torch.Generator().manual_seed(3))
    qs[1], qs[2], qs[3], qs[4] = 0.0, -1.0, math.nan, math.inf
    t = nd.Int8Table(64)
    t.load(rc.cuda(), rs.cuda())
    for nq in (6, 80):
        for bias in (None, rand(4, n)):
            s = scores_of(qc[:nq], qs[:nq], rc, rs, bias)
            same(t.scores((qc[:nq].cuda(), qs[:nq].cuda()), bias=None if bias is None else bias.cuda()), s)
            for k in (3, 200):
                ids, sc = t.search((qc[:nq].cuda(), qs[:nq].cuda()), k, bias=None if bias is None else bias.cuda())
                same(ids, best(s, k)[0])
                same(sc, best(s, k)[1])


@pytest.mark.parametrize("nq,n,k", [(1, 500, 7), (40, 3000, 300), (300, 60_000, 20)])
def test_search_takes_minus_zero_and_zero_for_equal(nq, n, k):
    c = torch.zeros(n, 32, dtype=torch.int8)
    s = torch.ones(n)
    s[::2] = -1.0
    t = nd.Int8Table(32)
    t.load(c.cuda(), s.cuda())
    ids, sc = t.search(torch.ones(nq, 32, device="cuda"), k)
    same(ids, torch.arange(k)[None].repeat(nq, 1))
    assert not sc.any() and not torch.signbit(sc).any()


def test_search_of_an_empty_table_and_of_no_queries():
    t = nd.Int8Table(8)
    ids, sc = t.search(torch.ones(3, 8, device="cuda"), 4)
    assert bool((ids == -1).all()) and bool((sc == -math.inf).all())
    assert t.scores(torch.ones(3, 8, device="cuda")).shape == (3, 0)
    t.load(torch.ones(5, 8).cuda())
    assert t.search(torch.ones(0, 8, device="cuda"), 4)[0].shape == (0, 4)
    assert t.scores(torch.ones(0, 8, device="cuda")).shape == (0, 5)


def test_search_of_an_empty_table_with_more_places_than_a_grid_has_threads():
    nq, k = 2**22 + 1, 1024
    ids, sc = nd.Int8Table(1).search(torch.zeros(nq, 1, device="cuda"), k)
    for q in range(0, nq, 1 << 18):
        assert bool((ids[q:q + (1 << 18)] == -1).all()) and bool((sc[q:q + (1 << 18)] == -math.inf).all()), q
    del ids, sc
    torch.cuda.empty_cache()


def test_search_more_queries_than_one_pass_takes():
    n, dim, nq = 300, 32, 9001
    rows, q = rand(1, n, dim), rand(2, nq, dim)
    mask = pack(np.random.default_rng(0).random((nq, n)) < 0.5)
    t = nd.Int8Table(dim)
    t.load(rows.cuda())
    s = scores_of(*quantise(q), *quantise(rows))
    ids, sc = t.search(q.cuda(), 5, mask=mask.cuda())
    same(ids, best(s, 5, mask)[0])
    same(sc, best(s, 5, mask)[1])
    same(t.scores(q.cuda()), s)


def test_search_of_host_arrays():
    rows, q = rand(1, 3000, 96), rand(2, 9, 96)
    t = nd.Int8Table(96)
    t.load(rows.numpy())
    bias = rand(4, 3000)
    s = scores_of(*quantise(q), *quantise(rows), bias=bias)
    for mask in (None, pack(np.random.default_rng(0).random((9, 3000)) < 0.5), pack(np.random.default_rng(0).random((1, 3000)) < 0.5)):
        ids, sc = t.search(q.numpy(), 12, bias=bias.numpy(), mask=None if mask is None else mask.numpy())
        same(torch.from_numpy(ids), best(s, 12, mask)[0])
        same(torch.from_numpy(sc), best(s, 12, mask)[1])


def test_table_beyond_four_gigabytes():
    n, dim = 6_000_000, 768
    t = nd.Int8Table(dim)
    rows = torch.empty(n, dim, dtype=BF16, device="cuda")
    for at in range(0, n, 1_000_000):
        rows[at:at + 1_000_000] = torch.randn(1_000_000, dim, device="cuda")
    t.load(rows)
    want = torch.tensor([0, 31, 2_796_203, 5_592_406, 5_999_999], device="cuda")    # around 2^31 and 2^32 bytes
    q = rows[want].float()
    ids, sc = t.search(q, 2)
    same(ids[:, 0], want)
    same(sc[:, :1], scores_of(*quantise(q), *quantise(q)).diagonal()[:, None].contiguous())
    ids, _ = t.search(q.repeat(20, 1), 1)
    same(ids[:, 0], want.repeat(20))


# ------------------------------------------------------------------ penalties, biases, masks

def adjust(s, off, ids, pen, bias, mask):
    t = s.cpu().float().clone()
    for q in range(t.shape[0]):
        if off is not None:
            at = ids[int(off[q]):int(off[q + 1])]
            at = at[(at >= 0) & (at < t.shape[1])].long()
            c = torch.bincount(at, minlength=t.shape[1]).float()
            r, p, f = pen[q]
            t[q] = torch.where(c > 0, torch.where(t[q] > 0, t[q] / r, t[q] * r) - (p + c * f), t[q])
    if bias is not None:
        t = t + bias
    if mask is not None:
        t = t.masked_fill(~unpack(mask, t.shape[1]), -math.inf)
    return t.to(s.dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("nq,n,seen", [(1, 1, 3), (1, 31, 0), (2, 33, 5), (3, 2047, 100), (5, 2049, 1000), (2, 10_001, 40), (70, 130_000, 50),
                                       (3, 20_000, 30_000)])
def test_adjust(nq, n, seen, dtype):
    g = torch.Generator().manual_seed(n)
    s = (4 * torch.randn(nq, n, generator=g)).to(dtype)
    s[0, 0] = math.inf
    s[-1, n // 2] = -math.inf
    s[0, n - 1] = math.nan
    # lists of different lengths, the first query's empty; ids repeat, some are nobody's
    lens = torch.randint(0, seen + 1, (nq,), generator=g)
    lens[0] = 0 if nq > 1 else seen
    off = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])
    ids = torch.randint(-2, n + 2, (int(off[-1]),), generator=g).int()
    ids[::3] = n // 2
    pen = torch.rand(nq, 3, generator=g) + torch.tensor([0.5, -0.5, -0.5])
    bias, biasq = torch.randn(n, generator=g), torch.randn(nq, n, generator=g)
    bits = torch.rand(nq, n, generator=g).numpy() < 0.5
    bits[nq // 2] = False
    maskq, mask1 = pack(bits), pack(bits[:1])
    d = s.cuda()
    sn, pn = (off.cuda(), ids.cuda()), pen.cuda()
    same(nd.adjust_scores(d, sn, pn), adjust(s, off, ids, pen, None, None))
    same(nd.adjust_scores(d, bias=bias.cuda()), adjust(s, None, None, None, bias, None))
    same(nd.adjust_scores(d, mask=mask1[0].cuda()), adjust(s, None, None, None, None, mask1))
    same(nd.adjust_scores(d, sn, pn, biasq.cuda(), maskq.cuda()), adjust(s, off, ids, pen, biasq, maskq))
    same(d, s)
    got = nd.adjust_scores(d, sn, pn, bias.cuda(), maskq.cuda(), out=d)
    assert got.data_ptr() == d.data_ptr()
    same(d, adjust(s, off, ids, pen, bias, maskq))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_adjust_strides(dtype):
    s = rand(1, 9, 333, dtype=dtype)
    wide = torch.full((9, 400), 3.0, dtype=dtype, device="cuda")
    wide[:, 5:338] = s.cuda()
    mask = pack(np.random.default_rng(1).random((9, 333)) < 0.5)
    wmask = torch.zeros(9, 20, dtype=torch.int32)
    wmask[:, :11] = mask
    bias = rand(2, 9, 500)
    ref = adjust(s, None, None, None, bias[:, 7:340], mask)
    out = torch.full((9, 351), 5.0, dtype=dtype, device="cuda")
    same(nd.adjust_scores(wide[:, 5:338], bias=bias.cuda()[:, 7:340], mask=wmask.cuda(), out=out[:, 2:335]), ref)
    assert bool((out[:, :2] == 5).all()) and bool((out[:, 335:] == 5).all())
    nd.adjust_scores(wide[:, 5:338], bias=bias.cuda()[:, 7:340], mask=wmask.cuda(), out=wide[:, 5:338])
    same(wide[:, 5:338], ref)
    assert bool((wide[:, :5] == 3).all()) and bool((wide[:, 338:] == 3).all())


def test_adjust_offsets_outside_the_ids():
    """offsets that run out of the list, or backwards, count what there is"""
    s = rand(1, 4, 50)
    ids = torch.tensor([1, 2, 2, 3], dtype=torch.int32)
    pen = torch.tensor([[2.0, 0.5, 0.25]]).repeat(4, 1)
    off = torch.tensor([-7, 2, 1, 1 << 40, 5])
    got = nd.adjust_scores(s.cuda(), (off.cuda(), ids.cuda()), pen.cuda())
    same(got[:1], adjust(s[:1], torch.tensor([0, 2]), ids, pen, None, None))
    same(got[1:2], s[1:2])
    same(got[2:3], adjust(s[2:3], torch.tensor([1, 4]), ids, pen, None, None))
    same(got[3:], s[3:])


# ------------------------------------------------------------------ together, streams, graphs

def test_adjust_as_many_queries_as_an_int_counts():
    n = 2**31 - 1
    s = torch.zeros(n + 64, 1, dtype=F16, device="cuda")
    nd.adjust_scores(s[:n], bias=torch.ones(1, device="cuda"), out=s[:n])
    for q in range(0, n, 1 << 28):
        assert bool((s[q:min(q + (1 << 28), n)] == 1).all()), q
    assert not bool(s[n:].any())


def test_scores_adjusted_and_ranked_are_the_search():
    """the way a session is served: the product, the rows it has been given pushed down, a filter — and, where there is only
    a bias and a filter, the search that does it in one call"""
    n, dim, nq, k = 5000, 96, 40, 20
    rows, q, bias = rand(1, n, dim).cuda(), rand(2, nq, dim).cuda(), rand(3, n).cuda()
    mask = pack(np.random.default_rng(5).random((nq, n)) < 0.2).cuda()
    codes, scales = nd.quantize_rows(rows)
    t = nd.Int8Table(dim)
    t.load(codes, scales)
    s = t.scores(q)
    a = nd.adjust_scores(s, bias=bias, mask=mask)
    ids, sc = t.search(q, k, bias=bias, mask=mask)
    same(ids, best(a.cpu(), k)[0])
    same(sc, torch.gather(a, 1, ids))
    # what was returned goes below everything else in the next round
    off = torch.arange(nq + 1, device="cuda") * k
    pen = torch.tensor([[1.0, 1e6, 0.0]], device="cuda").repeat(nq, 1)
    b = nd.adjust_scores(a, (off, ids.int().reshape(-1).contiguous()), pen)
    nxt = b.topk(k, 1).indices
    assert not (nxt[:, :, None] == ids[:, None, :]).any()


def _everything(t, q, bias, mask, off, ids, pen):
    c, s = nd.quantize_rows(q)
    a = t.scores((c, s), bias=bias)
    b = nd.adjust_scores(a, (off, ids), pen, mask=mask)
    i, v = t.search(q, 7, bias=bias, mask=mask)
    return nd.dequantize_rows(c, s), a, b, i, v


@pytest.mark.parametrize("nq", [1, 5, 100, 300])
def test_captured_and_replayed(nq):
    n, dim = 4000, 128
    rows = rand(1, n, dim).cuda()
    t = nd.Int8Table(dim)
    t.load(rows)
    bias = rand(3, n).cuda()
    off = (torch.arange(nq + 1, device="cuda") * 6)
    pen = torch.rand(nq, 3, device="cuda") + 0.5
    graphs = []
    for g in range(2):                      # two graphs of one table, each with buffers of its own
        q = rand(10 + g, nq, dim).cuda()
        mask = pack(np.random.default_rng(g).random((nq, n)) < 0.5).cuda()
        ids = torch.randint(0, n, (6 * nq,), device="cuda").int()
        _everything(t, q, bias, mask, off, ids, pen)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _everything(t, q, bias, mask, off, ids, pen)
        graphs.append((graph, q, mask, ids, out))
    side = torch.cuda.Stream()
    for rep in range(4):
        for g, (graph, q, mask, ids, out) in enumerate(graphs):
            q.copy_(rand(100 + 10 * rep + g, nq, dim))
            ids.copy_(torch.randint(0, n, (6 * nq,)))
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(side):       # at the same time
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for graph, q, mask, ids, out in graphs:
            for x, y in zip(out, _everything(t, q, bias, mask, off, ids, pen)):
                same(x, y)


def test_streams_of_torch_and_of_the_library():
    """calls follow torch's current stream — a side stream, the default stream — and leave the thread's stream as it was"""
    n, dim = 60_000, 256
    t = nd.Int8Table(dim)
    t.load(rand(1, n, dim).cuda())
    q = rand(2, 64, dim)
    qd = q.cuda()
    ids0, sc0 = t.search(qd, 5)
    side = torch.cuda.Stream()
    for s in (side, torch.cuda.default_stream()):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            late = torch.zeros(64, dim, device="cuda")
            torch.cuda._sleep(20_000_000)
            late.copy_(qd)                  # the call must wait for this
            ids, sc = t.search(late, 5)
            c, _ = nd.quantize_rows(late)
            late.zero_()                    # and this must wait for the call
        torch.cuda.current_stream().wait_stream(s)
        same(ids, ids0)
        same(sc, sc0)
        same(c, quantise(q)[0])
    import ctypes as C
    cur = C.c_void_p()
    _lib.check(_lib.lib().ndbhip_swap_thread_stream(None, C.byref(cur)))
    assert not cur.value


def test_two_threads_search_one_table_at_the_same_time():
    import threading
    n, dim = 50_000, 128
    t = nd.Int8Table(dim)
    t.load(rand(1, n, dim).cuda())
    qs = [rand(2, 300, dim).cuda(), rand(3, 7, dim).cuda()]
    refs = [t.search(q, 20) for q in qs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    ids, sc = t.search(qs[i], 20)
                    if not (torch.equal(ids, refs[i][0]) and torch.equal(sc, refs[i][1])):
                        bad.append(i)
        except Exception as e:          # noqa: BLE001 (reported below)
            bad.append(e)

    th = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [x.start() for x in th]
    [x.join() for x in th]
    assert not bad


def test_results_do_not_change_from_call_to_call():
    t = nd.Int8Table(64)
    t.load(rand(1, 30_000, 64).cuda())
    q = rand(2, 200, 64).cuda()
    first = t.search(q, 50)
    for _ in range(5):
        t.search(rand(3, 10, 64).cuda(), 3)
        again = t.search(q, 50)
        same(first[0], again[0])
        same(first[1], again[1])


# ------------------------------------------------------------------ refusals

def test_refusals():
    dev = "cuda"
    t = nd.Int8Table(16)
    t.load(torch.ones(70, 16, device=dev))
    q = torch.ones(4, 16, device=dev)
    s = torch.ones(4, 70, device=dev)
    w = torch.zeros(4, 3, dtype=torch.int32, device=dev)
    off, ids, pen = torch.zeros(5, dtype=torch.int64, device=dev), torch.zeros(2, dtype=torch.int32, device=dev), torch.ones(4, 3, device=dev)
    calls = [
        lambda: nd.Int8Table(0), lambda: nd.Int8Table(32768),
        lambda: t.load(torch.ones(3, 15, device=dev)), lambda: t.load(torch.ones(3, 16)), lambda: t.load(np.ones((3, 15), np.float32)),
        lambda: t.load(torch.ones(3, 16, dtype=torch.int8, device=dev)), lambda: t.load(torch.ones(3, 16, device=dev), torch.ones(3, device=dev)),
        lambda: t.load(torch.ones(3, 16, dtype=torch.float64, device=dev)),
        lambda: t.scores(torch.ones(4, 15, device=dev)), lambda: t.scores(q.cpu()), lambda: t.scores(q, bias=torch.ones(69, device=dev)),
        lambda: t.scores(q, out=torch.ones(4, 71, device=dev)), lambda: t.scores(q, out=torch.ones(70, 4, device=dev).t()),
        lambda: t.scores(q, dtype=torch.float64), lambda: t.scores((q, torch.ones(4, device=dev))),
        lambda: t.scores((q.to(torch.int8), torch.ones(3, device=dev))), lambda: t.scores(q.to(torch.int8)),
        lambda: t.search(q, 0), lambda: t.search(q, 1025), lambda: t.search(q, 3, mask=w[:, :2]), lambda: t.search(q, 3, mask=w[:3]),
        lambda: t.search(q, 3, mask=w.float()), lambda: t.search(q, 3, bias=torch.ones(4, 70, device=dev)),
        lambda: t.search(np.ones((4, 15), np.float32), 3), lambda: t.search(np.ones((4, 16), np.float32), 0),
        lambda: t.search(np.ones((4, 16), np.float32), 3, mask=np.zeros((4, 2), np.int32)),
        lambda: nd.quantize_rows(torch.ones(4, device=dev)), lambda: nd.quantize_rows(q, codes=torch.ones(4, 15, dtype=torch.int8, device=dev)),
        lambda: nd.quantize_rows(q, scales=torch.ones(3, device=dev)), lambda: nd.quantize_rows(q.int()),
        lambda: nd.dequantize_rows(q.to(torch.int8), torch.ones(3, device=dev)), lambda: nd.dequantize_rows(q, torch.ones(4, device=dev)),
        lambda: nd.adjust_scores(s, seen=(off, ids)), lambda: nd.adjust_scores(s, penalties=pen), lambda: nd.adjust_scores(s, (off[:4], ids), pen),
        lambda: nd.adjust_scores(s, (off, ids.long()), pen), lambda: nd.adjust_scores(s, (off, ids), pen[:, :2]),
        lambda: nd.adjust_scores(s, bias=torch.ones(69, device=dev)), lambda: nd.adjust_scores(s, mask=w[:, :2]),
        lambda: nd.adjust_scores(s, out=s.half()), lambda: nd.adjust_scores(s, out=torch.ones(70, 4, device=dev).t()),
        lambda: nd.adjust_scores(s.int()),
    ]
    for i, c in enumerate(calls):
        with pytest.raises(NdbHipError) as e:
            c()
        assert e.value.code == _lib.ERR_INVALID, i
    assert t.nrows == 70
    # the workspace is checked, not trusted
    L = _lib.lib()
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=dev)
    out = torch.empty(4, 70, device=dev)
    assert L.ndbhip_i8_product_device(t._h, q.data_ptr(), 0, None, 4, 16, None, out.data_ptr(), 0, 70, ws.data_ptr(), 100) == _lib.ERR_INVALID
    assert "workspace" in _lib.last_error()
    assert L.ndbhip_i8_product_device(t._h, q.data_ptr(), 0, None, 4, 16, None, out.data_ptr(), 0, 70, ws.data_ptr() + 8, 1 << 19) == _lib.ERR_INVALID
