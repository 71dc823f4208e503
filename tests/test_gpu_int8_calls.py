"""The way from Python and C to the 8-bit kernels, on the device: what a call costs and leaves behind."""
import math
import threading
import time

import numpy as np
import pytest
import torch

import neurondb_amd as nd
from neurondb_amd._lib import NdbHipError

pytestmark = pytest.mark.gpu


def us(calls, reps=300, rounds=9):
    """the least time a call of each took, back to back, the calls' rounds taking turns"""
    best = [float("inf")] * len(calls)
    for _ in range(rounds):
        for i, c in enumerate(calls):
            c()
            torch.cuda.synchronize()
            t = time.perf_counter()
            for _ in range(reps):
                c()
            torch.cuda.synchronize()
            best[i] = min(best[i], (time.perf_counter() - t) / reps * 1e6)
    return best


@pytest.mark.parametrize("nq,n", [(1, 1), (1, 10_000), (16, 3000)])
def test_one_term_on_few_scores_costs_no_more_than_an_addition(nq, n):
    """a third is left for the noise of a shared host; a call in several crossings took 1.8 to 2 times the addition"""
    s, b = torch.randn(nq, n, device="cuda"), torch.randn(n, device="cuda")
    own, plain = us([lambda: nd.adjust_scores(s, bias=b), lambda: s + b[None]])
    assert own < 1.33 * plain, (own, plain)


def test_one_term_on_scores_that_a_cache_holds_costs_no_more_than_an_addition():
    """(the kernel with the lists' counters took 1.17 times the addition)"""
    s, b = torch.randn(64, 333_333, device="cuda"), torch.randn(333_333, device="cuda")
    own, plain = us([lambda: nd.adjust_scores(s, bias=b), lambda: s + b[None]], reps=100)
    assert own < 1.1 * plain, (own, plain)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 3, 7, 1023, 1024, 1025, 2047, 2048, 2049, 4100])
def test_terms_without_lists(n, dtype):
    """one rounding to fp32 for the bias and one to the type, so equal bit for bit; what lies beside the result stays"""
    nq = 5
    g = torch.Generator().manual_seed(n)
    s = torch.randn(nq, n, generator=g).to(dtype)
    s[0, 0], s[1, n - 1], s[2, n // 2] = float("nan"), float("-inf"), float("inf")
    b, bq = torch.randn(n, generator=g), torch.randn(nq, n, generator=g)
    bits = torch.rand(nq, (n + 31) // 32 * 32, generator=g) < 0.5
    bits[3] = False
    words = (bits.view(nq, -1, 32).long() << torch.arange(32)).sum(2)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).int()
    bits = bits[:, :n]
    for bias in (None, b, bq):
        for mask in (None, words, words[:1]):
            want = s.float() if bias is None else s.float() + bias
            if mask is not None:
                want = want.masked_fill(~bits if mask.shape[0] > 1 else ~bits[:1], float("-inf"))
            out = torch.full((nq + 1, n + 9), 7.0, dtype=dtype, device="cuda")
            nd.adjust_scores(s.cuda(), bias=None if bias is None else bias.cuda(), mask=None if mask is None else mask.cuda(), out=out[:nq, 3:3 + n])
            assert torch.equal(out[:nq, 3:3 + n].cpu().nan_to_num(9.0, math.inf, -math.inf), want.to(dtype).nan_to_num(9.0, math.inf, -math.inf))
            assert bool((out[nq] == 7).all()) and bool((out[:, :3] == 7).all()) and bool((out[:, 3 + n:] == 7).all())


def test_a_saved_tensor_is_not_changed_unseen():
    """scores that some backward has kept, adjusted in place: autograd says so instead of using the new ones"""
    s = torch.randn(3, 50, device="cuda")
    w = torch.ones(3, 50, device="cuda", requires_grad=True)
    loss = (w * s).sum()
    nd.adjust_scores(s, bias=torch.ones(50, device="cuda"), out=s)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with pytest.raises(NdbHipError, match="gradient"):
        nd.adjust_scores(w)
    with torch.no_grad():
        assert torch.equal(nd.adjust_scores(w, bias=torch.ones(50, device="cuda")), w + 1)
    t = nd.Int8Table(50)
    t.load(w)                               # a copy
    assert not t.scores(w.detach()).requires_grad
    with torch.inference_mode():
        v = torch.ones(3, 3, device="cuda")
    nd.adjust_scores(v, out=v)
    t.scores(w.detach(), out=v)


def test_a_batch_in_passes_that_fill_no_tile():
    """a table so long that a search's passes are shorter than a tile is wide: as in pieces, and every row finds itself"""
    n, dim, nq = 460_000_000, 16, 300
    g = torch.Generator("cuda").manual_seed(1)
    codes = torch.randint(-127, 128, (n, dim), device="cuda", generator=g, dtype=torch.int8)
    scales = torch.cat([1 / c.float().norm(dim=1) for c in codes.split(1 << 25)])
    t = nd.Int8Table(dim)
    t.load(codes, scales)
    want = torch.arange(nq, device="cuda") * 1_533_331
    q = (codes[want], scales[want])
    assert t._workspace(nd.int8._state, 256, 3)[1] == t._workspace(nd.int8._state, 224, 3)[1] < 16 << 30
    torch.cuda.empty_cache()
    ids, sc = t.search(q, 3)
    for at in range(0, nq, 50):
        i, s = t.search((q[0][at:at + 50], q[1][at:at + 50]), 3)
        assert torch.equal(ids[at:at + 50], i) and torch.equal(sc[at:at + 50], s)
    found = (codes[ids[:, 0]] == q[0]).all(1) | (sc[:, 0] > 1 - 1e-5)      # (another row may lie in the same direction)
    assert bool(found.all())
    del codes, scales, t
    torch.cuda.empty_cache()


def test_two_threads_search_host_arrays_at_the_same_time():
    """each with a workspace of its own, kept from search to search and made larger where one is"""
    n, dim = 20_000, 96
    t = nd.Int8Table(dim)
    rng = np.random.default_rng(0)
    t.load(rng.standard_normal((n, dim)).astype(np.float32))
    q = [rng.standard_normal((m, dim)).astype(np.float32) for m in (1, 7, 40, 300)]
    mask = rng.integers(0, 2 ** 32, ((n + 31) // 32,), dtype=np.uint32)
    bias = rng.standard_normal(n).astype(np.float32)
    dev = [t.search(torch.from_numpy(x).cuda(), 20, bias=torch.from_numpy(bias).cuda(), mask=torch.from_numpy(mask.view(np.int32)).cuda()) for x in q]
    want = [(i.cpu().numpy(), s.cpu().numpy()) for i, s in dev]
    bad = []

    def work(order):
        try:
            for _ in range(15):
                for i in order:
                    ids, sc = t.search(q[i], 20, bias=bias, mask=mask)
                    if not (np.array_equal(ids, want[i][0]) and np.array_equal(sc, want[i][1])):
                        bad.append(i)
        except Exception as e:          # noqa: BLE001 (reported below)
            bad.append(e)

    th = [threading.Thread(target=work, args=(o,)) for o in ((0, 1, 2, 3), (3, 1, 0, 2), (2, 0, 3, 1))]
    [x.start() for x in th]
    [x.join() for x in th]
    assert not bad
    t.load(rng.standard_normal((50, dim)).astype(np.float32))
    assert t.search(q[0], 3)[0].max() < 50
