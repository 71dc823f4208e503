"""The 8-bit scoring operators, case by case: what a caller holds before the call, the call, and the same result
computed with elementary torch operations.

    quantise   rows -> signed bytes with one scale a row, and the values those bytes stand for
    product    every query against every row of an 8-bit table: int8 x int8 -> int32, times the query's and the row's
               scale, plus a bias a row
    adjust     a matrix of scores: penalties for ids a query has already been given, biases, a bit mask
    search     the k best rows of an 8-bit table for every query, under a bias and a bit mask

Definitions (RN = round to nearest even, fp32 unless said otherwise):
    top = max |x| of the row;  top < 2^-100: scale = 0, bytes 0;  top NaN or infinite: scale = NaN, bytes 0
    else scale = RN(top / 127), inv = RN(127 / top), byte = the integer nearest to x * inv (that product taken exactly,
    halves to even)
    score = RN(RN(RN(dot) * row scale) * query scale), then RN(score + bias) where there is a bias
    search: a row takes part where its mask bit is 1 and its score is neither NaN nor -inf; larger scores first, equal
    ones in the order of their ids; places that no row fills hold id -1 and score -inf
    adjust, in fp32 and rounded once to the scores' type: for an id the query has been given c > 0 times
    s = s / repeat where s > 0, else s * repeat, then s - (presence + c * frequency); then s + bias; then -inf where the
    mask bit is 0
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TINY = 2.0 ** -100


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one embedding on its way to an 8-bit table: the smallest call, all latency
        dict(name="quantise one query", op="quantise", rows=1, dim=768, dtype="f32"),
        # loading the 1M x 768 float4 table of the headline benchmark
        dict(name="quantise a float4 table", op="quantise", rows=1_000_000, dim=768, dtype="f32"),
        # a halfvec column of 1536 dimensions, a ragged number of rows
        dict(name="quantise halfvec rows", op="quantise", rows=100_003, dim=1536, dtype="f16"),
        # one query scored against the 10k x 128 table
        dict(name="product one query", op="product", nq=1, n=10_000, dim=128, qtype="f32", otype="f32", bias=False),
        # a batch of halfvec queries of odd size against rows of odd length, boosted rows, 16-bit scores
        dict(name="product odd batch", op="product", nq=77, n=50_021, dim=300, qtype="f16", otype="bf16", bias=True),
        # a large batch scored in full for a hybrid ranking: the matrix product itself
        dict(name="product large", op="product", nq=1024, n=131_072, dim=1536, qtype="f32", otype="f32", bias=False),
        # the scores of one query against 10k rows, a session that has seen a few of them
        dict(name="adjust one row", op="adjust", nq=1, n=10_000, dtype="f32", seen=20, bias=True, mask=True),
        # a batch of scores against a million rows, a filter for each query, long sessions
        dict(name="adjust a batch", op="adjust", nq=64, n=1_000_000, dtype="f32", seen=500, bias=True, mask=True),
        # one query, the small table: all latency
        dict(name="search small", op="search", nq=1, n=10_000, dim=128, k=10, qtype="f32", bias=False, mask=0),
        # one query, the headline table: one pass over 768 MB
        dict(name="search one query", op="search", nq=1, n=1_000_000, dim=768, k=10, qtype="f32", bias=False, mask=0),
        # filtered batches of halfvec queries, a longer list for a later stage to rank again
        dict(name="search filtered", op="search", nq=50, n=300_007, dim=1536, k=100, qtype="f16", bias=True, mask=2),
        # the headline table under a large batch
        dict(name="search large batch", op="search", nq=1024, n=1_000_000, dim=768, k=10, qtype="f32", bias=False, mask=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantise", "product", "adjust", "search"])
    dim = rng.choice([_log(rng, 3, 1536), rng.choice([64, 128, 384, 768, 1024, 1536])])
    if op == "quantise":
        dtype = rng.choice(["f32", "f16", "bf16"])
        return dict(op=op, rows=_log(rng, 1, 768_000_000 // max(dim, 768)), dim=dim, dtype=dtype)
    if op == "adjust":
        n = _log(rng, 1, 1_000_000)
        nq = _log(rng, 1, min(2048, 64_000_000 // n))
        return dict(op=op, nq=nq, n=n, dtype=rng.choice(["f32", "f16", "bf16"]), seen=rng.choice([0, _log(rng, 1, 500)]),
                    bias=rng.random() < 0.5, mask=rng.random() < 0.5)
    nq = _log(rng, 1, 1024)
    if op == "product":
        return dict(op=op, nq=nq, n=_log(rng, 1, 131_072), dim=dim, qtype=rng.choice(["f32", "f16", "bf16"]),
                    otype=rng.choice(["f32", "f16", "bf16"]), bias=rng.random() < 0.5)
    return dict(op=op, nq=nq, n=_log(rng, 10, min(1_000_000, 768_000_000 // max(dim, 768))), dim=dim, k=_log(rng, 1, 128),
                qtype=rng.choice(["f32", "f16", "bf16"]), bias=rng.random() < 0.5, mask=rng.choice([0, 1, 2]))


# ---------------------------------------------------------------- what a caller has in hand

def _normal(g, shape, dtype="f32"):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(TYPES[dtype])


def _table(g, n, dim):
    """i.i.d. N(0, 1) rows as the benchmark's, one row in fifty a copy of another (equal scores), a few of zeros"""
    x = _normal(g, (n, dim))
    m = len(range(0, n, 50))
    x[::50] = x[torch.randint(0, n, (m,), generator=g, device="cuda")]
    x[25::2500] = 0.0
    return x


def _mask(g, rows, n):
    """half of all bits set; one query in sixteen (the last of each sixteen) has no row left"""
    w = (n + 31) // 32
    m = torch.randint(-(1 << 31), 1 << 31, (rows, w), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    if rows > 1:
        m[15::16] = 0
    return m


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, s = case["op"], dict(case)
    if op == "quantise":
        s["x"] = _normal(g, (case["rows"], case["dim"]), case["dtype"])
        return s
    n, nq = case["n"], case["nq"]
    s["bias_v"] = _normal(g, (n,)) if case["bias"] else None
    if op == "adjust":
        s["scores"] = (4 * _normal(g, (nq, n))).to(TYPES[case["dtype"]])
        s["mask_v"] = _mask(g, nq, n) if case["mask"] else None
        # ids a query has been given: half of them from a short range, so that several come more than once
        k = case["seen"]
        ids = torch.randint(0, n, (nq, k), generator=g, device="cuda")
        ids[:, : k // 2] %= max(1, k // 3)
        s["seen_ids"] = ids.reshape(-1).to(torch.int32)
        s["seen_off"] = torch.arange(nq + 1, device="cuda", dtype=torch.int64) * k
        pen = torch.rand((nq, 3), generator=g, device="cuda")
        s["penalties"] = torch.stack([1 + pen[:, 0], pen[:, 1], 0.5 * pen[:, 2]], 1).contiguous()
        return s
    rows = _table(g, n, case["dim"])
    s["q"] = _normal(g, (nq, case["dim"]), case["qtype"])
    if op == "search":
        s["mask_v"] = _mask(g, 1 if case["mask"] == 1 else nq, n) if case["mask"] else None
    if own:
        from neurondb_amd import Int8Table
        s["table"] = Int8Table(case["dim"])
        s["table"].load(rows)
    else:
        s["codes"], s["scales"] = _quantise(rows)
    return s


# ---------------------------------------------------------------- plain forms

def _quantise(x):
    """(signed bytes, scales): the products that decide a byte are taken in 64 bits, where they are exact"""
    x = x.float()
    top = x.abs().amax(1, keepdim=True)
    fine = torch.isfinite(top) & (top >= TINY)
    safe = torch.where(fine, top, torch.ones_like(top)).double()
    scale, inv = (safe / 127.0).float(), (127.0 / safe).float()
    codes = torch.where(fine, (x.double() * inv.double()).round(), torch.zeros((), dtype=torch.float64, device=x.device))
    scale = torch.where(fine, scale, torch.where(torch.isfinite(top), torch.zeros_like(top), torch.full_like(top, math.nan)))
    return codes.to(torch.int8), scale[:, 0]


def _scores(qc, qs, codes, scales, bias):
    """32 bits hold the integer sums exactly up to 1040 dimensions; beyond, 64"""
    wide = torch.float32 if codes.shape[1] * 127 * 127 < 1 << 24 else torch.float64
    s = (qc.to(wide) @ codes.to(wide).t()).float()
    s = (s * scales[None]) * qs[:, None]
    return s if bias is None else s + bias[None]


def _bits(mask, n):
    bits = (mask[:, :, None] >> torch.arange(32, device=mask.device, dtype=torch.int32)) & 1
    return bits.reshape(mask.shape[0], -1)[:, :n] != 0


def _best(s, k):
    """the k largest, equal ones by lowest id: order-preserving integers of the scores, the id below them"""
    nq, n = s.shape
    none = s.isnan() | (s == -math.inf)
    b = (s + 0.0).view(torch.int32)
    b = b ^ ((b >> 31) & 0x7FFFFFFF)
    key = (b.long() << 32) + (0xFFFFFFFF - torch.arange(n, device=s.device))[None]
    key = key.masked_fill(none, -(1 << 63))
    got = key.topk(min(k, n), dim=1).values
    ids = 0xFFFFFFFF - (got & 0xFFFFFFFF)
    out = torch.gather(s, 1, ids.clamp(max=n - 1))
    gone = got == -(1 << 63)
    ids, out = ids.masked_fill(gone, -1), out.masked_fill(gone, -math.inf)
    if k > n:
        ids = torch.cat([ids, ids.new_full((nq, k - n), -1)], 1)
        out = torch.cat([out, out.new_full((nq, k - n), -math.inf)], 1)
    return ids, out


def _adjust(s, seen_off, seen_ids, penalties, bias, mask):
    nq, n = s.shape
    t = s.float()
    if seen_ids.numel():
        q = torch.repeat_interleave(torch.arange(nq, device=s.device), seen_off.diff())
        c = torch.bincount(q * n + seen_ids.long(), minlength=nq * n).reshape(nq, n).float()
        repeat, presence, frequency = penalties[:, 0:1], penalties[:, 1:2], penalties[:, 2:3]
        t = torch.where(c > 0, torch.where(t > 0, t / repeat, t * repeat) - (presence + c * frequency), t)
    if bias is not None:
        t = t + bias[None]
    if mask is not None:
        t = t.masked_fill(~_bits(mask, n), -math.inf)
    return t.to(s.dtype)


def run(state):
    s = state
    if s["op"] == "quantise":
        if own:
            from neurondb_amd import dequantize_rows, quantize_rows
            codes, scales = quantize_rows(s["x"])
            return {"values": dequantize_rows(codes, scales), "scales": scales}
        codes, scales = _quantise(s["x"])
        return {"values": codes.float() * scales[:, None], "scales": scales}
    if s["op"] == "adjust":
        if own:
            from neurondb_amd import adjust_scores
            return adjust_scores(s["scores"], seen=(s["seen_off"], s["seen_ids"]), penalties=s["penalties"],
                                 bias=s["bias_v"], mask=s["mask_v"])
        return _adjust(s["scores"], s["seen_off"], s["seen_ids"], s["penalties"], s["bias_v"], s["mask_v"])
    if s["op"] == "product":
        if own:
            return s["table"].scores(s["q"], bias=s["bias_v"], dtype=TYPES[s["otype"]])
        qc, qs = _quantise(s["q"])
        return _scores(qc, qs, s["codes"], s["scales"], s["bias_v"]).to(TYPES[s["otype"]])
    if own:
        ids, scores = s["table"].search(s["q"], s["k"], bias=s["bias_v"], mask=s["mask_v"])
        return {"ids": ids, "scores": scores}
    qc, qs = _quantise(s["q"])
    t = _scores(qc, qs, s["codes"], s["scales"], s["bias_v"])
    if s["mask_v"] is not None:
        t = t.masked_fill(~_bits(s["mask_v"], s["n"]), -math.inf)
    ids, scores = _best(t, s["k"])
    return {"ids": ids, "scores": scores}


# ---------------------------------------------------------------- work

def work(case):
    size = lambda t: 4 if t == "f32" else 2  # noqa: E731
    if case["op"] == "quantise":
        e = case["rows"] * case["dim"]
        return {"bytes": e * size(case["dtype"]) + 4 * e + 4 * case["rows"], "flops": 4 * e}
    nq, n = case["nq"], case["n"]
    extra = 4 * n if case["bias"] else 0
    if case["op"] == "adjust":
        b = 2 * nq * n * size(case["dtype"]) + extra + nq * (4 * case["seen"] + 8 + 12)
        return {"bytes": b + (nq * n // 8 if case["mask"] else 0), "flops": 3 * nq * n}
    b = n * case["dim"] + 4 * n + extra + nq * case["dim"] * size(case["qtype"])
    if case["op"] == "product":
        b += nq * n * size(case["otype"])
    else:
        b += 12 * nq * case["k"] + ({0: 0, 1: 1, 2: nq}[case["mask"]] * n) // 8
    return {"bytes": b, "flops": 2 * nq * n * case["dim"]}


# ---------------------------------------------------------------- 64 bits

def _bytes64(x):
    """bytes and scales (both as float64) of rows, from the definition; the scale a row is stored with is an fp32 number"""
    x = x.to(torch.float64)
    top = x.abs().max(dim=1).values
    inv = torch.as_tensor(127.0, dtype=torch.float64, device=x.device).div(top).to(torch.float32).to(torch.float64)
    live = (top >= TINY) & (top < math.inf)
    code = torch.where(live[:, None], torch.round(x.mul(inv[:, None])), torch.zeros_like(x))
    scale = top.div(torch.as_tensor(127.0, dtype=torch.float64, device=x.device))
    return code, torch.where(live, scale, torch.zeros_like(scale)), live


def exact(case, seed):
    s = prepare_rows(case, seed)
    if case["op"] == "quantise":
        out_v, out_s = [], []
        for x in s["x"].split(1 << 18):
            code, scale, _ = _bytes64(x)
            out_v.append(code * scale[:, None])
            out_s.append(scale)
        return {"values": torch.cat(out_v), "scales": torch.cat(out_s)}
    if case["op"] == "adjust":
        v = s["scores"].to(torch.float64).cpu().numpy()
        off, ids, pen = s["seen_off"].cpu().numpy(), s["seen_ids"].cpu().numpy(), s["penalties"].double().cpu().numpy()
        for q in range(case["nq"]):
            at, c = np.unique(ids[off[q]:off[q + 1]], return_counts=True)
            old = v[q, at]
            v[q, at] = np.where(old > 0, old / pen[q, 0], old * pen[q, 0]) - (pen[q, 1] + c * pen[q, 2])
        if s["bias_v"] is not None:
            v += s["bias_v"].double().cpu().numpy()
        if s["mask_v"] is not None:
            b = np.unpackbits(s["mask_v"].cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, : case["n"]]
            v[b == 0] = -np.inf
        return v
    qb, qs, _ = _bytes64(s["q"])
    best = None
    out = []
    step = max(1, (1 << 27) // max(case["nq"], case["dim"]))
    for at in range(0, case["n"], step):
        rb, rs, _ = _bytes64(s["rows"][at:at + step])
        v = torch.mm(qb * qs[:, None], (rb * rs[:, None]).t().contiguous())
        if s["bias_v"] is not None:
            v += s["bias_v"][at:at + step].double()
        if case["op"] == "product":
            out.append(v)
            continue
        if s["mask_v"] is not None:
            i = torch.arange(at, at + v.shape[1], device=v.device)
            v[(((s["mask_v"][:, i // 32] >> (i % 32).int()) & 1) == 0).expand_as(v)] = -math.inf
        v = v if best is None else torch.cat([best, v], 1)
        best = v.topk(min(case["k"], v.shape[1]), dim=1, sorted=True).values
    if case["op"] == "product":
        return torch.cat(out, 1)
    if best.shape[1] < case["k"]:
        best = torch.cat([best, best.new_full((case["nq"], case["k"] - best.shape[1]), -math.inf)], 1)
    return {"ids": None, "scores": best}    # ids of scores closer than fp32 tells apart have no 64-bit value


def prepare_rows(case, seed):
    """the inputs of prepare(case, seed), the table as the rows it is loaded from"""
    if case["op"] in ("quantise", "adjust"):
        return prepare(case, seed)
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"bias_v": _normal(g, (case["n"],)) if case["bias"] else None}
    s["rows"] = _table(g, case["n"], case["dim"])
    s["q"] = _normal(g, (case["nq"], case["dim"]), case["qtype"])
    if case["op"] == "search":
        s["mask_v"] = _mask(g, 1 if case["mask"] == 1 else case["nq"], case["n"]) if case["mask"] else None
    return s
