"""The 8-bit row operators on cases of their real use: quantisation, the root-mean-square norm that ends in 8-bit rows, the
block-scaled product, and the search of an 8-bit Flat index.

An 8-bit row is e4m3 codes with one power-of-two scale for every 128 of them: the smallest power of two s with
max|x| <= 448 s, code = x / s rounded to nearest even.  The scale is kept as its biased exponent in one byte.

With `own` false every operator is computed from elementary torch operations; with `own` true by semantic_search_amd."""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SPARE = 16  # candidates beyond k that are scored again in 64 bits


def listed():
    return [
        # the last norm of an embedding model for one text (a single query): latency
        {"name": "norm one row", "op": "norm", "n": 1, "d": 4096, "type": "bf16", "residual": True, "weight": True, "unit": True},
        # rows of a small model of odd width, already added up, on their way into an index: unit length
        {"name": "norm odd rows", "op": "norm", "n": 1023, "d": 777, "type": "f32", "residual": False, "weight": True, "unit": True},
        # the norm inside a layer over a long prefill
        {"name": "norm prefill", "op": "norm", "n": 32768, "d": 4096, "type": "bf16", "residual": True, "weight": True, "unit": False},
        # a bulk add: 2048-d embeddings as the embedder hands them over
        {"name": "quantise bulk", "op": "quantise", "n": 200000, "d": 2048, "type": "f32"},
        # a handful of fresh rows of odd width
        {"name": "quantise few", "op": "quantise", "n": 33, "d": 1000, "type": "f16"},
        # one token through a projection: bound by the weights
        {"name": "product one row", "op": "product", "m": 1, "n": 4096, "k": 4096, "type": "bf16"},
        # a small decoding batch through a wide projection
        {"name": "product batch", "op": "product", "m": 48, "n": 12288, "k": 4096, "type": "f16"},
        # ragged in every direction
        {"name": "product odd", "op": "product", "m": 1001, "n": 2051, "k": 1100, "type": "bf16"},
        # prefill or bulk embedding: bound by the matrix cores
        {"name": "product large", "op": "product", "m": 8192, "n": 8192, "k": 8192, "type": "bf16"},
        # the smallest index of the baseline, one query
        {"name": "search small", "op": "search", "rows": 10000, "d": 4096, "nq": 1, "k": 10},
        # the default workload, one query: bound by the rows
        {"name": "search one", "op": "search", "rows": 1000000, "d": 4096, "nq": 1, "k": 10},
        # a large batch over the same rows: bound by the matrix cores
        {"name": "search batch", "op": "search", "rows": 1000000, "d": 4096, "nq": 1024, "k": 10},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "quantise", "product", "product", "search", "search"])
    if op == "norm":
        d = _log(rng, 64, 8192)
        return {"op": op, "n": _log(rng, 1, min(32768, (1 << 27) // d)), "d": d, "type": rng.choice(["f32", "f16", "bf16"]),
                "residual": rng.random() < 0.6, "weight": rng.random() < 0.8, "unit": rng.random() < 0.5}
    if op == "quantise":
        d = _log(rng, 64, 8192)
        return {"op": op, "n": _log(rng, 1, (1 << 28) // d), "d": d, "type": rng.choice(["f32", "f16", "bf16"])}
    if op == "product":
        return {"op": op, "m": _log(rng, 1, 8192), "n": _log(rng, 64, 8192), "k": _log(rng, 64, 8192),
                "type": rng.choice(["f16", "bf16"])}
    d = _log(rng, 64, 4096)
    return {"op": op, "rows": _log(rng, 1000, min(1000000, (1 << 32) // d)), "d": d, "nq": _log(rng, 1, 1024),
            "k": _log(rng, 1, 200)}


# ---- the 8-bit rows, plain ----

def _quantise(x):
    """(codes (n, whole blocks) float8_e4m3fn, biased exponents (n, blocks) uint8) of finite rows (n, d), in 32 bits."""
    n, d = x.shape
    blocks = (d + 127) // 128
    x = torch.nn.functional.pad(x.float(), (0, blocks * 128 - d)).view(n, blocks, 128)
    m, e = torch.frexp(x.abs().amax(dim=2))             # amax = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m == 0, -127, e - 8 - (m <= 0.875).int()).clamp(min=-127)
    codes = torch.ldexp(x, -e.unsqueeze(2)).to(torch.float8_e4m3fn)
    return codes.view(n, blocks * 128), (e + 127).to(torch.uint8)


def _dequantise(codes, exps, d):
    n, blocks = exps.shape
    s = torch.ldexp(torch.ones((), device=codes.device), exps.int() - 127)
    return (codes.float().view(n, blocks, 128) * s.unsqueeze(2)).view(n, blocks * 128)[:, :d]


def _values64(codes, exps, d):
    """The rows in 64 bits, from the bits of the codes: sign, exponent (bias 7) and three bits of fraction."""
    n, blocks = exps.shape
    table = [(-1.0 if c & 128 else 1.0) * (math.ldexp(c & 7, -9) if not c & 120 else math.ldexp(8 + (c & 7), ((c >> 3) & 15) - 10)) for c in range(256)]
    v = torch.tensor(table, dtype=torch.float64, device=codes.device)[codes.view(torch.uint8).int()]
    s = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=codes.device), exps.double() - 127)
    return (v.view(n, blocks, 128) * s.unsqueeze(2)).view(n, blocks * 128)[:, :d]


def _round64(x):
    """Rows in 64 bits -> the values of their 8-bit rows in 64 bits, by comparisons with the borders."""
    n, d = x.shape
    blocks = (d + 127) // 128
    v = torch.nn.functional.pad(x, (0, blocks * 128 - d)).view(n, blocks, 128)
    amax = v.abs().amax(dim=2, keepdim=True)
    e = torch.ceil(torch.log2(amax.clamp(min=1e-300) / 448)).clamp(min=-127)
    e = torch.where(torch.exp2(e - 1) * 448 >= amax, e - 1, e)
    e = torch.where(torch.exp2(e) * 448 < amax, e + 1, e).clamp(min=-127)
    u = v / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(u / step) * step * torch.exp2(e)).view(n, blocks * 128)[:, :d]


# ---- inputs ----

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFF)


def _rows(n, d, g, kind=None):
    """Rows with a few channels that are much larger than the others, as hidden states have them."""
    x = torch.randn(n, d, generator=g, device="cuda")
    x *= torch.exp(0.6 * torch.randn(d, generator=g, device="cuda"))
    return x if kind is None else x.to(_TYPES[kind])


def _index_rows(case, g):
    return _quantise(torch.nn.functional.normalize(torch.randn(case["rows"], case["d"], generator=g, device="cuda")))


def _queries(case, g):
    return torch.nn.functional.normalize(torch.randn(case["nq"], case["d"], generator=g, device="cuda"))


def _inputs(case, seed):
    g = _gen(seed)
    if case["op"] == "norm":
        x = _rows(case["n"], case["d"], g, case["type"])
        r = _rows(case["n"], case["d"], g, case["type"]) if case["residual"] else None
        w = (1 + 0.2 * torch.randn(case["d"], generator=g, device="cuda")).to(_TYPES[case["type"]]) if case["weight"] else None
        return {"x": x, "r": r, "w": w}
    if case["op"] == "quantise":
        return {"x": _rows(case["n"], case["d"], g, case["type"])}
    if case["op"] == "product":
        a = _quantise(_rows(case["m"], case["k"], g))
        return {"a": a, "b": _quantise(torch.randn(case["n"], case["k"], generator=g, device="cuda") / math.sqrt(case["k"]))}
    return {"rows": _index_rows(case, g), "q": _queries(case, g)}


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    if case["op"] == "norm" and s["r"] is not None:
        s["sum"] = torch.empty_like(s["r"])  # the stream of residuals that the norm updates
    if own:
        import semantic_search_amd as ssa
        if case["op"] == "product":
            s["a"], s["b"] = (ssa.F8Rows.from_parts(c, e, case["k"]) for c, e in (s["a"], s["b"]))
        elif case["op"] == "search":
            s["index"] = ssa.IndexFlatIP(case["d"], storage="f8")
            s["index"].set_timing(False)
            s["index"].add(ssa.F8Rows.from_parts(*s.pop("rows"), case["d"]))
    return s


# ---- one pass ----

def _run_own(s, case):
    import semantic_search_amd as ssa
    if case["op"] == "norm":
        if s["r"] is None:
            return ssa.rms_norm_f8(s["x"], weight=s["w"], eps=1e-6, unit=case["unit"]).dequantize(torch.bfloat16)
        y = ssa.rms_norm_f8(s["x"], weight=s["w"], residual=s["r"], residual_out=s["sum"], eps=1e-6, unit=case["unit"])
        return y.dequantize(torch.bfloat16), s["sum"]
    if case["op"] == "quantise":
        return ssa.quantize_f8(s["x"]).dequantize(torch.bfloat16)
    if case["op"] == "product":
        return ssa.matmul_f8(s["a"], s["b"], out_dtype=_TYPES[case["type"]])
    return s["index"].search(s["q"], case["k"])


def _run_plain(s, case):
    if case["op"] == "norm":
        h = s["x"].float()
        if s["r"] is not None:
            s["sum"].copy_(h + s["r"].float())         # rounded to the residual's type: what the next layer reads
            h = s["sum"].float()
        y = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + 1e-6)
        if s["w"] is not None:
            y = y * s["w"].float()
        if case["unit"]:
            y = y / y.square().sum(dim=1, keepdim=True).sqrt().clamp(min=1e-12)
        y = _dequantise(*_quantise(y), case["d"]).to(torch.bfloat16)
        return y if s["r"] is None else (y, s["sum"])
    if case["op"] == "quantise":
        return _dequantise(*_quantise(s["x"]), case["d"]).to(torch.bfloat16)
    if case["op"] == "product":
        return (_dequantise(*s["a"], case["k"]) @ _dequantise(*s["b"], case["k"]).T).to(_TYPES[case["type"]])
    # scores in 32 bits choose k and some more; their order is decided in 64 bits, ties by the lower id
    d, k = case["d"], case["k"]
    q = _dequantise(*_quantise(s["q"]), d)
    x = _dequantise(*s["rows"], d)
    ids = torch.topk(q @ x.T, min(k + _SPARE, case["rows"]), dim=1).indices.sort(dim=1).values
    best = (x[ids.view(-1)].view(*ids.shape, d).double() * q.double().unsqueeze(1)).sum(dim=2)
    best, order = best.sort(dim=1, descending=True, stable=True)
    return best[:, :k].float(), ids.gather(1, order)[:, :k]


def run(state):
    return _run_own(state, state["case"]) if own else _run_plain(state, state["case"])


# ---- what a pass cannot do without ----

def work(case):
    e = {"f32": 4, "f16": 2, "bf16": 2}.get(case.get("type"))
    row = lambda d: (d + 127) // 128 * 129  # noqa: E731  codes and scales of a row
    if case["op"] == "norm":
        n, d = case["n"], case["d"]
        # x and residual in; 8-bit rows, their values in 16 bits and the sum out
        return {"bytes": n * (d * e * (3 if case["residual"] else 1) + row(d) + 2 * d) + (d * e if case["weight"] else 0), "flops": 8 * n * d}
    if case["op"] == "quantise":
        n, d = case["n"], case["d"]
        return {"bytes": n * (d * e + row(d) + 2 * d), "flops": 2 * n * d}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * row(k) + 2 * m * n, "flops": 2 * m * n * k}
    n, d, nq, k = case["rows"], case["d"], case["nq"], case["k"]
    return {"bytes": n * row(d) + 4 * nq * d + 12 * nq * k, "flops": 2 * nq * n * d}


# ---- the definition in 64 bits ----

def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "norm":
        h = s["x"].double()
        if s["r"] is not None:
            h = (h + s["r"].double()).to(_TYPES[case["type"]]).double()
        y = h / torch.sqrt((h * h).sum(dim=1, keepdim=True) / case["d"] + 1e-6)
        y = y if s["w"] is None else y * s["w"].double()
        if case["unit"]:
            y = y / torch.sqrt((y * y).sum(dim=1, keepdim=True)).clamp(min=1e-12)
        y = _round64(y)
        return y if s["r"] is None else (y, h)
    if case["op"] == "quantise":
        return _round64(s["x"].double())
    if case["op"] == "product":
        return _values64(*s["a"], case["k"]) @ _values64(*s["b"], case["k"]).T
    x, k = _values64(*s["rows"], case["d"]), case["k"]
    score = _round64(s["q"].double()) @ x.T
    ids = torch.topk(score, min(k + 4, case["rows"]), dim=1).indices.sort(dim=1).values
    best, order = score.gather(1, ids).sort(dim=1, descending=True, stable=True)
    return best[:, :k], ids.gather(1, order)[:, :k]
