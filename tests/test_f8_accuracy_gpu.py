"""8-bit rows whose products differ in size by a lot: strong channels, as the last hidden states of a model have them, and large
products that cancel.  What is left over has to be there."""
import numpy as np
import pytest
import torch

import f8_plain as plain
from conftest import SALT

pytestmark = pytest.mark.gpu


def strong(n, d, channels, factor, seed):
    """Gaussian rows with a few channels that are `factor` times the others in every row."""
    g = torch.Generator(device="cuda").manual_seed(SALT + seed)
    x = torch.randn(n, d, generator=g, device="cuda")
    x[:, torch.randperm(d, generator=torch.Generator().manual_seed(channels * 7 + d))[:channels].tolist()] *= factor
    return x


def check(out, a, b):
    """Half a step of the output's type, and what fp32 sums may lose: an instruction adds 16 products (eight of them to a block of 128) and is
    off by less than 1.25 * 2^-23 of the magnitudes at hand per step of its own, none of which exceeds the sum of all the products'."""
    A, B = a.dequantize().double(), b.dequantize().double()
    want, mass = A @ B.T, A.abs() @ B.abs().T
    half, least = (2.0 ** -11, 2.0 ** -25) if out.dtype == torch.float16 else (2.0 ** -8, 0.0)
    sums = (8 * plain.blocks(a.d) + 8) * 1.25 * 2.0 ** -23
    # (the sum that is rounded may lie across a power of two from the exact one: its step, not the exact one's)
    assert ((out.double() - want).abs() <= (want.abs() + sums * mass) * half + least + sums * mass).all()


# a size for each tile of the product
SIZES = [(1, 500, 700), (48, 1000, 640), (130, 2000, 1024), (256, 4096, 640), (512, 4096, 1024), (1024, 4090, 1024), (4096, 4096, 1024), (33, 65, 128)]


@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("channels,factor", [(1, 100.0), (3, 30.0), (8, 1000.0)])
def test_product_of_rows_with_strong_channels(ssa, t, m, n, k, channels, factor):
    x, y = strong(m, k, channels, factor, m + k), strong(n, k, channels, factor, n + k + 1)
    scale = 1 / (factor * factor * channels) if t == torch.float16 else 1.0   # (within fp16's range)
    a, b = ssa.quantize_f8(x * scale), ssa.quantize_f8(y)
    check(ssa.matmul_f8(a, b, out_dtype=t), a, b)


@pytest.mark.parametrize("m,n,k", SIZES)
def test_products_that_cancel_leave_the_others(ssa, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(SALT + m)
    # whole numbers of one sign: the sums are exact, in whatever order
    x, y = (torch.randint(1, 4, (c, k), generator=g, device="cuda").float() for c in (m, n))
    i, j = (3, 4) if k > 4 else (0, 1)
    x[:, i], x[:, j] = 448, 448
    y[:, i], y[:, j] = 448, -448
    a, b = ssa.quantize_f8(x), ssa.quantize_f8(y)
    want = (x.double() @ y.double().T).bfloat16()
    assert torch.equal(ssa.matmul_f8(a, b), want)
    assert (want > 0).all()


def exact_search(rows, queries, k):
    """Score descending, ties by the lower id, over the 64-bit products of what the 8-bit rows stand for (none is NaN)."""
    S = queries.dequantize().double() @ rows.dequantize().double().T
    best, ids = torch.sort(S, dim=1, descending=True, stable=True)
    return best[:, :k], ids[:, :k]


def check_search(ssa, rows, queries, k):
    index = ssa.IndexFlatIP(rows.d, storage="f8")
    index.add(rows)
    D, I = index.search(queries, k)
    best, ids = exact_search(rows, queries, k)
    kk = best.shape[1]
    A, B = queries.dequantize().double(), rows.dequantize().double()
    # a 64-bit sum in another order may part in its last bits: rows may trade places there and nowhere else
    slack = 1e-13 * (A.norm(dim=1, keepdim=True) * B.norm(dim=1).max())
    got = (A @ B.T).gather(1, I[:, :kk])
    assert ((got - best).abs() <= slack).all()
    assert ((I[:, :kk] == ids) | ((got - best).abs() <= slack)).all()
    assert ((D[:, :kk].double() - best).abs() <= best.abs() * 2.0 ** -24 + slack).all()
    assert (I[:, kk:] == -1).all()
    assert all(len(set(r)) == kk for r in I[:, :kk].tolist())
    index.close()
    return I


@pytest.mark.parametrize("n,d", [(20000, 512), (6000, 768), (3000, 1024), (30000, 128)])
@pytest.mark.parametrize("channels,share", [(1, 0.5), (1, 0.98), (3, 0.98), (8, 0.98), (4, 0.9999)])
@pytest.mark.parametrize("nq,k", [(1, 1), (1, 10), (1, 100), (1, 1008), (8, 1), (8, 10), (20, 1), (20, 10), (20, 100), (128, 1), (128, 10), (128, 100),
                                  (300, 1), (300, 10), (300, 100), (300, 1008)])
def test_search_of_rows_with_strong_channels(ssa, n, d, channels, share, nq, k):
    """Unit rows, `share` of whose length lies in a few channels, as raw last hidden states have it."""
    g = torch.Generator(device="cuda").manual_seed(SALT + n + d + channels)
    make = lambda c: torch.nn.functional.normalize(torch.randn(c, d, generator=g, device="cuda"))  # noqa: E731
    x, q = make(n), make(nq)
    where = list(range(5, 5 + 8 * channels, 8)) if channels < 8 else list(range(8, 8 + channels))   # apart, or side by side
    for v in (x, q):
        v *= (1 - share * share) ** 0.5
        v[:, where] = share / channels ** 0.5 * (1 + 0.01 * torch.randn(len(v), channels, generator=g, device="cuda"))
    check_search(ssa, ssa.quantize_f8(x), ssa.quantize_f8(q), k)


@pytest.mark.parametrize("nq", [1, 3, 8, 20, 100, 300])
@pytest.mark.parametrize("n,d,k", [(5000, 300, 10), (3000, 4096, 100), (70000, 128, 30), (40, 200, 10)])
def test_search_among_rows_that_hardly_differ(ssa, n, d, k, nq):
    """More rows than there are spare candidates within a rounding of fp32 of each other: their order is that of the exact sums."""
    g = torch.Generator(device="cuda").manual_seed(SALT + n + d)
    x = torch.randn(1, d, generator=g, device="cuda").repeat(n, 1)
    q = torch.randn(nq, d, generator=g, device="cuda")
    few = torch.arange(0, d, 7, device="cuda")
    x[:, 0], q[:, 0] = 400.0, 400.0
    x[:, few[1:]] = torch.randint(-3, 4, (n, len(few) - 1), generator=g, device="cuda").float() * 2.0 ** -6   # they differ here,
    q[:, few[1:]] = torch.randint(-3, 4, (nq, len(few) - 1), generator=g, device="cuda").float() * 2.0 ** -6  # and by 2^-12 in 160000
    check_search(ssa, ssa.quantize_f8(x), ssa.quantize_f8(q), k)


@pytest.mark.parametrize("nq", [1, 5, 40, 300])
@pytest.mark.parametrize("n,k", [(9000, 1), (9000, 20), (9000, 1008), (300, 300)])
def test_search_among_copies_returns_the_lowest_ids(ssa, n, k, nq):
    """The whole index is copies of five rows: ties that no list of candidates holds."""
    g = torch.Generator(device="cuda").manual_seed(SALT + n + k)
    few = torch.nn.functional.normalize(torch.randn(5, 260, generator=g, device="cuda"))
    which = torch.randint(0, 5, (n,), generator=g, device="cuda")
    x, q = ssa.quantize_f8(few[which]), ssa.quantize_f8(torch.randn(nq, 260, generator=g, device="cuda"))
    I = check_search(ssa, x, q, k)
    S = q.dequantize().double() @ ssa.quantize_f8(few).dequantize().double().T
    order = S.argsort(dim=1, descending=True)
    for i in range(min(nq, 10)):
        want = torch.cat([(which == c).nonzero()[:, 0] for c in order[i]])[:k]
        assert torch.equal(I[i], want)


@pytest.mark.parametrize("scale_x,scale_q", [(1e37, 1.0), (1e30, 1e30), (1e-37, 1.0), (1e-20, 1e-20), (3e38, 1e-38)])
@pytest.mark.parametrize("nq", [1, 20, 300])
def test_search_at_the_ends_of_fp32(ssa, scale_x, scale_q, nq):
    """Sums that leave fp32 on the way, or vanish in it: the answer is the 64-bit one (what fp32 cannot hold of it: infinite or 0)."""
    g = torch.Generator(device="cuda").manual_seed(SALT + nq)
    x, q = (torch.nn.functional.normalize(torch.randn(c, 200, generator=g, device="cuda")) for c in (2000, nq))
    rows, queries = ssa.quantize_f8(x * scale_x), ssa.quantize_f8(q * scale_q)
    index = ssa.IndexFlatIP(200, storage="f8")
    index.add(rows)
    D, I = index.search(queries, 10)
    A = torch.from_numpy(plain.values(queries.codes.view(torch.uint8).cpu().numpy(), queries.scales.cpu().numpy(), 200))
    B = torch.from_numpy(plain.values(rows.codes.view(torch.uint8).cpu().numpy(), rows.scales.cpu().numpy(), 200))
    best, ids = torch.sort(A @ B.T, dim=1, descending=True, stable=True)
    assert torch.equal(I.cpu(), ids[:, :10])
    want = best[:, :10].float()
    assert ((D.cpu() == want) | ((D.cpu() - want).abs() <= want.abs() * 2.0 ** -22 + 2.0 ** -149)).all()


@pytest.mark.parametrize("nq", [1, 8, 40, 300])
@pytest.mark.parametrize("where", [[777], [0, 2999], list(range(100, 400))])
def test_search_among_rows_of_very_different_lengths(ssa, where, nq):
    """Some rows a million times the others: what fp32 loses beside them is more than the gaps between the others' scores."""
    g = torch.Generator(device="cuda").manual_seed(SALT)
    x, q = (torch.nn.functional.normalize(torch.randn(c, 200, generator=g, device="cuda")) for c in (3000, nq))
    x[where] *= 1e6
    for k in (10, 200):
        check_search(ssa, ssa.quantize_f8(x), ssa.quantize_f8(q), k)


@pytest.mark.parametrize("offset", [-700, -1, 5, 1 << 40])
@pytest.mark.parametrize("nq", [1, 30])
def test_offsets_and_floors_of_queries_that_take_the_exact_pass(ssa, nq, offset):
    g = torch.Generator(device="cuda").manual_seed(SALT + 3)
    x, q = (torch.nn.functional.normalize(torch.randn(c, 200, generator=g, device="cuda")) for c in (3000, nq))
    x[700:760] = x[700]          # copies for some,
    x[5] *= 1e5                  # and a long row for all
    rows, queries = ssa.quantize_f8(x), ssa.quantize_f8(q)
    index = ssa.IndexFlatIP(200, storage="f8")
    index.add(rows)
    best, ids = exact_search(rows, queries, 100)
    D, I = index.search(queries, 100, id_offset=offset)
    assert torch.equal(I, ids + offset)
    floor = float(best[0, 50])
    Df, If = index.search(queries, 100, id_offset=offset, min_score=floor)
    keep = D >= np.float32(floor)
    assert torch.equal(If, torch.where(keep, I, -1)) and torch.equal(Df, torch.where(keep, D, torch.full_like(D, -np.finfo(np.float32).max)))


def norm_case(name, t):
    g = torch.Generator(device="cuda").manual_seed(SALT + len(name))
    n, d = {"odd rows": (1023, 777), "residual": (900, 4096), "long": (60, 16384), "dominant": (2000, 1000), "dominant long": (40, 15001), "narrow": (3000, 128)}[name]
    x, r = (torch.randn(n, d, generator=g, device="cuda") for _ in range(2))
    if "dominant" in name:
        x[torch.arange(n), torch.randint(0, d, (n,), generator=g, device="cuda")] = 3e4   # what fp32 sums of squares lose the others beside
    w = 1 + 0.3 * torch.randn(d, generator=g, device="cuda")
    return x.to(t), r.to(t) if name == "residual" else None, w.to(t)


@pytest.mark.parametrize("t", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("unit", [False, True])
@pytest.mark.parametrize("name", ["odd rows", "residual", "long", "dominant", "dominant long", "narrow"])
def test_norm_is_the_64_bit_norm_rounded_once(ssa, name, unit, t):
    """The sums of up to 16384 squares, here and in the test, are each off by 2^14 * 2^-53 at most, halved by the root, and a handful of roundings of
    2^-53 follow: 2^-38 covers both.  An element may part from the exact row's only if that much moves it, or its block's scale, over a border."""
    x, r, w = norm_case(name, t)
    rows = ssa.rms_norm_f8(x, weight=w, residual=r, residual_out=None if r is None else torch.empty_like(r), eps=1e-6, unit=unit)
    h = x.double() if r is None else (x.float() + r.float()).to(t).double()
    y = h / torch.sqrt((h * h).mean(dim=1, keepdim=True) + 1e-6) * w.double()
    if unit:
        y = y / y.norm(dim=1, keepdim=True).clamp(min=1e-12)
    y = y.cpu().numpy()
    lo, hi = plain.round_rows(y * (1 - 2.0 ** -38)), plain.round_rows(y * (1 + 2.0 ** -38))
    got = plain.values(rows.codes.view(torch.uint8).cpu().numpy(), rows.scales.cpu().numpy(), rows.d)
    assert ((got == lo) | (got == hi)).all()
    assert np.mean(lo != hi) < 1e-6   # (the borders leave the rest nothing to hide in)


@pytest.mark.parametrize("k", [1, 10, 32, 33])
@pytest.mark.parametrize("d", [64, 300, 1024])
@pytest.mark.parametrize("kind", ["generic", "strong", "copies", "all", "half"])
def test_large_batches_whose_lists_are_proven_by_different_sums(ssa, kind, d, k):
    """Enough rows and queries for the largest tiles: queries that their first sums answer, queries that need better ones, queries that
    need all rows in 64 bits, in tiles of their own and together."""
    n, nq = 140000, 700
    g = torch.Generator(device="cuda").manual_seed(SALT + d + k)
    unit = torch.nn.functional.normalize
    x, q = unit(torch.randn(n, d, generator=g, device="cuda")), unit(torch.randn(nq, d, generator=g, device="cuda"))
    if kind in ("strong", "all"):
        some, few = (slice(0, n), slice(0, nq)) if kind == "strong" else (slice(90000, n), slice(400, 500))
        x[some] *= 0.02
        x[some, 7] = 1
        q[few] *= 0.02
        q[few, 7] = 1
    if kind in ("copies", "all"):
        x[1000:1300] = x[1000]
        q[300:310] = x[1000]
    if kind == "half":   # more copies than are listed, and long rows that leave the other queries rows in question
        x[:5000] = x[0]
        q[:350] = x[0]
        x[70000] *= 1e5
    check_search(ssa, ssa.quantize_f8(x), ssa.quantize_f8(q), k)


def test_searches_with_open_queries_on_two_streams(ssa):
    """Both keep their open queries in the handle's workspaces: one waits for the other."""
    g = torch.Generator(device="cuda").manual_seed(SALT + 9)
    x, q = (torch.nn.functional.normalize(torch.randn(c, 300, generator=g, device="cuda")) for c in (30000, 400))
    x[100:200] = x[100]
    q[::3] = x[100]
    x[7] *= 1e5
    rows, queries = ssa.quantize_f8(x), ssa.quantize_f8(q)
    index = ssa.IndexFlatIP(300, storage="f8")
    index.add(rows)
    _, ids = exact_search(rows, queries, 20)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(12):
        lo, hi = [(0, 400), (0, 1), (5, 9), (100, 130)][i % 4]
        part = queries[lo:hi]
        with torch.cuda.stream(streams[i % 2]):
            got.append((lo, hi, part, index.search(part, 20)[1]))
    torch.cuda.synchronize()
    for lo, hi, _, I in got:
        assert torch.equal(I, ids[lo:hi])
