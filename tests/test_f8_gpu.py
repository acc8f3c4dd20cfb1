"""8-bit rows on the GPU against 64 bits (tests/f8_plain.py): quantiser, norm, product, and the Flat index that keeps them."""
import numpy as np
import pytest
import torch

import f8_plain as plain
from conftest import SALT, unit_rows

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # half a step, relative


def cuda(x, t=torch.float32):
    return torch.as_tensor(np.asarray(x)).to("cuda", t)


def raw(rows):
    return rows.codes.view(torch.uint8).cpu().numpy(), rows.scales[:, :plain.blocks(rows.d)].cpu().numpy()


def rows64(rows):
    return plain.values(*raw(rows), rows.d)


def wild(n, d, seed):
    """Rows over many magnitudes with the values where the format changes its mind."""
    r = np.random.default_rng(SALT + seed)
    x = (r.standard_normal((n, d)) * np.exp(4 * r.standard_normal((n, 1)))).astype(np.float32)
    edge = [0.0, 448.0, 448.00003, 464.0, 3.5, 3.5000002, 2.0 ** -126, 2.0 ** -133, 2.0 ** -149, 1e38, -448.0, 17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10]
    for i in range(min(n, len(edge))):
        x[i, (7 * i) % d] = edge[i]
        if i % 3 == 0:
            x[i] = np.where(np.arange(d) % 128 == (7 * i) % 128, edge[i], x[i] * 1e-3)
    if n > 2:
        x[-1] = 0
        x[-2] = -0.0
    return x


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,d", [(1, 1), (3, 127), (17, 128), (5, 129), (40, 777), (9, 1000), (33, 2048), (4, 4096), (2, 8192), (2, 20001), (1, 65536), (1100, 300), (1030, 2049)])
def test_quantise_is_the_definition_bit_for_bit(ssa, kind, n, d):
    x = cuda(wild(n, d, 11 * n + d), TYPES[kind])
    if kind == "f16":
        x = x.clamp(-60000, 60000)
    q = ssa.quantize_f8(x)
    c, s = plain.quantize(x.double().cpu().numpy())
    got = raw(q)
    assert np.array_equal(got[1], s) and np.array_equal(got[0], c)
    # what the rows stand for, and quantising that gives the same values again
    v = q.dequantize()
    assert np.array_equal(v.double().cpu().numpy(), plain.values(c, s, d))
    again = raw(ssa.quantize_f8(v))
    assert np.array_equal(plain.values(*again, d), plain.values(c, s, d))


def test_quantise_values_that_are_not_finite(ssa):
    x = np.ones((4, 300), dtype=np.float32)
    x[0, 5], x[1, 130], x[2, 299] = np.inf, np.nan, -np.inf
    q = ssa.quantize_f8(cuda(x))
    c, s = plain.quantize(x)
    assert np.array_equal(raw(q)[0], c) and np.array_equal(raw(q)[1], s)
    v = q.dequantize(torch.bfloat16).float().cpu().numpy()
    assert np.isnan(v[0, :128]).all() and np.isfinite(v[0, 128:]).all() and np.isnan(v[1, 128:256]).all() and np.isnan(v[2, 256:]).all()
    assert (v[3] == 1).all()


def test_quantise_strided_unaligned_and_empty_rows(ssa):
    base = cuda(wild(40, 515, 5))
    for x in (base[:, 1:388], base[::2, :512], base[3:4], base.t()[:300], base[:, ::2]):
        c, s = plain.quantize(x.double().cpu().numpy())
        got = raw(ssa.quantize_f8(x))
        assert np.array_equal(got[0], c) and np.array_equal(got[1], s)
    assert ssa.quantize_f8(base[:0]).n == 0 and ssa.quantize_f8(base[:0]).dequantize().shape == (0, 515)
    out = ssa.F8Rows.empty(50, 515, "cuda")
    out.codes.view(torch.uint8).fill_(0x55)
    out.scales.fill_(0x55)
    ssa.quantize_f8(base, out=out[:40])
    assert np.array_equal(raw(out[:40])[0], plain.quantize(base.cpu().numpy())[0])
    assert (out.codes.view(torch.uint8)[40:] == 0x55).all() and (out.scales[40:] == 0x55).all()   # rows behind stay


@pytest.mark.parametrize("t", [torch.float32, torch.float16, torch.bfloat16])
def test_dequantise_every_code_and_scale(ssa, t):
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").repeat(256, 1)
    scales = torch.arange(256, dtype=torch.uint8, device="cuda")[:, None].expand(256, 2).contiguous()
    rows = ssa.F8Rows.from_parts(codes, scales, 256)
    got = rows.dequantize(t).double().cpu().numpy()
    with np.errstate(all="ignore"):
        want = torch.from_numpy(plain.values(codes.cpu().numpy(), scales.cpu().numpy(), 256)).float().to(t).double().numpy()
    assert np.array_equal(got, want, equal_nan=True)


def norm64(x, r, w, eps, unit, t):
    h = x.double() if r is None else (x.float() + r.float()).to(t).double()
    y = h / torch.sqrt((h * h).mean(dim=1, keepdim=True) + eps)
    y = y if w is None else y * w.double()
    if unit:
        y = y / y.norm(dim=1, keepdim=True).clamp(min=1e-12)
    return h.cpu().numpy(), y.cpu().numpy()


def check_norm(rows, y):
    """Half a step of e4m3 (2^-4 relative; 2^-10 s below its normal range, s <= amax / 224), and the fp32 path in front: two sums
    of squares whose d terms are added in trees and chains of at most 64 with 2^-24 each, halved by the root, and five more
    roundings: 40 * 2^-24 covers them, which may also move the block's largest element over a border of s (a factor 2)."""
    v = rows64(rows)
    n, d = y.shape
    pad = np.zeros((n, plain.blocks(d) * 128))
    pad[:, :d] = np.abs(y)
    amax = np.repeat(pad.reshape(n, -1, 128).max(axis=2), 128, axis=1)[:, :d]
    assert (np.abs(v - y) <= np.abs(y) * (2.0 ** -4 + 40 * 2.0 ** -24) + amax / 224 * 2.0 ** -10 * 1.001 + 1e-40).all()
    # nearly every element is the rounding of the exact one: they part only where y lies within 2^-18 of a border
    assert np.mean(v != plain.round_rows(y)) <= 1e-3 + 2.0 / y.size


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,d", [(1, 1), (2, 64), (1, 4096), (7, 777), (300, 1000), (1500, 128), (1100, 2048), (1030, 4096), (5, 8192), (1030, 8000), (2, 15001), (1, 16384)])
@pytest.mark.parametrize("residual,weight,unit", [(False, True, False), (True, True, True), (True, False, False), (False, False, True)])
def test_norm(ssa, kind, n, d, residual, weight, unit):
    t = TYPES[kind]
    r = np.random.default_rng(SALT + n + d)
    x, res = cuda(r.standard_normal((n, d)) * 3, t), cuda(r.standard_normal((n, d)), t)
    w = cuda(1 + 0.3 * r.standard_normal(d), torch.float32 if kind == "f16" else t) if weight else None
    h, y = norm64(x, res if residual else None, w, 1e-5, unit, t)
    before, keep = x.clone(), res.clone()
    if residual:
        out = torch.empty_like(res)
        first = ssa.rms_norm_f8(x, weight=w, residual=res, residual_out=out, eps=1e-5, unit=unit)
        assert torch.equal(res, keep) and np.array_equal(out.double().cpu().numpy(), h)
        rows = ssa.rms_norm_f8(x, weight=w, residual=res, eps=1e-5, unit=unit)   # in place
        assert torch.equal(res, out) and all(np.array_equal(a, b) for a, b in zip(raw(rows), raw(first)))
    else:
        rows = ssa.rms_norm_f8(x, weight=w, eps=1e-5, unit=unit)
    assert torch.equal(x, before)
    check_norm(rows, y)


def test_norm_of_zero_rows_and_rows_that_are_not_finite(ssa):
    x = torch.randn(4, 300, device="cuda")
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 7] = float("inf")
    v = ssa.rms_norm_f8(x, unit=True).dequantize().cpu().numpy()
    assert np.isfinite(v[:2]).all() and (v[1] == 0).all() and np.isnan(v[2]).all()
    assert np.isnan(v[3, :128]).all()                       # inf / inf; the other blocks are x / inf = 0
    assert ssa.rms_norm_f8(x[1:2], eps=0.0).dequantize().isnan().all()   # 0 / 0
    assert ssa.rms_norm_f8(x[:0]).n == 0


def product64(a, b):
    return rows64(a) @ rows64(b).T


def check_product(out, a, b):
    """Half a step of the output's type, and the matrix instruction: a product is off by less than 2^-13 of the largest of its
    block, 128 of them per block."""
    want = product64(a, b)
    nb = plain.blocks(a.d)
    big = 0.0
    if a.n and b.n:
        pad = lambda m: np.pad(np.abs(m), ((0, 0), (0, nb * 128 - a.d))).reshape(len(m), nb, 128).max(axis=2)  # noqa: E731
        big = pad(rows64(a)) @ pad(rows64(b)).T
    half = HALF[out.dtype]
    got = out.double().cpu().numpy()
    assert (np.abs(got - want) <= half * np.abs(want) + 128 * 2.0 ** -13 * big + (2.0 ** -24 if out.dtype == torch.float16 else 0)).all()
    norm = np.linalg.norm(want)
    assert np.linalg.norm(got - want) <= (half + 2.0 ** -13) * norm


@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 17, 128), (1, 4096, 4096), (2, 100, 129), (15, 33, 1000), (16, 16, 256), (17, 515, 300), (33, 64, 2048),
                                   (64, 130, 640), (65, 127, 384), (127, 129, 100), (128, 128, 512), (200, 1000, 1100), (513, 255, 130), (1000, 70, 77),
                                   (300, 5000, 256), (4100, 4200, 200)])
def test_product(ssa, t, m, n, k):
    r = np.random.default_rng(SALT + m + 3 * n + k)
    a, b = (ssa.quantize_f8(cuda(r.standard_normal((c, k)) * np.exp(0.7 * r.standard_normal((c, 1))))) for c in (m, n))
    check_product(ssa.matmul_f8(a, b, out_dtype=t), a, b)


def test_product_scales_of_all_sizes_strides_and_untouched_surroundings(ssa):
    r = np.random.default_rng(SALT + 1)
    for m, n, k in ((5, 70, 700), (90, 200, 520)):
        x = r.standard_normal((m, k)) * np.exp2(r.integers(-20, 20, (m, 1)))
        y = r.standard_normal((n, k)) * np.exp2(np.repeat(r.integers(-6, 6, (n, plain.blocks(k))), 128, axis=1)[:, :k])
        a, b = ssa.quantize_f8(cuda(x)), ssa.quantize_f8(cuda(y))
        big = ssa.F8Rows.from_parts(*(torch.nn.functional.pad(v, (0, 0, 3, 2)) for v in (b.codes.view(torch.uint8), b.scales)), k)[3:3 + n]
        wide = torch.full((m + 2, n + 9), 7.0, dtype=torch.bfloat16, device="cuda")
        out = ssa.matmul_f8(a, big, out=wide[1:m + 1, 3:3 + n])   # rows that are not 8-byte aligned
        check_product(out, a, b)
        wide[1:m + 1, 3:3 + n] = 7
        assert (wide == 7).all()
        assert torch.equal(ssa.matmul_f8(a, b), ssa.matmul_f8(a, big))
    assert ssa.matmul_f8(a[:0], b).shape == (0, n) and ssa.matmul_f8(a, b[:0]).shape == (m, 0)


def test_product_of_rows_that_are_not_finite(ssa):
    x = torch.randn(70, 400, device="cuda")
    x[3, 200] = float("inf")
    x[69, 0] = float("nan")
    y = torch.randn(100, 400, device="cuda")
    y[50, 399] = float("nan")
    for m in (10, 70):
        out = ssa.matmul_f8(ssa.quantize_f8(x[:m]), ssa.quantize_f8(y))
        bad = torch.zeros(70, 100, dtype=torch.bool, device="cuda")
        bad[3], bad[69], bad[:, 50] = True, True, True
        assert torch.equal(out.isnan(), bad[:m])
    zero = ssa.quantize_f8(torch.zeros(5, 400, device="cuda"))
    assert (ssa.matmul_f8(zero, ssa.quantize_f8(y[:50])) == 0).all()


def check_search(D, I, X, Q, k, id_offset=0):
    D, I = (v.cpu().numpy() if isinstance(v, torch.Tensor) else v for v in (D, I))
    Dr, Ir = plain.search(X, Q, k)
    Ir = np.where(Ir >= 0, Ir + id_offset, -1)
    assert np.array_equal(I, Ir)
    assert (np.abs(D.astype(np.float64) - Dr) <= np.spacing(np.abs(Dr))).all()   # the 64-bit sums may part in their last bit


def filled(ssa, X, **kw):
    index = ssa.IndexFlatIP(X.shape[1], storage="f8", **kw)
    index.add(X)
    return index


@pytest.mark.parametrize("n,d,nq,k", [(1, 1, 1, 1), (5, 64, 1, 10), (15, 128, 2, 3), (16, 129, 3, 16), (17, 100, 4, 1), (255, 512, 5, 7), (257, 640, 8, 48), (1000, 777, 9, 10),
                                      (3000, 1000, 1, 200), (2000, 300, 3, 100), (4000, 1536, 16, 20), (1500, 2048, 33, 5), (5000, 64, 64, 10), (3333, 200, 65, 49),
                                      (700, 256, 130, 12), (300, 130, 300, 300), (2500, 96, 2, 1008), (2500, 96, 70, 1008), (20000, 4096, 1, 10), (9000, 384, 257, 10)])
def test_search_is_the_64_bit_search_of_the_8_bit_rows(ssa, n, d, nq, k):
    X, Q = unit_rows(n, d, SALT + n + d), unit_rows(nq, d, SALT + nq)
    index = filled(ssa, X)
    assert index.storage == "f8" and index.ntotal == n and index.d == d
    X64, Q64 = plain.round_rows(X), plain.round_rows(Q)
    check_search(*index.search(Q, k), X64, Q64, k)
    D, I = index.search(cuda(Q), k, id_offset=1000)
    check_search(D, I, X64, Q64, k, 1000)
    D2, I2 = index.search(ssa.quantize_f8(cuda(Q)), k, id_offset=1000)
    assert torch.equal(D, D2) and torch.equal(I, I2)
    index.close()


def test_a_query_gets_the_same_answer_in_any_batch(ssa):
    X, Q = unit_rows(6000, 512, SALT + 1), unit_rows(200, 512, SALT + 2)
    index = filled(ssa, X)
    D, I = index.search(Q, 20)
    for lo, hi in ((0, 1), (3, 5), (10, 18), (20, 60), (50, 150)):
        d, i = index.search(Q[lo:hi], 20)
        assert np.array_equal(d, D[lo:hi]) and np.array_equal(i, I[lo:hi])
    index.close()


@pytest.mark.parametrize("nq", [1, 7, 40])
def test_equal_scores_go_to_the_lowest_id(ssa, nq):
    r = np.random.default_rng(SALT + 3)
    few = unit_rows(12, 200, SALT + 4)
    X = few[r.integers(0, 12, 900)]
    Q = unit_rows(nq, 200, SALT + 5)
    index = filled(ssa, X)
    check_search(*index.search(Q, 100), plain.round_rows(X), plain.round_rows(Q), 100)
    same = filled(ssa, np.repeat(few[:1], 500, axis=0))
    assert np.array_equal(same.search(Q, 30)[1], np.tile(np.arange(30), (nq, 1)))


@pytest.mark.parametrize("nq", [1, 6, 20])
def test_search_with_a_score_floor(ssa, nq):
    X, Q = unit_rows(2000, 256, SALT + 6), unit_rows(nq, 256, SALT + 7)
    index = filled(ssa, X)
    D, I = index.search(Q, 30)
    floor = float(np.sort(D.ravel())[D.size // 2])
    Df, If = index.search(Q, 30, min_score=floor)
    keep = D >= floor
    assert np.array_equal(If, np.where(keep, I, -1))
    assert np.array_equal(Df, np.where(keep, D, np.float32(-np.finfo(np.float32).max)))
    Dd, Id = index.search(ssa.quantize_f8(cuda(Q)), 30, min_score=floor)
    assert np.array_equal(Id.cpu().numpy(), If)
    assert (index.search(Q, 5, min_score=1e30)[1] == -1).all()


@pytest.mark.parametrize("nq", [1, 5, 20])
def test_rows_and_queries_that_are_not_finite_are_no_results(ssa, nq):
    X, Q = unit_rows(300, 260, SALT + 8), unit_rows(nq, 260, SALT + 9)
    X[17, 3], X[200, 259] = np.nan, np.inf
    Q[nq - 1, 0] = np.nan if nq > 1 else Q[0, 0]
    index = filled(ssa, X)
    with np.errstate(invalid="ignore"):
        check_search(*index.search(Q, 300), plain.round_rows(X), plain.round_rows(Q), 300)


def test_rows_in_many_segments(ssa, monkeypatch):
    monkeypatch.setenv("SSMI_SEG_SHIFT", "8")
    X = unit_rows(2100, 300, SALT + 10)
    index = ssa.IndexFlatIP(300, storage="f8")
    for lo, hi in ((0, 1), (1, 200), (200, 900), (900, 901), (901, 2100)):
        index.add(X[lo:hi] if lo % 2 else cuda(X[lo:hi]))
    X64 = plain.round_rows(X)
    for nq, k in ((1, 10), (5, 40), (70, 12)):
        Q = unit_rows(nq, 300, SALT + nq)
        check_search(*index.search(Q, k), X64, plain.round_rows(Q), k)
    ids = [0, 255, 256, 2099, 777]
    assert np.array_equal(index.reconstruct_batch(ids), X64[ids].astype(np.float32))


def test_add_of_every_kind_reconstruct_and_candidate_scores(ssa):
    X = unit_rows(70, 333, SALT + 11)
    index = ssa.IndexFlatIP(333, storage="f8")
    index.add(X[:20])
    index.add(cuda(X[20:30]))
    index.add(cuda(X[30:40], torch.float16))
    index.add(cuda(X[40:50], torch.bfloat16))
    index.add(ssa.quantize_f8(cuda(X[50:])))
    index.add(ssa.quantize_f8(cuda(X[:0])))
    want = X.astype(np.float64)
    want[30:40] = cuda(X[30:40], torch.float16).double().cpu().numpy()
    want[40:50] = cuda(X[40:50], torch.bfloat16).double().cpu().numpy()
    want = plain.round_rows(want)
    assert index.ntotal == 70
    assert np.array_equal(index.reconstruct_n(), want.astype(np.float32))
    assert np.array_equal(index.reconstruct_batch_device([3, 69]).cpu().numpy(), want[[3, 69]].astype(np.float32))
    N = unit_rows(4, 333, SALT + 12)
    got = index.score_ids([5, 69, 5], N)
    assert (np.abs(got - want[[5, 69, 5]] @ N.T.astype(np.float64)) <= 333 * 2.0 ** -24).all()   # unit rows, fp32 chains
    with pytest.raises(RuntimeError):
        index.reconstruct(70)


def test_files_keep_the_rows_bit_for_bit(ssa, tmp_path):
    X, Q = unit_rows(500, 200, SALT + 13), unit_rows(3, 200, SALT + 14)
    index = filled(ssa, X)
    path = str(tmp_path / "f8.faiss")
    ssa.write_index(index, path)
    index.add(X[:100])
    ssa.write_index(index, path, incremental=True)
    back = ssa.read_index(path, storage="f8")
    assert back.storage == "f8" and back.ntotal == 600
    assert np.array_equal(back.reconstruct_n(), index.reconstruct_n())
    for a, b in zip(back.search(Q, 9), index.search(Q, 9)):
        assert np.array_equal(a, b)
    wide = ssa.read_index(path)   # fp32 rows of the same values
    assert np.array_equal(wide.reconstruct_n(), index.reconstruct_n())


def test_random_unit_rows_and_an_empty_index(ssa):
    index = ssa.IndexFlatIP(500, storage="f8")
    D, I = index.search(unit_rows(2, 500, 1), 4)
    assert (I == -1).all()
    D, I = index.search(ssa.quantize_f8(cuda(unit_rows(2, 500, 1))), 4)
    assert (I == -1).all()
    index.add_random_unit(300, seed=5)
    ref = ssa.IndexFlatIP(500)
    ref.add_random_unit(300, seed=5)
    assert np.array_equal(index.reconstruct_n(), plain.round_rows(ref.reconstruct_n()).astype(np.float32))


def test_the_whole_path_on_another_stream(ssa):
    """Hidden states -> norm -> rows of an index and queries -> search, all on a stream of its own, then a second stream."""
    torch.manual_seed(SALT + 1)
    h, r = torch.randn(700, 1024, device="cuda").bfloat16(), torch.randn(700, 1024, device="cuda").bfloat16()
    w = torch.rand(1024, device="cuda").bfloat16() + 0.5
    _, y = norm64(h, r, w, 1e-6, True, torch.bfloat16)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    index = ssa.IndexFlatIP(1024, storage="f8")
    with torch.cuda.stream(s1):
        rows = ssa.rms_norm_f8(h, weight=w, residual=r, unit=True)
        index.add(rows)
        D, I = index.search(rows[5:12], 3)
        S = ssa.matmul_f8(rows[5:12], rows)
    s2.wait_stream(s1)
    with torch.cuda.stream(s2):
        D2, I2 = index.search(rows[:100], 3)
    torch.cuda.synchronize()
    X64 = rows64(rows)
    check_norm(rows, y)
    check_search(D, I, X64, X64[5:12], 3)
    check_search(D2, I2, X64, X64[:100], 3)
    assert (I[:, 0].cpu() == torch.arange(5, 12)).all()
    check_product(S, rows[5:12], rows)


def test_norm_and_products_in_a_graph(ssa):
    x = torch.randn(20, 512, device="cuda").bfloat16()
    res = torch.zeros_like(x)
    b = ssa.quantize_f8(torch.randn(300, 512, device="cuda"))
    big = ssa.quantize_f8(torch.randn(90, 512, device="cuda"))
    rows, out, out2 = ssa.F8Rows.empty(20, 512, "cuda"), torch.empty(20, 300, dtype=torch.float16, device="cuda"), torch.empty(90, 300, dtype=torch.bfloat16, device="cuda")

    def step():
        ssa.rms_norm_f8(x, residual=res, out=rows)
        ssa.matmul_f8(rows, b, out=out)
        ssa.matmul_f8(big, b, out=out2)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    res.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for _ in range(4):
        x.copy_(torch.randn_like(x, dtype=torch.float32))
        before = res.clone()
        g.replay()
        want_rows = ssa.rms_norm_f8(x, residual=before)
        assert torch.equal(before, res)
        assert torch.equal(out, ssa.matmul_f8(want_rows, b, out_dtype=torch.float16))
        assert torch.equal(out2, ssa.matmul_f8(big, b))
        torch.cuda.synchronize()


def test_factory_and_several_devices_take_the_storage(ssa):
    X, Q = unit_rows(400, 128, SALT + 15), unit_rows(2, 128, SALT + 16)
    made = ssa.IndexFactory.create_index(ssa.IndexConfig(index_type=ssa.IndexType.FLAT, dimension=128, extra={"storage": "f8"}))
    for index in (made, ssa.IndexFlatIP(128, storage="f8", devices=[0, 0])):
        index.add(X)
        check_search(*index.search(Q, 7), plain.round_rows(X), plain.round_rows(Q), 7)


def test_refusals_of_a_live_index(ssa):
    index = filled(ssa, unit_rows(50, 128, 1))
    plain_index = ssa.IndexFlatIP(128)
    q = cuda(unit_rows(2, 128, 2))
    rows = ssa.quantize_f8(q)
    with pytest.raises(RuntimeError, match="k=1009"):
        index.search(q, 1009)
    with pytest.raises(RuntimeError, match="k=1009"):
        index.search(rows, 1009)
    with pytest.raises(RuntimeError, match="search_static"):
        index.search_static(q, 3, (torch.empty(2, 3, device="cuda"), torch.empty(2, 3, dtype=torch.int64, device="cuda")))
    with pytest.raises(RuntimeError, match="8-bit"):
        plain_index.add(rows)
    with pytest.raises(RuntimeError, match="8-bit"):
        plain_index.search(rows, 3)
    with pytest.raises(AssertionError, match="dimension"):
        index.add(ssa.quantize_f8(q[:, :100]))
    with pytest.raises(RuntimeError, match="Flat"):
        ssa.IndexIVFFlat(None, 128, 4, storage="f8")


# one size at least for every tile (16 x 16 to 256 x 256), whole and ragged, and every length of their rings
@pytest.mark.parametrize("m,n", [(1, 4096), (16, 200), (97, 1000), (64, 4090), (128, 4096), (250, 4090), (512, 4096), (1000, 4090), (2040, 4096), (4090, 4096), (4100, 8200)])
@pytest.mark.parametrize("k", [100, 256, 300, 512, 513, 700, 1100])
def test_product_in_every_tile(ssa, m, n, k):
    torch.manual_seed(SALT + m + n + k)
    # -1, 0 and 1 times a power of two a row: every product and sum is exact, in whatever order
    xa, xb = (torch.randint(-1, 2, (c, k), device="cuda").float() for c in (m, n))
    xa[:, 0] = xb[:, 0] = 1
    sa, sb = (torch.exp2(torch.randint(-3, 4, (c, 1), device="cuda").float()) for c in (m, n))
    a, b = ssa.quantize_f8(xa * sa), ssa.quantize_f8(xb * sb)
    want = ((xa.double() @ xb.double().T) * sa.double() * sb.double().T).bfloat16()
    assert torch.equal(ssa.matmul_f8(a, b), want)


@pytest.mark.parametrize("n,d,nq,k", [(70000, 130, 129, 10), (140000, 64, 300, 49), (66000, 200, 700, 100), (40000, 128, 1025, 1), (513, 400, 200, 48), (20000, 1100, 150, 300),
                                      (70000, 64, 100, 10), (70000, 520, 20, 30),
                                      (140000, 64, 520, 10), (140000, 300, 400, 60), (128 * 1024 + 1, 130, 500, 48), (10000, 768, 900, 10)])
def test_search_of_large_batches_over_many_row_tiles(ssa, n, d, nq, k):
    X, Q = unit_rows(n, d, SALT + n + d), unit_rows(nq, d, SALT + nq)
    index = filled(ssa, cuda(X))
    check_search(*index.search(Q, k), plain.round_rows(X), plain.round_rows(Q), k)


@pytest.mark.parametrize("nq", [20, 100, 300, 800])
@pytest.mark.parametrize("k", [10, 60])
def test_search_of_rows_that_get_better_and_better(ssa, nq, k):
    """Every row tile beats all before it: each threshold is late.  The values are exact, with many equal ones."""
    n, d = 80000, 256
    X = np.zeros((n, d), np.float32)
    X[:, :5] = (np.arange(n)[:, None] // 160 >> np.arange(8, -1, -2) & 3) * 4.0 ** np.arange(4, -1, -1)   # digits of base 4 that add up to i // 160
    X[:, 128:133] = X[:, :5]
    Q = np.zeros((nq, d), np.float32)
    Q[np.arange(nq) % 3 != 1, :5] = 1
    Q[np.arange(nq) % 3 != 0, 128:133] = 1
    Q[:, 200] = np.arange(nq)   # (no row answers to it)
    check_search(*filled(ssa, X).search(Q, k), plain.round_rows(X), plain.round_rows(Q), k)


def test_large_batches_over_many_segments(ssa, monkeypatch):
    monkeypatch.setenv("SSMI_SEG_SHIFT", "8")
    X, Q = unit_rows(20000, 300, SALT + 20), unit_rows(310, 300, SALT + 21)
    index = filled(ssa, X)
    for nq in (16, 128, 310):
        check_search(*index.search(Q[:nq], 12), plain.round_rows(X), plain.round_rows(Q[:nq]), 12)
    monkeypatch.setenv("SSMI_SEG_SHIFT", "11")
    X, Q = unit_rows(120000, 64, SALT + 24), unit_rows(560, 64, SALT + 25)
    check_search(*filled(ssa, X).search(Q, 12), plain.round_rows(X), plain.round_rows(Q), 12)


@pytest.mark.parametrize("n,nq", [(3000, 12), (3000, 100), (3000, 300), (130000, 520)])
def test_large_batches_of_rows_and_queries_that_are_not_finite(ssa, n, nq):
    X, Q = unit_rows(n, 256, SALT + 22), unit_rows(nq, 256, SALT + 23)
    X[::2, 7] = np.nan    # half the rows of every tile
    X[1:600:2, 200] = np.inf
    Q[3, 0] = np.nan
    with np.errstate(invalid="ignore"):
        check_search(*filled(ssa, X).search(Q, 10), plain.round_rows(X), plain.round_rows(Q), 10)


def test_an_index_over_several_devices_refuses_rows_that_are_8_bit_already(ssa):
    rows = ssa.quantize_f8(cuda(unit_rows(5, 128, 3)))
    index = ssa.IndexFlatIP(128, storage="f8", devices=[0, 0])
    for call in (lambda: index.add(rows), lambda: index.search(rows, 2)):
        with pytest.raises(RuntimeError, match="plain rows"):
            call()


def test_the_manager_keeps_8_bit_rows(ssa, tmp_path):
    """add / search / save / reload / compact of the manager over 8-bit rows: what an index of the rounded rows gives."""
    from semantic_search_amd.index_manager import SemanticIndex
    d, n = 96, 600
    X, q = unit_rows(n, d, SALT + 30), unit_rows(1, d, SALT + 31)[0]
    make = lambda: SemanticIndex("eight", d, "flat", base_path=tmp_path, check_files_exist=False, storage="f8")  # noqa: E731
    ix = make()
    for s in range(0, n, 50):
        ix.add_vectors(X[s:s + 50], [f"/img/{i}.jpg" for i in range(s, s + 50)], [""] * 50, [(0.0, 0)] * 50)
    ids = lambda r: [(x.vector_id, x.file_path) for x in r.results]  # noqa: E731
    _, want = plain.search(plain.round_rows(X), plain.round_rows(q[None]), 20)
    assert [i for i, _ in ids(ix.search(q, 20))] == want[0].tolist()
    first = ids(ix.search(q, 20))
    ix.save()
    ix.close()
    ix = make()
    assert ix._faiss_index.storage == "f8" and ids(ix.search(q, 20)) == first
    for i in range(0, n, 3):
        assert ix.db.remove_image(f"/img/{i}.jpg")
    assert ix.compact()["success"]
    left = np.array([i for i in range(n) if i % 3])
    assert ix._faiss_index.storage == "f8" and ix._faiss_index.ntotal == len(left)
    _, want = plain.search(plain.round_rows(X[left]), plain.round_rows(q[None]), 20)
    assert [p for _, p in ids(ix.search(q, 20))] == [f"/img/{left[i]}.jpg" for i in want[0]]
    ix.close()


def test_two_graphs_and_eager_products_at_once(ssa):
    """Products and norms keep nothing between calls: two captured graphs and eager work on three streams do not meet."""
    torch.manual_seed(SALT + 32)
    b = ssa.quantize_f8(torch.randn(4096, 1024, device="cuda"))
    sets = []
    for m in (1, 40, 700):
        x = torch.randn(m, 1024, device="cuda").bfloat16()
        rows, out = ssa.F8Rows.empty(m, 1024, "cuda"), torch.empty(m, 4096, dtype=torch.bfloat16, device="cuda")
        sets.append((x, rows, out, ssa.matmul_f8(ssa.rms_norm_f8(x), b)))

    def step(s):
        ssa.rms_norm_f8(s[0], out=s[1])
        ssa.matmul_f8(s[1], b, out=s[2])
    torch.cuda.synchronize()
    graphs = []
    for s in sets[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(s)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        for s in sets:
            s[2].zero_()
        torch.cuda.synchronize()
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                graphs[i].replay() if i < 2 else step(sets[2])
        torch.cuda.synchronize()
        for s in sets:
            assert torch.equal(s[2], s[3])


def test_one_operand_twice_and_wide_strides(ssa):
    x = torch.randn(300, 500, device="cuda")
    a = ssa.quantize_f8(x)
    s = ssa.matmul_f8(a, a)
    assert torch.equal(s, s.T.contiguous())
    # rows far apart in one allocation: every 7th row of a table, by its strides
    wide = torch.zeros(300 * 7, 512, dtype=torch.uint8, device="cuda")
    wide_s = torch.zeros(300 * 7, 4, dtype=torch.uint8, device="cuda")
    wide[::7], wide_s[::7] = a.codes.view(torch.uint8), a.scales
    far = ssa.F8Rows.from_parts(wide[::7], wide_s[::7], 500)
    assert far.codes.stride(0) == 7 * 512
    assert torch.equal(ssa.matmul_f8(far, a), s) and torch.equal(far.dequantize(), a.dequantize())
    with pytest.raises(TypeError, match="tensor"):
        ssa.matmul_f8(a, a, out=[1])
