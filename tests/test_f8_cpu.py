"""8-bit rows without a GPU: the plain form against itself, and what the entry points refuse before they touch a device."""
import ctypes

import numpy as np
import pytest
import torch

import f8_plain as plain
from conftest import unit_rows


def test_plain_form_agrees_with_the_cast_of_torch():
    x = (np.random.default_rng(0).standard_normal((50, 300)) * np.exp(np.random.default_rng(1).standard_normal((50, 1)) * 3)).astype(np.float32)
    c, s = plain.quantize(x)
    v = np.zeros((50, 384), dtype=np.float32)
    v[:, :300] = x
    u = torch.from_numpy(v.reshape(50, 3, 128) * np.ldexp(np.float32(1), 127 - s.astype(int))[..., None].astype(np.float32))
    assert np.array_equal(u.to(torch.float8_e4m3fn).view(torch.uint8).numpy().reshape(50, 384), c)
    r = plain.values(c, s, 300)
    assert (np.abs(r - x) <= np.abs(x) * 2.0 ** -4 + np.repeat(np.ldexp(1.0, s.astype(int) - 127), 128, axis=1)[:, :300] * 2.0 ** -10).all()
    # the same values again (a block whose largest code rounded down to 224 may come back with half the scale and twice the codes)
    assert np.array_equal(plain.round_rows(r), r)


def rows(lib, name, *a):
    rc = getattr(lib, name)(*a)
    return rc, lib.ssmi_last_error().decode()


GOOD = dict(codes=4096, stride=256, scales=4096, sstride=4)


@pytest.mark.parametrize("change,text", [
    (dict(codes=None), "NULL"), (dict(scales=None), "NULL"), (dict(codes=4097), "16-byte"), (dict(scales=4098), "4-byte"),
    (dict(stride=128), "multiple of 16"), (dict(stride=264), "multiple of 16"), (dict(stride=1 << 24), "at most"),
    (dict(sstride=0), "multiple of 4"), (dict(sstride=6), "multiple of 4"), (dict(n=-1), "negative"), (dict(n=1 << 27), "exceed"),
    (dict(d=0), "dimension"), (dict(d=65537), "dimension")])
def test_bad_8_bit_rows_are_refused(ssa, change, text):
    from semantic_search_amd import _lib
    lib = _lib.load()
    a = dict(GOOD, n=3, d=200) | change
    m = (a["codes"], a["stride"], a["scales"], a["sstride"])
    rc, msg = rows(lib, "ssmi_f8_quantize", 0, a["n"], a["d"], 4096, _lib.F32, max(a["d"], 1), *m, None)
    assert rc and text in msg
    rc, msg = rows(lib, "ssmi_f8_dequantize", 0, a["n"], a["d"], *m, 4096, _lib.F32, max(a["d"], 1), None)
    assert rc and text in msg
    rc, msg = rows(lib, "ssmi_f8_rms_norm", 0, a["n"], a["d"], 4096, _lib.F32, max(a["d"], 1), None, 0, None, 0, None, 0, 1e-6, 0, *m, None)
    assert rc and text in msg
    good = (GOOD["codes"], max(256, 65536 if a["d"] > 256 else 256), GOOD["scales"], 512)
    rc, msg = rows(lib, "ssmi_f8_matmul", 0, 3, a["n"], a["d"], *good, *m, 4096, _lib.BF16, 1 << 28, None)
    assert rc and text in msg


def test_bad_plain_rows_and_outputs_are_refused(ssa):
    from semantic_search_amd import _lib
    lib = _lib.load()
    m = tuple(GOOD.values())
    norm = lambda **k: rows(lib, "ssmi_f8_rms_norm", 0, 3, 200, k.get("x", 4096), k.get("dtype", 0), k.get("xs", 200), k.get("r"), k.get("rs", 200),  # noqa: E731
                            k.get("ro"), k.get("ros", 200), k.get("w"), k.get("wd", 0), k.get("eps", 1e-6), 0, *m, None)
    for kw, text in ((dict(x=None), "NULL"), (dict(dtype=3), "dtype"), (dict(xs=199), "stride"), (dict(x=4098), "aligned"), (dict(r=4096), "residual_out"),
                     (dict(ro=4096), "without"), (dict(r=4096, ro=4096, ros=100), "stride"), (dict(w=4096, wd=7), "dtype"), (dict(w=4097, wd=1), "aligned"),
                     (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps")):
        rc, msg = norm(**kw)
        assert rc and text in msg, (kw, msg)
    mm = lambda **k: rows(lib, "ssmi_f8_matmul", 0, 3, 5, 200, *m, *m, k.get("out", 4096), k.get("dtype", 2), k.get("os", 5), None)  # noqa: E731
    for kw, text in ((dict(dtype=0), "fp16 or bf16"), (dict(dtype=3), "fp16 or bf16"), (dict(os=4), "stride"), (dict(out=None), "NULL"), (dict(out=4097), "aligned")):
        rc, msg = mm(**kw)
        assert rc and text in msg, (kw, msg)
    for name, a in (("ssmi_index_add_f8", (None, 1, *m)), ("ssmi_index_search_f8", (None, 1, *m, 5, 0.0, None, None, 0, None))):
        rc, msg = rows(lib, name, *a)
        assert rc and "NULL index" in msg
    # nothing to do is no error
    assert lib.ssmi_f8_quantize(0, 0, 200, None, 0, 200, None, 256, None, 4, None) == 0
    assert lib.ssmi_f8_matmul(0, 0, 5, 200, None, 256, None, 4, *m, 4096, 2, 5, None) == 0


def test_python_refusals(ssa):
    x = torch.zeros(3, 200)
    with pytest.raises(ValueError, match="ROCm"):
        ssa.quantize_f8(x)
    with pytest.raises(TypeError, match="torch tensor"):
        ssa.rms_norm_f8(np.zeros((3, 200), dtype=np.float32))
    with pytest.raises(TypeError, match="F8Rows"):
        ssa.matmul_f8(x, x)
    c, s = torch.zeros(3, 256, dtype=torch.uint8), torch.zeros(3, 4, dtype=torch.uint8)
    with pytest.raises(ValueError, match="ROCm"):
        ssa.F8Rows.from_parts(c, s, 200)
    with pytest.raises(ValueError, match="as many rows"):
        ssa.F8Rows.from_parts(c, s[:2], 200)
    a = ssa.F8Rows(c.view(torch.float8_e4m3fn), s, 200)
    with pytest.raises(ValueError, match="elements"):
        ssa.matmul_f8(a, ssa.F8Rows(c.view(torch.float8_e4m3fn), s, 201))
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        ssa.matmul_f8(a, a, out_dtype=torch.float32)
    with pytest.raises(TypeError, match="slices"):
        a[1]
    assert len(a[1:]) == 2 and a[1:].d == 200


def test_plain_search_orders_ties_by_id():
    X = unit_rows(3, 16, 1)[[0, 1, 0, 2]].astype(np.float64)
    D, I = plain.search(X, X[:1], 6)
    assert I[0, :2].tolist() == [0, 2] and I[0, 4:].tolist() == [-1, -1] and D[0, 4] < -3e38
