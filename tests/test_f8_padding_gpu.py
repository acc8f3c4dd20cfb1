"""Codes behind the last element of a row: whatever a caller has there, it is not part of the row and not written."""
import numpy as np
import pytest
import torch

import f8_plain as plain
from conftest import SALT, unit_rows

pytestmark = pytest.mark.gpu


def padded(ssa, n, d, seed):
    """Rows as the quantiser makes them, and the same codes with other ones behind them (NaN among them)."""
    x = torch.from_numpy(unit_rows(n, d, SALT + seed)).cuda()
    rows = ssa.quantize_f8(x)
    dirty = rows.codes.view(torch.uint8).clone()
    dirty[:, d:] = torch.randint(0, 256, (n, dirty.shape[1] - d), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(torch.uint8)
    return rows, dirty


@pytest.mark.parametrize("d", [1, 100, 200, 300])
def test_rows_from_parts_leave_the_parts_alone(ssa, d):
    rows, dirty = padded(ssa, 40, d, 1)
    other, _ = padded(ssa, 30, d, 2)
    before, scales, version = dirty.clone(), rows.scales.clone(), dirty._version
    made = ssa.F8Rows.from_parts(dirty, scales, d)
    assert torch.equal(dirty, before) and dirty._version == version and made.codes.data_ptr() != dirty.data_ptr()
    assert torch.equal(made.dequantize(), rows.dequantize())
    assert torch.equal(ssa.matmul_f8(made, other), ssa.matmul_f8(rows, other))
    clean = rows.codes.view(torch.uint8)
    assert ssa.F8Rows.from_parts(clean, scales, d).codes.data_ptr() == clean.data_ptr()   # nothing to hide: as it is


def test_rows_from_parts_while_a_graph_is_captured(ssa):
    rows, dirty = padded(ssa, 40, 200, 3)
    other, _ = padded(ssa, 30, 200, 4)
    scales = rows.scales.clone()
    out = torch.empty(40, 30, dtype=torch.bfloat16, device="cuda")
    ssa.matmul_f8(ssa.F8Rows.from_parts(dirty, scales, 200), other, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ssa.matmul_f8(ssa.F8Rows.from_parts(dirty, scales, 200), other, out=out)
    want = ssa.matmul_f8(rows, other)
    for _ in range(3):
        out.zero_()
        g.replay()
        assert torch.equal(out, want)
        torch.cuda.synchronize()


def index_of(ssa, d, rows, dirty):
    """An index whose rows came through the C entry point with codes behind them."""
    from semantic_search_amd import _lib
    index = ssa.IndexFlatIP(d, storage="f8")
    scales = rows.scales.contiguous()
    torch.cuda.synchronize()
    _lib.check(_lib.load().ssmi_index_add_f8(index._handle(), len(rows), dirty.data_ptr(), dirty.stride(0), scales.data_ptr(), scales.stride(0)))
    return index


@pytest.mark.parametrize("d", [1, 100, 200, 300])
def test_an_index_does_not_keep_codes_behind_its_rows(ssa, d, monkeypatch):
    monkeypatch.setenv("SSMI_SEG_SHIFT", "8")
    rows, dirty = padded(ssa, 700, d, 5)
    before = dirty.clone()
    index = index_of(ssa, d, rows, dirty)
    assert torch.equal(dirty, before)
    X = plain.values(rows.codes.view(torch.uint8).cpu().numpy(), rows.scales.cpu().numpy(), d)
    for nq in (1, 5, 60, 300):
        queries, dirty_q = padded(ssa, nq, d, 6 + nq)
        Q = plain.values(queries.codes.view(torch.uint8).cpu().numpy(), queries.scales.cpu().numpy(), d)
        want = plain.search(X, Q, 9)[1]
        assert np.array_equal(index.search(queries, 9)[1].cpu().numpy(), want)
        assert np.array_equal(index.search(ssa.F8Rows.from_parts(dirty_q, queries.scales, d), 9)[1].cpu().numpy(), want)
