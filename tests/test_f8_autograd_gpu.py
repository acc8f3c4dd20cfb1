"""The 8-bit operators write through pointers: torch has to hear of it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def saved_by_a_graph(t):
    """A scalar whose backward pass needs the values that t holds now."""
    return (torch.ones_like(t, requires_grad=True) * t).sum()


@pytest.mark.parametrize("which", ["residual", "residual_out", "x", "out"])
def test_a_backward_pass_that_saved_what_is_overwritten_raises(ssa, which):
    x, r, ro = (torch.randn(5, 300, device="cuda") for _ in range(3))
    a, out = ssa.quantize_f8(x), torch.randn(5, 5, device="cuda").half()
    loss = saved_by_a_graph({"residual": r, "residual_out": ro, "x": x, "out": out}[which])
    untouched = saved_by_a_graph(r if which != "residual" else x)
    if which == "out":
        assert ssa.matmul_f8(a, a, out=out) is out
    else:
        ssa.rms_norm_f8(x, residual=r, residual_out={"residual": None, "residual_out": ro, "x": x}[which])
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    untouched.backward()


def test_rows_that_are_written_again_count_as_changed(ssa):
    x = torch.randn(5, 300, device="cuda")
    codes, scales = torch.zeros(5, 384, dtype=torch.uint8, device="cuda"), torch.zeros(5, 4, dtype=torch.uint8, device="cuda")
    for rows, seen in ((ssa.F8Rows.empty(5, 300, "cuda"), None), (ssa.F8Rows.from_parts(codes, scales, 300), scales)):
        for call in (lambda: ssa.quantize_f8(x, out=rows), lambda: ssa.rms_norm_f8(x, out=rows)):
            before = rows.codes._version, rows.scales._version
            call()
            assert rows.codes._version > before[0] and rows.scales._version > before[1]
    assert scales._version > 0


def test_outputs_that_require_a_gradient_are_refused_where_one_would_be_lost(ssa):
    x, r = torch.randn(5, 300, device="cuda"), torch.randn(5, 300, device="cuda", requires_grad=True)
    a, out = ssa.quantize_f8(x), torch.randn(5, 5, device="cuda", dtype=torch.float16, requires_grad=True)
    before = r.detach().clone()
    for call in (lambda: ssa.rms_norm_f8(x, residual=r), lambda: ssa.rms_norm_f8(x, residual=x, residual_out=r), lambda: ssa.matmul_f8(a, a, out=out)):
        with pytest.raises(ValueError, match="requires one"):
            call()
    assert torch.equal(r, before)
    ssa.rms_norm_f8(x, weight=torch.ones(300, device="cuda", requires_grad=True), residual=r, residual_out=torch.empty_like(x))   # inputs may
    with torch.no_grad():
        ssa.rms_norm_f8(x, residual=r)
        ssa.matmul_f8(a, a, out=out)
    assert not torch.equal(r, before)
    with torch.inference_mode():
        y = torch.randn(5, 300, device="cuda")
        ssa.rms_norm_f8(x, residual=y)
