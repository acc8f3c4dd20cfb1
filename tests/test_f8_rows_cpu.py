"""What F8Rows takes as it is, on the CPU: no kernel reads it here."""
import pytest
import torch


def parts(n=3, blocks=2, words=4):
    return torch.zeros(n, blocks * 128, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(n, words, dtype=torch.uint8)


def test_rows_in_the_layout_of_the_kernels_are_taken(ssa):
    c, s = parts()
    for d in (129, 200, 256):
        rows = ssa.F8Rows(c, s, d)
        assert len(rows) == 3 and rows.codes.data_ptr() == c.data_ptr() and rows[1:2].d == d
    ssa.F8Rows(c[:0], s[:0], 256)
    ssa.F8Rows(c[1:2], s[1:2], 256)
    wide, words = parts(9, 4, 12)
    rows = ssa.F8Rows(wide[::3, 128:384], words[::3, 4:8], 256)   # every third row, the middle of it
    assert rows._args[1] == 3 * 512 and rows._args[3] == 3 * 12


@pytest.mark.parametrize("case", ["columns apart", "scale columns apart", "short codes", "short scales", "rows", "unaligned codes", "unaligned scales",
                                  "stride", "scale stride", "repeated row", "type", "scale type", "dimensions", "no tensor", "d", "transposed"])
def test_other_layouts_are_refused(ssa, case):
    c, s = parts()
    d = 200
    u8 = c.view(torch.uint8)
    f8 = torch.float8_e4m3fn
    if case == "columns apart":
        c = torch.zeros(3, 512, dtype=torch.uint8).view(f8)[:, ::2]
    elif case == "scale columns apart":
        s = torch.zeros(3, 8, dtype=torch.uint8)[:, ::2]
    elif case == "short codes":
        c = c[:, :200]
    elif case == "short scales":
        s = s[:, :2]
    elif case == "rows":
        s = s[:2]
    elif case == "unaligned codes":
        c = torch.zeros(3, 272, dtype=torch.uint8).view(f8)[:, 1:257]
    elif case == "unaligned scales":
        s = torch.zeros(3, 8, dtype=torch.uint8)[:, 1:5]
    elif case == "stride":
        c = torch.zeros(3, 264, dtype=torch.uint8).view(f8)[:, :256]
    elif case == "scale stride":
        s = torch.zeros(3, 6, dtype=torch.uint8)[:, :4]
    elif case == "repeated row":
        c = c[:1].expand(3, 256)
    elif case == "type":
        c = u8
    elif case == "scale type":
        s = s.to(torch.int32)
    elif case == "dimensions":
        c = c[0]
    elif case == "no tensor":
        s = [1, 2]
    elif case == "d":
        d = 0
    elif case == "transposed":
        c = torch.zeros(256, 3, dtype=torch.uint8).view(f8).t()
    with pytest.raises(ValueError, match="F8Rows"):
        ssa.F8Rows(c, s, d)
