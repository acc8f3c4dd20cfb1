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
