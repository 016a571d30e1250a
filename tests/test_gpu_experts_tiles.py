"""Layers of experts on both sides of the rules that choose their kernels."""
import pytest
from test_gpu_experts import BF16, F16, F32, _check_linear

import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_few_rows(dtype):
    """Weights past LDS, and tiles where the products or the workgroups are many."""
    _check_linear([3, 0, 9, 1, 15, 0, 1, 1], 2, 2048, 1100, dtype)
    _check_linear([16, 0, 2, 30, 1, 15, 16, 1], 9, 1025, 2048, dtype)
    _check_linear([40, 0, 23, 16, 1, 7, 16, 19], 6, 2047, 2050, dtype, bias=False)
    _check_linear([0, 2] * 120 + [11] * 40, 5, 24, 130, dtype)
    _check_linear([4] * 250, 3, 83, 128, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_both_kernels_of_few_rows_agree(dtype):
    """A row's result from either kernel: 1024 places of 64 experts and the first 60 of them."""
    from npa_amd import experts as E
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(1024, 1024, device="cuda", generator=g).to(dtype)
    w = (torch.randn(64, 1024, 1024, device="cuda", generator=g) / 32).to(dtype)
    offsets = torch.arange(0, 1025, 16, dtype=torch.int32, device="cuda")
    y = E.linear(x, w, None, offsets)
    few = E.linear(x[:60], w, None, offsets.clamp_max(60))
    # two float32 sums of 1024 products, each within (1024 + 8) 2 u of the sum of absolute values, each rounded once
    size = torch.cat([x[i:i + 1].double().abs() @ w[i // 16].double().abs().T for i in range(60)])
    half = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
    limit = 2 * 1032 * 2 * 2.0 ** -24 * size + 2 * half * (few.double().abs() + 1032 * 2 * 2.0 ** -24 * size)
    assert ((y[:60].double() - few.double()).abs() <= limit).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_weight_gradients_whole_and_in_chunks(dtype):
    """Weight tiles that fill the card, up to 32768 places and past them, rows laid out or as they are."""
    for rows in (32768, 32769):
        _check_linear([rows // 2, 0, *[rows // 32] * 14, 100], rows - rows // 2 - 14 * (rows // 32) - 100, 776, 760, dtype)
    counts = [500] * 36 + [0, 7, 333]
    _check_linear(counts, 5, 513, 520, dtype, bias=False)
    _check_linear(counts + [14600], 5, 513, 520, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("counts", [[4095, 9, 700], [33000, 9, 700]])
def test_large_weight_tiles(counts, dtype):
    """16-bit weight gradients in tiles of 256: whole, and in chunks."""
    _check_linear(counts, 5, 4000, 4080, dtype)
