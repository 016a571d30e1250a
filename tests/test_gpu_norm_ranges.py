"""Layer norm of rows at the ends of their type's range (npa_amd.norm): a finite
row the squares of whose deviations pass float32's range gives the bias and no
gradient to x, masks of the lowest value among them; other rows are as ever."""
import pytest
import torch
from test_gpu_norm import BF16, F16, F32, U, _case, _check, _reference, _within

pytestmark = pytest.mark.gpu


def _large_rows(x):
    """Rows of x whose squared deviations overflow, in place; their numbers."""
    top, cols = torch.finfo(x.dtype).max, x.shape[1]
    x[0, 0] = -top                      # a mask of one place
    x[1, 1:3] = -top                    # of two: their sum overflows
    x[2, :cols // 2] = -top             # of half of the row
    x[3] = -top                         # largest values of one sign: one that differs
    x[3, cols - 1] = top
    x[4] = top
    x[4, 0] = -top
    x[5, ::2], x[5, 1::2] = top, -top   # and of both
    x[6, cols // 3] = 1e25
    return range(7)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [8, 31, 83, 200, 1000, 4097, 6145, 9000, 20000, 65536])
def test_rows_whose_squares_overflow(cols, dtype):
    from npa_amd import norm
    x, w, b, dy = _case(40, cols, dtype, True, cols)
    large = list(_large_rows(x))
    fine = [i for i in range(40) if i not in large]
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = norm.layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(y[large], b.detach().to(dtype).expand(len(large), cols)) and not dx[large].any()
    ry, rx, rw, rb = _reference(x.detach()[fine], w.detach(), b.detach(), 1e-5, dy[fine])
    _within("y", y.detach()[fine], *ry)
    _within("dx", dx[fine], *rx)
    _within("dw", dw, *rw)
    sums = dy.double().sum(0)
    _within("db", db, sums, (40 / 512 + 176) * U * dy.double().abs().sum(0))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [31, 83, 4097, 20000])
def test_rows_of_one_large_value(cols, dtype):
    """No deviations but the rounding of the mean: y is the bias, whatever of x's gradient is left is finite."""
    from npa_amd import norm
    x, w, b, dy = _case(6, cols, dtype)
    top = torch.finfo(dtype).max
    for i, v in enumerate((top, -top, 1e38, -3e37, 1e30, 2.0 ** 100)):
        x[i] = v
    x.requires_grad_(True)
    y = norm.layer_norm(x, w, b)
    # a deviation that is a rounding of the mean alone: all of a row's are alike, and their mean is taken off
    assert (y.detach().float() - b).abs().max() <= 1e-2 + 2.0 ** -8 * b.abs().max()
    assert torch.isfinite(torch.autograd.grad(y, x, dy)[0]).all()


@pytest.mark.parametrize("size", [1e10, 1e15, 1e17])
def test_large_rows_in_range(size):
    for cols in (83, 4097, 9000):
        x, w, b, dy = _case(30, cols, F32)
        _check(x * size, w, b, dy)


def test_small_rows():
    """Deviations far below eps, and with eps = 0."""
    for cols in (83, 9000):
        x, w, b, dy = _case(30, cols, F32)
        _check(x * 1e-12, w, b, dy)
        _check(x * 1e-12, w, b, dy, eps=0.0)


@pytest.mark.parametrize("cols", [83, 4097, 20000])
def test_float16_masks(cols):
    """float16's lowest value squared is well inside float32's range: rows like any others."""
    x, w, b, dy = _case(40, cols, F16, True)
    x[0, 0], x[1, 1:3], x[2, :cols // 2] = -65504, -65504, -65504
    x[3] = -65504
    x[3, 5] = 65504
    _check(x, w, b, dy)


@pytest.mark.parametrize("cols", [83, 4097, 20000])
def test_rows_that_are_not_finite_beside_large_ones(cols):
    from npa_amd import norm
    x, w, b, dy = _case(6, cols, F32)
    x[:, :5] = torch.finfo(F32).min
    x[1, 7], x[2, 7], x[3, 7] = float("inf"), float("-inf"), float("nan")
    x[4] = float("inf")
    y = norm.layer_norm(x, w, b)
    assert torch.isnan(y[1:5]).all() and torch.equal(y[[0, 5]], b.expand(2, cols))
