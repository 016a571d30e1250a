"""Values at the ends of float32's range in the experts' MLP of 128 hidden units:
a factor above 3.396e38 rounds to an infinity in bfloat16, and no result may show
that.  Against float64; u = 2^-24, a float32 sum of n products within (n + 8) 2 u
of the sum of their absolute values."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TOP = torch.finfo(torch.float32).max
COLS, OUTS, ROWS, HIDDEN = 40, 12, 100, 128


def _bound(n):
    return (n + 8) * 2 * U


def _within(name, got, ref, bound):
    err = (got.double() - ref).abs()
    limit = bound + U * ref.abs() + torch.finfo(torch.float32).tiny
    assert (err <= limit).all(), f"{name}: {(err / limit).nan_to_num(1e300).max().item():.3g} bounds off"


def _largest_input(x, dy, w1, w2):
    """A mask's lowest and largest value in one column, in rows without an upstream and in others."""
    x[3, 7], x[4, 7], x[50, 7], x[51, 7] = -TOP, TOP, -TOP, 3.4e38
    w1[:, :, 7] *= 1e-3
    dy[3:5], dy[50:52] = 0, 1e-6 * dy[50:52]


def _largest_hidden(x, dy, w1, w2):
    """One hidden unit, of one row, above 3.396e38."""
    x[20], w1[:, 9] = 0, 0
    x[20, 5], w1[:, 9, 5] = 3.4e38, 1
    w1[:, :9, 5], w1[:, 10:, 5] = 0, 0
    w2[:, :, 9] = 1e-3
    dy[20] *= 1e-6


def _largest_upstream(x, dy, w1, w2):
    """Rows whose upstream, and its product with W2, lie above 3.396e38 in one place."""
    dy[30], dy[31] = 0, 0
    dy[30, 2], dy[31, 3] = 3.4e38, -TOP
    w2[:, 2], w2[:, 3] = 0, 0
    w2[:, 2, 11], w2[:, 3, 11] = 1, 1
    x[30:32] *= 1e-3
    w1 *= 1e-3


@pytest.mark.parametrize("change", [_largest_input, _largest_hidden, _largest_upstream])
def test_fused_mlp_of_the_largest_values(change):
    from npa_amd import experts as E
    g = torch.Generator(device="cuda").manual_seed(1)
    randn = lambda *s: torch.randn(*s, dtype=torch.float32, device="cuda", generator=g)
    x, dy = randn(ROWS, COLS), randn(ROWS, OUTS)
    w1, w2 = randn(2, HIDDEN, COLS) / COLS ** 0.5, randn(2, OUTS, HIDDEN) / HIDDEN ** 0.5
    b1, b2 = 0.1 * randn(2, HIDDEN), 0.1 * randn(2, OUTS)
    if change is _largest_upstream:
        b1 *= 0.1  # dy times the hidden value stays in range
    change(x, dy, w1, w2)
    at = [0, 60, ROWS]
    offsets = torch.tensor(at, dtype=torch.int32, device="cuda")
    wide = [t.double() for t in (x, w1, b1, w2, b2)]
    for e in range(2):  # rows with a hidden value within rounding of 0 get no upstream
        s = slice(at[e], at[e + 1])
        a = wide[0][s] @ wide[1][e].T + wide[2][e]
        near = (a.abs() <= 2 * _bound(COLS) * (wide[0][s].abs() @ wide[1][e].abs().T + wide[2][e].abs())).any(1)
        dy[s][near] = 0
    leaves = [t.requires_grad_(True) for t in (x, w1, b1, w2, b2)]
    y = E.mlp(*leaves, offsets)
    dx, dw1, db1, dw2, db2 = torch.autograd.grad(y, leaves, dy)
    for e in range(2):
        s = slice(at[e], at[e + 1])
        n = at[e + 1] - at[e]
        xd, up, w1d, w2d = wide[0][s], dy[s].double(), wide[1][e], wide[3][e]
        a = xd @ w1d.T + wide[2][e]
        ea = _bound(COLS) * (xd.abs() @ w1d.abs().T + wide[2][e].abs())
        h = a.clamp_min(0)
        eh = torch.where(a > -ea, ea, torch.zeros_like(ea))
        _within("y", y.detach()[s], h @ w2d.T + wide[4][e],
                _bound(HIDDEN) * (h @ w2d.abs().T + wide[4][e].abs()) + eh @ w2d.abs().T)
        on = (a > 0).double()
        dh, edh = (up @ w2d) * on, _bound(OUTS) * (up.abs() @ w2d.abs()) * on
        _within("dx", dx[s], dh @ w1d, _bound(HIDDEN) * (dh.abs() @ w1d.abs()) + edh @ w1d.abs())
        _within("dW1", dw1[e], dh.T @ xd, _bound(n) * (dh.abs().T @ xd.abs()) + edh.T @ xd.abs())
        _within("db1", db1[e], dh.sum(0), _bound(n) * dh.abs().sum(0) + edh.sum(0))
        _within("dW2", dw2[e], up.T @ h, _bound(n) * (up.abs().T @ h) + up.abs().T @ eh)
        _within("db2", db2[e], up.sum(0), _bound(n) * up.abs().sum(0))
