"""The MLP trained with its input in 8 bits where sizes differ: columns, hidden
units, outputs, rows, weights, biases and upstreams over the range of float32.

y is that of the float32 MLP at z itself, the gradients those at the kept rows,
each within the roundings of float32 sums: an fp32 sum of n products is within (n
+ 8) 2^-24 of the sum of their absolute values (8: the roundings of the factors'
pieces and of the joining of partial sums).  The bounds are each element's own, so
sizes elsewhere in the row, the weights or the other hidden units buy nothing."""
import pytest
import torch

from test_gpu_int8 import EPS, _gen, _kept, _net

pytestmark = pytest.mark.gpu

TINY = 2.0 ** -120  # what subnormal pieces of a product may lose
LOWEST = torch.finfo(torch.float32).min
SHAPES = [(83, 19), (163, 35), (4, 4), (33, 40), (130, 33), (168, 64), (161, 32), (100, 64)]


def _within(name, got, ref, bound):
    err = (got.double() - ref).abs()
    over = ~(err <= bound + TINY)
    assert not over.any(), f"{name}: {int(over.sum())} elements, worst {(err / (bound + TINY)).nan_to_num(1e300).max().item():.3g} bounds off"


def _case(shape, rows, seed=0):
    net, g = _net(*shape, True, seed + sum(shape))
    z = torch.randn(rows, shape[0], device="cuda", generator=g)
    up = torch.randn(rows, shape[1], device="cuda", generator=g)
    return net, z, up


def _check(net, z, up, skip=()):
    from npa_amd import mlp as M
    rows, nin = z.shape
    nout = up.shape[1]
    w1, b1, w2, b2 = (p.detach().double() for p in net.parameters())

    def hidden(v):
        """Pre-activations, their bound, and the bound where the ReLU lets anything through."""
        a, e = v @ w1.T + b1, (nin + 8) * EPS * (v.abs() @ w1.abs().T + b1.abs())
        return a, e, torch.where(a > -e, e, torch.zeros_like(e))

    zd = _kept(z)
    a, ea, el = hidden(zd)
    up = up.clone()
    up[((a.abs() <= 2 * ea) & torch.isfinite(a)).any(1)] = 0  # within rounding of the ReLU's kink
    assert (up != 0).any(1).sum() * 2 >= rows
    zr = z.clone().requires_grad_(True)
    y = M.mlp(net, zr, checkpoint="int8")
    az, _, ez = hidden(z.double())
    h = az.clamp_min(0)
    _within("y", y.detach(), h @ w2.T + b2, 136 * EPS * (h @ w2.abs().T + b2.abs()) + ez @ w2.abs().T)
    got = torch.autograd.grad(y, [zr, *net.parameters()], up)
    h, ud, on = a.clamp_min(0), up.double(), (a > 0).double()
    da, eda = (ud @ w2) * on, (nout + 8) * EPS * (ud.abs() @ w2.abs()) * on
    n = (rows + 8) * EPS
    want = dict(dz=(da @ w1, 136 * EPS * (da.abs() @ w1.abs()) + eda @ w1.abs()),
                dW1=(da.T @ zd, n * (da.abs().T @ zd.abs()) + eda.T @ zd.abs()),
                db1=(da.sum(0), n * da.abs().sum(0) + eda.sum(0)),
                dW2=(ud.T @ h, n * (ud.abs().T @ h) + ud.abs().T @ el),
                db2=(ud.sum(0), n * ud.abs().sum(0)))
    for grad, (name, (ref, bound)) in zip(got, want.items()):
        if name not in skip:
            _within(name, grad, ref, bound)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("size", [-30, -20, 16, 20, 24, 30])
def test_one_column_of_another_size(shape, size):
    """One column 2^size times larger, its weights as much smaller."""
    for rows in (33, 1500):
        net, z, up = _case(shape, rows)
        z[:, 2] *= 2.0 ** size
        with torch.no_grad():
            net[0].weight[:, 2] *= 2.0 ** -size
        _check(net, z, up)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("size", [-30, -20, 20, 30])
def test_hidden_units_of_another_size(shape, size):
    """Two hidden units 2^size times larger, their outgoing weights as much smaller; one of them in use by half the rows."""
    net, z, up = _case(shape, 1500)
    with torch.no_grad():
        for unit in (5, 77):
            net[0].weight[unit] *= 2.0 ** size
            net[0].bias[unit] *= 2.0 ** size
            net[2].weight[:, unit] *= 2.0 ** -size
    _check(net, z, up)
    with torch.no_grad():
        net[2].weight[:, [5, 77]] *= 2.0 ** size
    _check(net, z, up)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("size", [-40, -20, 20, 40])
def test_outputs_of_another_size(shape, size):
    """One output 2^size times larger, its upstream as much smaller, and the other way round."""
    net, z, up = _case(shape, 1500)
    with torch.no_grad():
        net[2].weight[1] *= 2.0 ** size
        net[2].bias[1] *= 2.0 ** size
    _check(net, z, up)
    up[:, 1] *= 2.0 ** -size
    _check(net, z, up)


@pytest.mark.parametrize("shape", SHAPES)
def test_rows_and_upstreams_of_any_size(shape):
    """Rows and upstreams from 2^-60 to 2^60 side by side; biases of 0, so that small rows count."""
    net, z, up = _case(shape, 1500)
    g = _gen(3)
    with torch.no_grad():
        net[0].bias.zero_()
        net[2].bias.zero_()
    z *= 2.0 ** torch.randint(-60, 61, (1500, 1), device="cuda", generator=g)
    up *= 2.0 ** torch.randint(-60, 61, (1500, 1), device="cuda", generator=g)
    _check(net, z, up)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("size", [-90, 100, 110, 118])
def test_rows_at_the_ends_of_the_range(shape, size):
    net, z, up = _case(shape, 33)
    with torch.no_grad():
        net[0].bias *= 2.0 ** size
        net[2].bias *= 2.0 ** size
    _check(net, z.clamp(-3, 3) * 2.0 ** size, up)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("size", [-40, 40])
def test_weights_of_another_size(shape, size):
    net, z, up = _case(shape, 1500)
    with torch.no_grad():
        net[0].weight *= 2.0 ** size
        net[0].bias *= 2.0 ** size
    _check(net, z, up)
    with torch.no_grad():
        net[2].weight *= 2.0 ** -size
    _check(net, z, up)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("bias", [-1e5, -1e30, LOWEST, float("-inf")])
def test_hidden_units_switched_off(shape, bias):
    """A bias that keeps a unit at zero takes nothing from the others."""
    net, z, up = _case(shape, 1500)
    with torch.no_grad():
        net[0].bias[[0, 31, 100]] = bias
    _check(net, z, up)


@pytest.mark.parametrize("shape", SHAPES)
def test_masked_columns(shape):
    """The type's lowest value in a column that no weight reads."""
    net, z, up = _case(shape, 1500)
    z[::2, 3] = LOWEST
    with torch.no_grad():
        net[0].weight[:, 3] = 0
    _check(net, z, up, skip=("dW1",))  # its column overflows float32


def test_rows_that_are_not_finite():
    """NaN through their own rows, y's and dz's other rows unchanged."""
    from npa_amd import mlp as M
    net, z, up = _case((83, 19), 99)
    y = M.mlp(net, z, checkpoint="int8").detach()
    bad = z.clone()
    bad[40, 82], bad[41, 0], bad[98, 7] = float("nan"), float("inf"), float("-inf")
    got = M.mlp(net, bad, checkpoint="int8").detach()
    keep = torch.ones(99, dtype=torch.bool, device="cuda")
    keep[[40, 41, 98]] = False
    assert torch.equal(got[keep], y[keep]) and torch.isnan(got[~keep]).all()

def test_lowest_value_comes_back_finite():
    """127 * (m / 127) rounds past float32's largest value for that value alone."""
    from npa_amd import int8
    big = -LOWEST
    for cols in (1, 5, 83, 1030, 9000):
        x = torch.zeros(3, cols, device="cuda")
        x[0, cols // 2], x[1, 0], x[2, -1] = big, LOWEST, 3.0e38
        r = int8.quantize_rows(x)
        back = int8.restore_rows(r)
        assert torch.equal(back[:2], x[:2]) and torch.isfinite(back).all()
        assert torch.all((back.double() - x.double()).abs() <= 0.5 * r.scale.double()[:, None] * (1 + 2.0 ** -20))
        x[0, 0] = float("nan")
        back = int8.restore_rows(int8.quantize_rows(x))
        assert torch.isnan(back[0]).all() and torch.isfinite(back[1:]).all()


@pytest.mark.parametrize("large", [1, 200])
def test_relu_rows_stand_for_less_than_a_scale_more(large):
    """What the codes of relu(x) are off by: half a scale, and up to a scale upward
    for positive values below half of one, which are raised to the code 1."""
    from npa_amd import int8
    x = torch.randn(500, 256, device="cuda", generator=_gen(9))
    x[:, 0] = x[:, 0].abs() * large
    r = int8.quantize_rows(x, relu=True)
    true, scale = x.double().clamp_min(0), r.scale.double()[:, None] * (1 + 2.0 ** -20)
    off = int8.restore_rows(r).double() - true
    small = (true > 0) & (true < 0.5 * scale)
    assert torch.all((off.abs() <= 0.5 * scale)[~small]) and torch.all(((off >= 0) & (off < scale))[small])
    assert small.any() and torch.all(off[true == 0] == 0)


def test_bias_gradient_over_a_million_rows():
    """db1 of upstreams of either sign.  n additions of such values in one chain are
    off by about 0.3 n^(1/2) 2^-24 of the sum: 1024 of them by 5.7e-7, 64 by 1.4e-7.
    The limit stands between."""
    from npa_amd import mlp as M
    rows = 1 << 20
    net, z, up = _case((83, 19), rows, seed=11)
    w1, b1, w2 = (p.detach().double() for p in list(net.parameters())[:3])
    zd = _kept(z)
    a = zd @ w1.T + b1
    up[(a.abs() < 1e-5).any(1)] = 0
    ref = ((up.double() @ w2) * (a > 0)).sum(0)
    got = torch.autograd.grad(M.mlp(net, z, checkpoint="int8"), net[0].bias, up)[0]
    assert ((got.double() - ref).norm() <= 3.5e-7 * ref.norm()).item()
