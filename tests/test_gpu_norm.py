"""Layer norm (npa_amd.norm) against its formula in float64.

Bounds, u = 2^-24: the largest chain of float32 additions in a row's sum is 64
values of a lane and the joining of its lanes, 80 roundings in all; G = 128 u
covers it and the roundings of d = x - c, of the mean e of d and of the square
root.  Then |h' - h| <= G (1 + 2 |h|), since r mean |d| <= 1 and e stays small
beside the deviation (rows whose mean is up to 10^4 deviations: e < 0.06 of it).
A gradient's two means add G mean |g| and G mean |g h| (times |h|).  A sum over
rows is a chain of rows / 512 + 128 + 48 additions at most.  Each result is
rounded once more to its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
G = 128 * U
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _half(dtype):
    """Half a step of the type relative to a value, and of its smallest numbers."""
    f = torch.finfo(dtype)
    return f.eps / 2, f.tiny * f.eps / 2 if dtype == F16 else f.tiny


def _within(name, got, ref, bound):
    rel, tiny = _half(got.dtype)
    limit = bound * (1 + rel) + rel * ref.abs() + tiny
    err = (got.double() - ref).abs()
    assert (err <= limit).all(), f"{name}: {(err / limit).nan_to_num(1e30).max().item():.3g} bounds off"


def _reference(x, w, b, eps, dy):
    """(value, bound) of y, dx, dw and db."""
    xd, dyd = x.double(), dy.double()
    wd = torch.ones(x.shape[-1], dtype=torch.float64, device="cuda") if w is None else w.double()
    bd = torch.zeros_like(wd) if b is None else b.double()
    m = xd.mean(-1, keepdim=True)
    r = ((xd - m).square().mean(-1, keepdim=True) + eps).rsqrt()
    h = (xd - m) * r
    eh = G * (1 + 2 * h.abs())
    y = h * wd + bd
    ey = wd.abs() * eh + 3 * U * ((h * wd).abs() + bd.abs())
    g = dyd * wd
    mean = lambda t: t.mean(-1, keepdim=True)
    dx = r * (g - mean(g) - h * mean(g * h))
    ex = 4 * G * r * (g.abs() + mean(g.abs()) + (1 + 2 * h.abs()) * (mean((g * h).abs()) + mean(g.abs())))
    rows = xd.numel() // xd.shape[-1]
    flat = lambda t: t.reshape(rows, -1)
    chain = (rows / 512 + 128 + 48) * U
    dw, db = flat(dyd * h).sum(0), flat(dyd).sum(0)
    ew = chain * flat(dyd * h).abs().sum(0) + flat(dyd.abs() * eh).sum(0)
    return (y, ey), (dx, ex), (dw, ew), (db, chain * flat(dyd).abs().sum(0))


def _check(x, w, b, dy, eps=1e-5):
    from npa_amd import norm
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    lx = leaves[0]
    lw, lb = (leaves[1] if w is not None else None), (leaves[-1] if b is not None else None)
    y = norm.layer_norm(lx, lw, lb, eps)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    with torch.no_grad():
        assert torch.equal(norm.layer_norm(x, w, b, eps), y)
    grads = list(torch.autograd.grad(y, leaves, dy))
    again = torch.autograd.grad(norm.layer_norm(lx, lw, lb, eps), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))  # in a fixed order
    ry, rx, rw, rb = _reference(x, w, b, eps, dy)
    _within("y", y.detach(), *ry)
    _within("dx", grads[0], *rx)
    if w is not None:
        _within("dw", grads[1], *rw)
    if b is not None:
        _within("db", grads[-1], *rb)


def _case(rows, cols, dtype, wide=True, seed=0):
    g = _gen(seed)
    size = torch.exp(torch.randn(cols, device="cuda", generator=g))
    x = (torch.randn(rows, cols, device="cuda", generator=g) * size + torch.randn(rows, 1, device="cuda", generator=g))
    kind = F32 if wide else dtype
    w = (1 + 0.3 * torch.randn(cols, device="cuda", generator=g)).to(kind)
    b = (0.2 * torch.randn(cols, device="cuda", generator=g)).to(kind)
    return x.to(dtype), w, b, torch.randn(rows, cols, device="cuda", generator=g).to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cols", [1, 2, 3, 5, 8, 15, 31, 33, 66, 83, 130, 163, 257, 512, 1000, 1537, 2049, 4097, 6145,
                                  8192, 12289, 16385, 20000, 65536])
def test_columns(cols, dtype):
    for rows, wide in ((1, True), (7, False), (67, True)):
        _check(*_case(rows, cols, dtype, wide, cols))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [2, 64, 65, 513, 4099, 70001])
def test_rows(rows, dtype):
    _check(*_case(rows, 83, dtype, True, rows))
    if rows < 5000:
        _check(*_case(rows, 4097, dtype, True, rows))


def test_weights_may_be_missing():
    x, w, b, dy = _case(70, 83, BF16)
    for ww, bb in ((None, None), (w, None), (None, b), (None, b.to(BF16)), (w.to(BF16), None)):
        _check(x, ww, bb, dy)


def test_no_rows():
    from npa_amd import norm
    x = torch.empty(0, 5, device="cuda", requires_grad=True)
    w = torch.ones(5, device="cuda", requires_grad=True)
    y = norm.layer_norm(x, w, None)
    dx, dw = torch.autograd.grad(y, [x, w], torch.empty(0, 5, device="cuda"))
    assert y.shape == dx.shape == (0, 5) and torch.equal(dw, torch.zeros_like(dw))


@pytest.mark.parametrize("far", [10.0, 1e3, 1e4])
def test_rows_far_from_zero(far):
    """A mean of up to 10^4 deviations, which a float32 mean alone would miss by 3e-4 of one."""
    x, w, b, dy = _case(300, 163, F32)
    x = x / x.std(-1, keepdim=True) + far * torch.randn(300, 1, device="cuda", generator=_gen(1)).sign()
    _check(x, w, b, dy)


def test_rows_of_one_value():
    """No deviation at all: y is the bias; gradients through 1 / sqrt(eps)."""
    from npa_amd import norm
    x, w, b, dy = _case(33, 66, F32)
    x = torch.linspace(-5, 5, 33, device="cuda")[:, None].expand(33, 66).contiguous()
    _check(x, w, b, dy)
    assert torch.isnan(norm.layer_norm(x, w, b, 0.0)).all()  # 0 / 0


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rows_that_are_not_finite(dtype):
    """NaN and infinities stay in their rows; their gradients reach dw and db alone."""
    from npa_amd import norm
    x, w, b, dy = _case(200, 83, dtype)
    bad = x.clone()
    bad[5, 3], bad[77, 82], bad[199, 0] = float("nan"), float("inf"), float("-inf")
    fine = [i for i in range(200) if i not in (5, 77, 199)]
    leaf, ref = bad.requires_grad_(True), x.requires_grad_(True)
    y, want = norm.layer_norm(leaf, w, b), norm.layer_norm(ref, w, b)
    assert torch.isnan(y[[5, 77, 199]]).all() and torch.equal(y[fine], want[fine])
    dx, = torch.autograd.grad(y, leaf, dy)
    assert torch.equal(dx[fine], torch.autograd.grad(want, ref, dy)[0][fine])


def test_shapes_and_strides():
    from npa_amd import norm
    x, w, b, dy = _case(60, 40, F32)
    whole = norm.layer_norm(x, w, b)
    assert torch.equal(norm.layer_norm(x.view(3, 4, 5, 40), w, b), whole.view(3, 4, 5, 40))
    assert torch.equal(norm.layer_norm(x[7], w, b), whole[7])
    assert torch.equal(norm.layer_norm(x.t().contiguous().t(), w, b), whole)
    wide = torch.randn(60, 100, device="cuda", generator=_gen(2))
    for at in (slice(0, 40), slice(3, 43), slice(60, 100)):
        _check(wide[:, at], w, b, wide[:, 20:60])  # rows further apart, at any place
    _check(wide[::2, 1:41], w, b, torch.ones(1, 40, device="cuda").expand(30, 40))
    half = wide.to(BF16)
    _check(half[:, 1:42], *_case(60, 41, BF16)[1:3], half[:, 3:44])
    # weights that are not dense
    assert torch.equal(norm.layer_norm(x, torch.stack([w, w], 1)[:, 0], b), whole)


def test_module():
    from npa_amd import norm
    ours, torchs = norm.LayerNorm(83, device="cuda"), torch.nn.LayerNorm(83, device="cuda")
    x, w, b, dy = _case(50, 83, F32)
    with torch.no_grad():
        torchs.weight.copy_(w)
        torchs.bias.copy_(b)
    ours.load_state_dict(torchs.state_dict())
    assert torch.equal(ours(x), norm.layer_norm(x, w, b))
    plain = norm.LayerNorm(83, elementwise_affine=False, device="cuda")
    assert torch.equal(plain(x), norm.layer_norm(x))
    with pytest.raises(RuntimeError):
        ours(x[:, :82])
    with pytest.raises(ValueError):
        norm.LayerNorm((4, 83))


def test_gradients_against_differences():
    from npa_amd import norm
    x, w, b, dy = _case(6, 19, F32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(norm.layer_norm(*leaves), leaves, dy)

    def loss(*t):
        m = t[0].mean(-1, keepdim=True)
        return ((((t[0] - m) / ((t[0] - m).square().mean(-1, keepdim=True) + 1e-5).sqrt() * t[1] + t[2])) * dy.double()).sum()

    wide = [t.detach().double() for t in leaves]
    for i, g in enumerate(grads):
        way = torch.randn(wide[i].shape, device="cuda", generator=_gen(i), dtype=torch.float64)
        step = 1e-6
        moved = [[t + s * step * way if j == i else t for j, t in enumerate(wide)] for s in (1, -1)]
        slope = ((loss(*moved[0]) - loss(*moved[1])) / (2 * step)).item()
        # float32's roundings over 114 terms, and the difference's own 1e-6^2 and 1e-16 / 1e-6
        assert abs((g.double() * way).sum().item() - slope) <= 1e-5 * (g.double() * way).abs().sum().item() + 1e-6


def test_second_derivatives_raise():
    from npa_amd import norm
    x, w, b, dy = _case(6, 19, F32)
    x.requires_grad_(True)
    dx, = torch.autograd.grad(norm.layer_norm(x, w, b).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        dx.sum().backward()


def test_offsets_past_32_bits():
    from npa_amd import norm
    rows, cols = (1 << 20) + 3, 2051
    x = torch.randn(rows, cols, device="cuda", generator=_gen(0), dtype=BF16)
    assert x.numel() > 1 << 31
    w, b = _case(1, cols, BF16)[1:3]
    x.requires_grad_(True)
    y = norm.layer_norm(x, w, b)
    dx, = torch.autograd.grad(y, x, x.detach())
    for at in (slice(0, 70), slice(-70, None)):
        ry, rx, _, _ = _reference(x.detach()[at], w, b, 1e-5, x.detach()[at])
        _within("y", y.detach()[at], *ry)
        _within("dx", dx[at], *rx)


def test_streams_and_graphs():
    from npa_amd import norm
    x, w, b, dy = _case(3000, 83, F32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    run = lambda: (lambda y: [y.detach(), *torch.autograd.grad(y, leaves, dy)])(norm.layer_norm(*leaves))
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i in range(3):
        with torch.no_grad():
            x.add_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, run()))


def test_refusals():
    from npa_amd import norm
    x, w, b, _ = _case(6, 19, BF16)
    for call in (lambda: norm.layer_norm(x.double(), w, b), lambda: norm.layer_norm(x.cpu(), w, b),
                 lambda: norm.layer_norm(x, w.double(), b), lambda: norm.layer_norm(x, w.to(F16)),
                 lambda: norm.layer_norm(x, w, b.to(BF16)), lambda: norm.layer_norm(x.float(), w.to(BF16)),
                 lambda: norm.layer_norm(x, w.cpu())):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: norm.layer_norm(x, w[:18]), lambda: norm.layer_norm(x, w[None]),
                 lambda: norm.layer_norm(x, None, b[:1]), lambda: norm.layer_norm(x[:, :0]),
                 lambda: norm.layer_norm(torch.zeros((), device="cuda")),
                 lambda: norm.layer_norm(torch.zeros(1, 65537, device="cuda"))):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        norm.layer_norm(x, w, b, -1.0)
    with pytest.raises(ValueError):
        norm.layer_norm(x, w, b, float("nan"))
