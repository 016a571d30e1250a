"""Mixtures of experts (npa_amd.experts): the sort against a stable sort on the
host, rows out and back, and the experts' layers against float64.

Bounds, u = 2^-24: a float32 sum of n products is within (n + 8) 2 u of the sum
of their absolute values (the matrix cores round a sum down, so by up to a whole
step; 8: the pieces of float32 factors and the joining of partial sums); a sum
over a row's entries within (k + 1) u.  Each result is rounded once more to its
type."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
NAN = float("nan")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _within(name, got, ref, bound):
    f = torch.finfo(got.dtype)
    rel, tiny = f.eps / 2, f.tiny * f.eps / 2 if got.dtype == F16 else f.tiny
    limit = bound * (1 + rel) + rel * ref.abs() + tiny
    err = (got.double() - ref).abs()
    ok = err <= limit
    assert ok.all(), (f"{name}: {int((~ok).sum())} elements, {(err / limit).nan_to_num(1e30).max().item():.3g} bounds "
                      f"off, first at {tuple((~ok).nonzero()[0].tolist())}")


def _index(rows, choices, experts, seed=0, none=0.1):
    g = _gen(seed)
    index = torch.randint(0, experts, (rows, choices), device="cuda", generator=g)
    return torch.where(torch.rand(rows, choices, device="cuda", generator=g) < none, torch.full_like(index, -1), index)


def _offsets(counts, behind=0):
    at = torch.tensor([0, *np.cumsum(counts)], dtype=torch.int32, device="cuda")
    return at, int(sum(counts)) + behind


# ------------------------------------------------------------------ the sort

def _check_sort(index, experts):
    from npa_amd import experts as E
    r = E.sort_rows(index, experts)
    key = index.cpu().numpy().reshape(-1).astype(np.int64)
    key = np.where((key < 0) | (key >= experts), experts, key)
    source = np.argsort(key, kind="stable")
    offsets = np.searchsorted(key[source], np.arange(experts + 1))
    slot = np.empty(len(key), np.int64)
    slot[source] = np.arange(len(key))
    slot = np.where(key == experts, ~slot, slot)
    assert all(t.dtype == torch.int32 and t.is_cuda for t in r) and r.slot.shape == index.shape
    assert np.array_equal(r.offsets.cpu().numpy(), offsets)
    assert np.array_equal(r.slot.cpu().numpy().reshape(-1), slot)
    assert np.array_equal(r.source.cpu().numpy(), source)
    return r


@pytest.mark.parametrize("experts", [1, 2, 3, 4, 7, 8, 63, 64, 65, 255, 511, 512, 513, 1023, 1024])
@pytest.mark.parametrize("rows,choices", [(1, 1), (1, 8), (63, 1), (64, 1), (65, 2), (511, 1), (513, 1), (1000, 3),
                                          (4096, 1), (4097, 1), (2731, 6), (16384, 1), (16385, 1), (8193, 7)])
def test_sort(rows, choices, experts):
    _check_sort(_index(rows, choices, experts, experts + rows), experts)


@pytest.mark.parametrize("n", [5, 700, 9000, 40000])
def test_sort_of_one_sided_choices(n):
    for experts in (1, 5, 300):
        _check_sort(torch.full((n, 1), experts - 1, device="cuda"), experts)
        _check_sort(torch.full((n, 1), -1, device="cuda"), experts)
        _check_sort(torch.arange(n, device="cuda")[:, None].flip(0).int(), experts)  # most of them past the experts
        _check_sort((torch.arange(n, device="cuda") % experts)[:, None], experts)


def test_sort_of_any_number():
    """Numbers outside the experts, of both widths, are no expert."""
    big = torch.tensor([[0, -1, 4, 2 ** 31 - 1, -2 ** 31, 3, 1, 0]], device="cuda")
    _check_sort(big.int(), 4)
    _check_sort(torch.cat([big, big + 2 ** 32, big - 2 ** 40, torch.full_like(big, 2 ** 63 - 1)]), 4)


def test_sort_of_nothing():
    r = _check_sort(torch.empty(0, 2, dtype=torch.int64, device="cuda"), 5)
    assert r.source.shape == (0,)


def test_sort_of_many():
    _check_sort(_index(1 << 20, 2, 200, 3), 200)
    _check_sort(_index(300001, 3, 1024, 4).int(), 1024)


def test_sort_shapes_and_strides():
    from npa_amd import experts as E
    index = _index(120, 2, 6)
    want = E.sort_rows(index, 6)
    for same in (index.view(4, 5, 6, 2), index.t().contiguous().t(), torch.stack([index, index], 2)[..., 0]):
        got = E.sort_rows(same, 6)
        assert all(torch.equal(p.reshape(-1), q.reshape(-1)) for p, q in zip(got, want))


# ------------------------------------------------------- rows out and back

def _reference_rows(x, slot):
    """The places' rows in float64."""
    rows, choices = slot.shape
    out = torch.zeros(rows * choices, x.shape[1], dtype=torch.float64, device="cuda")
    for j in range(choices):
        has = slot[:, j] >= 0
        out[slot[has, j].long()] = x.double()[has]
    return out


def _check_rows(rows, choices, experts, cols, dtype, none=0.1):
    from npa_amd import experts as E
    g = _gen(rows + cols)
    r = E.sort_rows(_index(rows, choices, experts, rows, none), experts)
    n, live, slot = rows * choices, int(r.offsets[-1]), r.slot
    has = slot >= 0
    x = _randn(g, rows, cols).to(dtype).requires_grad_(True)
    results = _randn(g, n, cols).to(dtype)
    results[live:] = NAN  # nothing reads behind the last
    weight = _randn(g, rows, choices)
    weight[~has] = NAN    # nor the weights of entries without an expert
    results.requires_grad_(True)
    weight.requires_grad_(True)
    spread = E.dispatch(x, r)
    assert spread.dtype == dtype and torch.equal(spread.double(), _reference_rows(x.detach(), slot))
    y = E.combine(results, weight, r)
    at = slot.clamp_min(0).long()
    parts = torch.where(has[..., None], weight.detach().double()[..., None] * results.detach().double()[at], 0.0)
    _within("y", y.detach(), parts.sum(1), (choices + 1) * U * parts.abs().sum(1))
    plain = E.combine(results, None, r)
    parts = torch.where(has[..., None], results.detach().double()[at], 0.0)
    _within("y without weights", plain.detach(), parts.sum(1), (choices + 1) * U * parts.abs().sum(1))
    # gradients
    up = _randn(g, n, cols).to(dtype)
    up[live:] = NAN
    dx, = torch.autograd.grad(spread, x, up)
    parts = torch.where(has[..., None], up.double()[at], 0.0)
    _within("dx", dx, parts.sum(1), (choices + 1) * U * parts.abs().sum(1))
    dy = _randn(g, rows, cols).to(dtype)
    none_at_all = ~has.any(1)
    dy[none_at_all] = NAN  # nothing came from these rows
    d_results, dw = torch.autograd.grad(y, [results, weight], dy)
    want = torch.zeros(n, cols, dtype=torch.float64, device="cuda")
    for j in range(choices):
        want[at[has[:, j], j]] = (weight.detach().double()[:, j, None] * dy.double())[has[:, j]]
    _within("d_results", d_results, want, U * want.abs())
    terms = torch.where(has[..., None], results.detach().double()[at] * dy.double()[:, None], 0.0)
    _within("dw", dw, terms.sum(2), (cols + 8) * U * terms.abs().sum(2))
    assert not dw[~has].any()
    for t, s in ((E.combine(results.detach(), weight, r), weight), (E.combine(results, weight.detach(), r), results)):
        one, = torch.autograd.grad(t, s, dy)
        assert torch.equal(one, dw if s is weight else d_results)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cols", [1, 3, 8, 17, 33, 66, 83, 163, 200, 257, 511, 1000, 1025, 2049, 4097, 9000, 20000])
def test_rows_out_and_back(cols, dtype):
    for rows, choices, experts in ((1, 1, 4), (37, 2, 5), (130, 3, 2)):
        _check_rows(rows, choices, experts, cols, dtype)


@pytest.mark.parametrize("rows,choices,experts", [(9, 64, 7), (5000, 1, 4), (3000, 8, 64), (70000, 1, 3)])
def test_more_rows(rows, choices, experts):
    _check_rows(rows, choices, experts, 20, F32)
    _check_rows(rows, choices, experts, 19, BF16)


def test_rows_without_experts():
    _check_rows(50, 2, 3, 40, F32, none=1.0)
    _check_rows(50, 2, 3, 40, BF16, none=0.9)


def test_the_same_expert_twice():
    from npa_amd import experts as E
    index = torch.tensor([[1, 1], [0, 1], [1, 0]], device="cuda")
    r = E.sort_rows(index, 2)
    x = torch.randn(3, 8, device="cuda", requires_grad=True)
    y = E.combine(E.dispatch(x, r), torch.tensor([[0.25, 0.5], [1.0, 2.0], [4.0, 8.0]], device="cuda"), r)
    scale = torch.tensor([0.75, 3.0, 12.0], device="cuda")[:, None]
    assert torch.allclose(y, x * scale, rtol=1e-6) and torch.allclose(
        torch.autograd.grad(y.sum(), x)[0], scale.expand(3, 8), rtol=1e-6)


def test_rows_of_any_shape_and_stride():
    from npa_amd import experts as E
    index = _index(60, 2, 5)
    r = E.sort_rows(index, 5)
    wide = _randn(_gen(1), 60, 100)
    want = E.dispatch(wide[:, 3:43].contiguous(), r)
    assert torch.equal(E.dispatch(wide[:, 3:43], r), want)
    assert torch.equal(E.dispatch(wide.t().contiguous().t()[:, 3:43], r), want)
    cube = E.sort_rows(index.view(3, 20, 2), 5)
    assert torch.equal(E.dispatch(wide[:, 3:43].reshape(3, 20, 40), cube), want)
    out = _randn(_gen(2), 120, 90)
    weight = _randn(_gen(3), 60, 2)
    y = E.combine(out[:, 7:50].contiguous(), weight, r)
    assert torch.equal(E.combine(out[:, 7:50], weight, r), y)
    assert torch.equal(E.combine(out[:, 7:50], weight.t().contiguous().t(), r), y)
    assert torch.equal(E.combine(out[:, 7:50], weight.view(3, 20, 2), cube), y.view(3, 20, 43))
    # upstreams that are not dense
    x = wide[:, :40].clone().requires_grad_(True)
    up = _randn(_gen(4), 40, 120)
    a, = torch.autograd.grad(E.dispatch(x, r), x, up.t())
    b, = torch.autograd.grad(E.dispatch(x, r), x, up.t().contiguous())
    assert torch.equal(a, b)
    res = out[:, :40].clone().requires_grad_(True)
    a, = torch.autograd.grad(E.combine(res, weight, r).sum(), res)
    assert torch.equal(a, torch.autograd.grad(E.combine(res, weight, r), res, torch.ones(60, 40, device="cuda"))[0])


def test_places_outside_are_left_out():
    """A slot that names no place of the call is neither read nor written."""
    from npa_amd import experts as E
    r = E.sort_rows(_index(20, 2, 3, none=0.0), 3)
    slot = r.slot.clone()
    slot[4, 1], slot[9, 0], slot[11, 1] = 40, 2 ** 31 - 1, -2 ** 31
    bad = E.Routing(r.offsets, slot, r.source)
    x = torch.ones(20, 5, device="cuda")
    E.dispatch(x, bad)
    y = E.combine(torch.ones(40, 5, device="cuda"), None, bad)
    assert torch.equal(y[:, 0], torch.tensor([1.0 if i in (4, 9, 11) else 2.0 for i in range(20)], device="cuda"))


# ------------------------------------------------------- the experts' layers

def _check_linear(counts, behind, cols, outs, dtype, bias=True, seed=0, x=None, dy=None):
    from npa_amd import experts as E
    g = _gen(seed + cols + outs)
    offsets, slots = _offsets(counts, behind)
    n = len(counts)
    if x is None:
        x = _randn(g, slots, cols).to(dtype)
    if dy is None:
        dy = _randn(g, slots, outs).to(dtype)
    w = (_randn(g, n, outs, cols) / cols ** 0.5).to(dtype)
    b = _randn(g, n, outs).to(dtype) if bias else None
    live = sum(counts)
    x, dy = x.clone(), dy.clone()
    x[live:], dy[live:] = NAN, NAN  # rows behind the last expert's count for nothing
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    y = E.linear(x, w, b, offsets)
    grads = torch.autograd.grad(y, leaves, dy)
    again = torch.autograd.grad(E.linear(x, w, b, offsets), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))  # in a fixed order
    with torch.no_grad():
        assert torch.equal(E.linear(x, w, b, offsets), y)
    assert y.dtype == dtype and not y[live:].any() and not grads[0][live:].any()
    xd, wd, dyd = x.detach().double(), w.detach().double(), dy.double()
    bd = b.detach().double() if bias else torch.zeros(n, outs, dtype=torch.float64, device="cuda")
    at = 0
    for e, c in enumerate(counts):
        s = slice(at, at + c)
        at += c
        k = lambda m: (m + 8) * 2 * U
        _within(f"y of {e}", y.detach()[s], xd[s] @ wd[e].T + bd[e], k(cols) * (xd[s].abs() @ wd[e].abs().T + bd[e].abs()))
        _within(f"dx of {e}", grads[0][s], dyd[s] @ wd[e], k(outs) * (dyd[s].abs() @ wd[e].abs()))
        _within(f"dW of {e}", grads[1][e], dyd[s].T @ xd[s], k(c) * (dyd[s].abs().T @ xd[s].abs()))
        if bias:
            _within(f"db of {e}", grads[2][e], dyd[s].sum(0), k(c) * dyd[s].abs().sum(0))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cols,outs", [(1, 1), (3, 5), (4, 4), (8, 16), (16, 8), (31, 33), (32, 32), (64, 64), (66, 128),
                                       (83, 128), (128, 19), (128, 128), (127, 129), (136, 72), (163, 35), (256, 264),
                                       (520, 100), (2049, 40), (40, 2050)])
def test_linear_sizes(cols, outs, dtype):
    _check_linear([37, 0, 130, 1], 5, cols, outs, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("counts,behind", [([1], 0), ([0], 0), ([0], 9), ([0, 0, 3], 0), ([16], 0), ([17], 3), ([128], 0),
                                           ([127, 129], 0), ([300], 200), ([1] * 40, 0), ([0, 1] * 70, 7), ([2, 700, 3], 1),
                                           ([5] * 200, 0), ([0] * 1023 + [9], 4), ([1] * 1024, 0)])
def test_linear_groups(counts, behind, dtype):
    _check_linear(counts, behind, 64, 48, dtype)
    _check_linear(counts, behind, 35, 20, dtype, bias=False)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_linear_of_wide_layers(dtype):
    _check_linear([200, 0, 333, 64], 10, 1024, 768, dtype)
    _check_linear([64, 65, 1], 0, 4096, 512, dtype)
    _check_linear([500, 600], 100, 256, 1536, dtype, bias=False)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_linear_of_large_tiles(dtype):
    """Enough tiles of 256 over the rows, and over the weights."""
    _check_linear([20000, 0, 29000, 257, 1], 300, 72, 264, dtype)
    _check_linear([20001, 255, 256, 30000], 0, 264, 392, dtype, bias=False)
    _check_linear([300, 0, 64, 65, 1, 63, 500, 31, 32, 33, 7, 128], 3, 1032, 1000, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_linear_of_cut_tiles(dtype):
    """Long sums over few tiles, which are cut along the sum: laid out first, as they are, short tiles, few outputs."""
    _check_linear([2000, 2200, 1, 0], 100, 1030, 1060, dtype)
    _check_linear([5500, 0, 4900], 100, 1999, 1801, dtype)
    _check_linear([1100, 3], 100, 2001, 2009, dtype, bias=False)
    _check_linear([600, 90, 1], 40, 2048, 1536, dtype, bias=False)
    _check_linear([300, 0, 77], 9, 1545, 125, dtype)
    _check_linear([300, 0, 77], 9, 1000, 33, dtype)
    _check_linear([30, 9, 18, 0], 200, 700, 520, dtype)
    _check_linear([530, 3], 0, 20, 1030, dtype)


@pytest.mark.parametrize("counts", [[4095, 9], [17000, 9]])
def test_linear_of_tall_weight_tiles(counts):
    """float32 weight gradients of many tiles, long sums: whole, and in chunks."""
    _check_linear(counts, 5, 4000, 4080, F32)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_of_many_rows(dtype):
    _check_linear([20000, 3, 0, 9000, 40001], 77, 83, 35, dtype)
    _check_linear([70000, 5000], 0, 24, 16, dtype)


def test_linear_without_rows():
    from npa_amd import experts as E
    offsets = torch.zeros(4, dtype=torch.int32, device="cuda")
    x = torch.empty(0, 6, device="cuda", requires_grad=True)
    w = torch.randn(3, 5, 6, device="cuda", requires_grad=True)
    b = torch.randn(3, 5, device="cuda", requires_grad=True)
    y = E.linear(x, w, b, offsets)
    grads = torch.autograd.grad(y, [x, w, b], torch.empty(0, 5, device="cuda"))
    assert y.shape == (0, 5) and grads[0].shape == (0, 6) and not grads[1].any() and not grads[2].any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_linear_strides(dtype):
    """Rows further apart and at any place, upstreams that repeat."""
    g = _gen(5)
    wide = _randn(g, 150, 300).to(dtype)
    for at, cols in ((0, 64), (1, 64), (3, 83), (8, 200)):
        from npa_amd import experts as E
        offsets, slots = _offsets([70, 80])
        w = _randn(g, 2, 40, cols).to(dtype).requires_grad_(True)
        dy = _randn(g, 150, 90).to(dtype)[:, 11:51]
        x = wide[:, at:at + cols].detach().requires_grad_(True)
        assert not x.is_contiguous()
        dense = x.detach().contiguous().requires_grad_(True)
        y, want = E.linear(x, w, None, offsets), E.linear(dense, w, None, offsets)
        assert torch.equal(y, want)
        for up in (dy, dy[:1].expand(150, 40), dy[:, :1].expand(150, 40)):
            a = torch.autograd.grad(y, [x, w], up, retain_graph=True)
            b = torch.autograd.grad(want, [dense, w], up.contiguous(), retain_graph=True)
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_linear_float32_keeps_its_bits():
    """Sizes of any kind side by side: each element within its own bound."""
    g = _gen(9)
    x = _randn(g, 300, 83) * 2.0 ** torch.randint(-40, 41, (300, 1), device="cuda", generator=g)
    x[:, 7] *= 2.0 ** 24
    dy = _randn(g, 300, 40) * 2.0 ** torch.randint(-30, 31, (300, 1), device="cuda", generator=g)
    _check_linear([100, 200], 0, 83, 40, F32, x=x, dy=dy)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_linear_rows_that_are_not_finite(dtype):
    """NaN and infinities stay in their rows and their expert's gradients."""
    from npa_amd import experts as E
    g = _gen(6)
    offsets, slots = _offsets([40, 50, 60], 6)
    x, w = _randn(g, slots, 70).to(dtype), _randn(g, 3, 36, 70).to(dtype)
    dy = _randn(g, slots, 36).to(dtype)
    bad = x.clone()
    bad[39, 69], bad[90, 0] = NAN, float("inf")  # the last row of one expert, the first of another
    fine = [i for i in range(slots) if i not in (39, 90)]
    out = []
    for t in (x, bad):
        leaves = [t.requires_grad_(True), w.clone().requires_grad_(True)]
        y = E.linear(leaves[0], leaves[1], None, offsets)
        out.append((y.detach(), *torch.autograd.grad(y, leaves, dy)))
    (y, dx, dw), (yb, dxb, dwb) = out
    assert torch.equal(y[fine], yb[fine]) and not torch.isfinite(yb[[39, 90]]).any()
    assert torch.equal(dx, dxb) and torch.equal(dw[1], dwb[1])
    assert not torch.isfinite(dwb[0][:, 69]).any() and not torch.isfinite(dwb[2][:, 0]).any()


def test_offsets_of_any_kind_stay_inside():
    """Offsets that no sort gives: some values, no access outside."""
    from npa_amd import experts as E
    x, w = torch.ones(50, 20, device="cuda"), torch.ones(3, 16, 20, device="cuda")
    for at in ([0, 10, 100, 50], [5, 4, 3, 2], [-7, 2 ** 31 - 1, -2 ** 31, 0], [60, 70, 80, 90]):
        offsets = torch.tensor(at, dtype=torch.int32, device="cuda")
        lx, lw = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = E.linear(lx, lw, None, offsets)
        torch.autograd.grad(y, [lx, lw], torch.ones_like(y))
        assert y.shape == (50, 16)


# --------------------------------------------------------------- the MLP

@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cols,hidden,outs", [(66, 128, 18), (83, 128, 19), (5, 7, 3), (64, 256, 64), (130, 96, 200)])
def test_mlp_is_its_layers(cols, hidden, outs, dtype):
    """Bit for bit the composition: a ReLU commutes with rounding."""
    from npa_amd import experts as E
    if dtype == F32 and hidden == 128:
        hidden = 132  # 128 hidden units in float32 have kernels of their own
    g = _gen(cols)
    offsets, slots = _offsets([70, 0, 200, 3], 9)
    x = _randn(g, slots, cols).to(dtype)
    x[-9:] = NAN
    w1, b1 = (_randn(g, 4, hidden, cols) / cols ** 0.5).to(dtype), _randn(g, 4, hidden).to(dtype)
    w2, b2 = (_randn(g, 4, outs, hidden) / hidden ** 0.5).to(dtype), _randn(g, 4, outs).to(dtype)
    dy = _randn(g, slots, outs).to(dtype)
    for biases in ((b1, b2), (None, None)):
        leaves = [t.detach().requires_grad_(True) for t in (x, w1, biases[0], w2, biases[1]) if t is not None]
        full = (lambda p: p if biases[0] is not None else (p[0], p[1], None, p[2], None))(leaves)
        y = E.mlp(*full, offsets)
        want = E.linear(torch.relu(E.linear(full[0], full[1], full[2], offsets)), full[3], full[4], offsets)
        assert torch.equal(y, want)
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves, dy),
                                                     torch.autograd.grad(want, leaves, dy)))
        with torch.no_grad():
            assert torch.equal(E.mlp(*full, offsets), want)
        for i in range(len(leaves)):  # any one of the gradients alone
            only = [t.detach().requires_grad_(i == j) for j, t in enumerate(leaves)]
            args = (lambda p: p if biases[0] is not None else (p[0], p[1], None, p[2], None))(only)
            one, = torch.autograd.grad(E.mlp(*args, offsets), only[i], dy)
            assert torch.equal(one, torch.autograd.grad(E.mlp(*full, offsets), leaves[i], dy)[0])


def _check_fused(counts, behind, cols, outs, biases=True, scale=None, seed=0):
    """The MLP of 128 hidden units in float32 against float64.  Hidden values are within (cols + 8) 2 u of their sums of
    absolute values; rows with one that near to 0 get no upstream, since either side's gradient is right there."""
    from npa_amd import experts as E
    g = _gen(seed + cols + outs)
    offsets, slots = _offsets(counts, behind)
    n, live = len(counts), sum(counts)
    x, dy = _randn(g, slots, cols), _randn(g, slots, outs)
    w1, w2 = _randn(g, n, 128, cols) / cols ** 0.5, _randn(g, n, outs, 128) / 11.3
    b1, b2 = (_randn(g, n, 128), _randn(g, n, outs)) if biases else (None, None)
    if scale is not None:
        scale(x, dy, w1, w2, g)
    k = lambda m: (m + 8) * 2 * U
    at, parts = 0, []
    for e, c in enumerate(counts):
        s = slice(at, at + c)
        at += c
        wd, xd = w1[e].double(), x[s].double()
        bd = b1[e].double() if biases else torch.zeros(128, dtype=torch.float64, device="cuda")
        a, ea = xd @ wd.T + bd, k(cols) * (xd.abs() @ wd.abs().T + bd.abs())
        dy[s][(a.abs() <= 2 * ea).any(1)] = 0
        parts.append((s, a, ea))
    assert (dy[:live] != 0).any(1).sum() * 2 >= live
    x[live:], dy[live:] = NAN, NAN
    args = [x, w1, b1, w2, b2]
    leaves = [t.requires_grad_(True) for t in args if t is not None]
    y = E.mlp(*args, offsets)
    grads = torch.autograd.grad(y, leaves, dy)
    again = torch.autograd.grad(E.mlp(*args, offsets), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))  # in a fixed order
    with torch.no_grad():
        assert torch.equal(E.mlp(*args, offsets), y)
    for i, t in enumerate(leaves):  # any one of the gradients alone
        only = [p.detach().requires_grad_(p is t) if p is not None else None for p in args]
        wanted = next(p for p in only if p is not None and p.requires_grad)
        assert torch.equal(torch.autograd.grad(E.mlp(*only, offsets), wanted, dy)[0], grads[i])
    grads = list(grads)
    dx, dw1 = grads[0], grads[1]
    db1, dw2, db2 = (grads[2], grads[3], grads[4]) if biases else (None, grads[2], None)
    assert not y[live:].any() and not dx[live:].any()
    for e, (s, a, ea) in enumerate(parts):
        c, h = a.shape[0], a.clamp_min(0)
        eh = torch.where(a > -ea, ea, torch.zeros_like(ea))
        w1d, w2d, xd, dyd = w1[e].detach().double(), w2[e].detach().double(), x[s].detach().double(), dy[s].double()
        b2d = b2[e].detach().double() if biases else torch.zeros(outs, dtype=torch.float64, device="cuda")
        _within(f"y of {e}", y.detach()[s], h @ w2d.T + b2d, k(128) * (h @ w2d.abs().T + b2d.abs()) + eh @ w2d.abs().T)
        on = (a > 0).double()
        da, eda = (dyd @ w2d) * on, k(outs) * (dyd.abs() @ w2d.abs()) * on
        _within(f"dx of {e}", dx[s], da @ w1d, k(128) * (da.abs() @ w1d.abs()) + eda @ w1d.abs())
        _within(f"dW1 of {e}", dw1[e], da.T @ xd, k(c) * (da.abs().T @ xd.abs()) + eda.T @ xd.abs())
        _within(f"dW2 of {e}", dw2[e], dyd.T @ h, k(c) * (dyd.abs().T @ h) + dyd.abs().T @ eh)
        if biases:
            _within(f"db1 of {e}", db1[e], da.sum(0), k(c) * da.abs().sum(0) + eda.sum(0))
            _within(f"db2 of {e}", db2[e], dyd.sum(0), k(c) * dyd.abs().sum(0))


@pytest.mark.parametrize("cols,outs", [(4, 4), (5, 64), (32, 32), (33, 17), (64, 20), (66, 18), (83, 19), (83, 35), (96, 48),
                                       (97, 33), (128, 30), (130, 50), (160, 8), (163, 35), (168, 64)])
def test_fused_mlp_sizes(cols, outs):
    _check_fused([37, 0, 130, 1, 300], 5, cols, outs)
    _check_fused([33], 0, cols, outs, biases=False)


@pytest.mark.parametrize("counts,behind", [([1], 0), ([0], 0), ([0], 9), ([0, 0, 3], 0), ([32], 0), ([31, 33], 0),
                                           ([300], 200), ([1] * 40, 0), ([0, 1] * 70, 7), ([5] * 300, 0),
                                           ([0] * 1023 + [9], 4), ([1] * 1024, 0), ([9000, 1, 8000, 0, 3000], 2000),
                                           ([17000] * 2, 1), ([100, 40000, 100], 0), ([64] * 200, 0)])
def test_fused_mlp_groups(counts, behind):
    _check_fused(counts, behind, 66, 18)
    if sum(counts) < 30000:
        _check_fused(counts, behind, 163, 35)


def test_fused_mlp_of_many_rows():
    _check_fused([300001, 5, 90000, 0, 12345], 321, 83, 19)


def test_fused_mlp_without_rows():
    from npa_amd import experts as E
    offsets = torch.zeros(4, dtype=torch.int32, device="cuda")
    args = [torch.empty(0, 6, device="cuda"), torch.randn(3, 128, 6, device="cuda"), torch.randn(3, 128, device="cuda"),
            torch.randn(3, 5, 128, device="cuda"), torch.randn(3, 5, device="cuda")]
    leaves = [t.requires_grad_(True) for t in args]
    y = E.mlp(*leaves, offsets)
    grads = torch.autograd.grad(y, leaves, torch.empty(0, 5, device="cuda"))
    assert y.shape == (0, 5) and not any(g.any() for g in grads[1:])


@pytest.mark.parametrize("size", [-30, -20, 20, 30])
def test_fused_mlp_of_other_sizes(size):
    """A column, a hidden unit, an output and rows of other sizes than the rest: each element within its own bound."""
    def column(x, dy, w1, w2, g):
        x[:, 2] *= 2.0 ** size
        w1[:, :, 2] *= 2.0 ** -size

    def unit(x, dy, w1, w2, g):
        w1[:, 5] *= 2.0 ** size
        w2[:, :, 5] *= 2.0 ** -size

    def output(x, dy, w1, w2, g):
        w2[:, 1] *= 2.0 ** size
        dy[:, 1] *= 2.0 ** -size

    def rows(x, dy, w1, w2, g):
        dy *= 2.0 ** torch.randint(-abs(size), abs(size) + 1, (len(dy), 1), device="cuda", generator=g)

    for scale in (column, unit, output, rows):
        _check_fused([200, 333], 0, 83, 19, scale=scale)


def test_fused_mlp_rows_that_are_not_finite():
    """NaN and infinities stay in their rows and their expert's gradients."""
    from npa_amd import experts as E
    g = _gen(6)
    offsets, slots = _offsets([40, 50, 60], 6)
    x, dy = _randn(g, slots, 66), _randn(g, slots, 18)
    w = [_randn(g, 3, 128, 66), _randn(g, 3, 128), _randn(g, 3, 18, 128), _randn(g, 3, 18)]
    bad = x.clone()
    bad[39, 65], bad[90, 0] = NAN, float("inf")
    fine = [i for i in range(slots) if i not in (39, 90)]
    out = []
    for t in (x, bad):
        leaves = [t.requires_grad_(True)] + [p.clone().requires_grad_(True) for p in w]
        y = E.mlp(*leaves, offsets)
        out.append((y.detach(), *torch.autograd.grad(y, leaves, dy)))
    (y, dx, *_), (yb, dxb, *gb) = out
    assert torch.equal(y[fine], yb[fine]) and torch.isnan(yb[39]).all() and not torch.isfinite(yb[90]).all()
    assert torch.equal(dx[fine], dxb[fine])
    for p, q in zip(out[0][2:], gb):
        assert torch.equal(p[1], q[1])


def test_fused_mlp_strides():
    from npa_amd import experts as E
    g = _gen(8)
    wide, up = _randn(g, 90, 200), _randn(g, 90, 60)
    offsets, _ = _offsets([40, 50])
    w = [_randn(g, 2, 128, 66), _randn(g, 2, 128), _randn(g, 2, 18, 128), _randn(g, 2, 18)]
    x = wide[:, 3:69].detach().requires_grad_(True)
    dense = x.detach().contiguous().requires_grad_(True)
    a = E.mlp(x, *[p.transpose(0, 1).contiguous().transpose(0, 1) for p in w], offsets)
    b = E.mlp(dense, *w, offsets)
    assert torch.equal(a, b)
    for dy in (up[:, 7:25], up[:1, :18].expand(90, 18)):
        assert torch.equal(torch.autograd.grad(a, x, dy, retain_graph=True)[0],
                           torch.autograd.grad(b, dense, dy.contiguous(), retain_graph=True)[0])


def test_fused_mlp_offsets_of_any_kind_stay_inside():
    from npa_amd import experts as E
    x, w = torch.ones(500, 20, device="cuda"), [torch.ones(3, 128, 20, device="cuda"), None,
                                                torch.ones(3, 16, 128, device="cuda"), None]
    for at in ([0, 10, 100, 50], [5, 4, 3, 2], [-7, 2 ** 31 - 1, -2 ** 31, 0], [600, 700, 800, 900], [0, 500, 0, 500]):
        offsets = torch.tensor(at, dtype=torch.int32, device="cuda")
        leaves = [x.clone().requires_grad_(True), w[0].clone().requires_grad_(True), None,
                  w[2].clone().requires_grad_(True), None]
        y = E.mlp(*leaves, offsets)
        torch.autograd.grad(y, [t for t in leaves if t is not None], torch.ones_like(y))
        assert y.shape == (500, 16)


def test_gradients_against_differences():
    """The mixture from rows to loss: each gradient along a random way."""
    from npa_amd import experts as E
    g = _gen(3)
    index = _index(40, 2, 3)
    r = E.sort_rows(index, 3)
    x, weight = _randn(g, 40, 10), torch.rand(40, 2, device="cuda", generator=g)
    w1, b1, w2, b2 = _randn(g, 3, 16, 10) / 3, _randn(g, 3, 16), _randn(g, 3, 6, 16) / 4, _randn(g, 3, 6)
    up = _randn(g, 40, 6)
    leaves = [t.requires_grad_(True) for t in (x, weight, w1, b1, w2, b2)]
    y = E.combine(E.mlp(E.dispatch(x, r), w1, b1, w2, b2, r.offsets), weight, r)
    grads = torch.autograd.grad(y, leaves, up)

    def loss(x, weight, w1, b1, w2, b2):
        has = index >= 0
        e = index.clamp_min(0)
        h = torch.relu((w1[e] * x[:, None, None]).sum(-1) + b1[e])
        out = (w2[e] * h[:, :, None]).sum(-1) + b2[e]
        return (torch.where(has[..., None], weight[..., None] * out, 0.0).sum(1) * up.double()).sum()

    wide = [t.detach().double() for t in leaves]
    assert abs((y.detach().double() * up.double()).sum() - loss(*wide)) <= 1e-5 * (y.detach() * up).abs().sum()
    for i, grad in enumerate(grads):
        way = torch.randn(wide[i].shape, device="cuda", generator=g, dtype=torch.float64)
        step = 1e-7
        moved = [[t + s * step * way if j == i else t for j, t in enumerate(wide)] for s in (1, -1)]
        slope = ((loss(*moved[0]) - loss(*moved[1])) / (2 * step)).item()
        # float32's roundings, and the difference's own 1e-15 / 1e-7
        assert abs((grad.double() * way).sum().item() - slope) <= 1e-5 * (grad.double() * way).abs().sum().item() + 1e-5


def test_second_derivatives_raise():
    from npa_amd import experts as E
    r = E.sort_rows(_index(20, 2, 3), 3)
    x, weight = torch.randn(20, 8, device="cuda", requires_grad=True), torch.rand(20, 2, device="cuda", requires_grad=True)
    w = torch.randn(3, 8, 8, device="cuda", requires_grad=True)
    res = torch.randn(40, 8, device="cuda", requires_grad=True)
    for f, t in ((lambda: E.dispatch(x, r), x), (lambda: E.combine(res, weight, r), weight),
                 (lambda: E.linear(res, w, None, r.offsets), w), (lambda: E.mlp(res, w, None, w, None, r.offsets), res)):
        d, = torch.autograd.grad(f().square().sum(), t, create_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            d.sum().backward()


# ------------------------------------------------ together, as programs run

def _mixture(rows, cols, hidden, outs, experts, choices, dtype, seed=0):
    """A pass through norm, sort, experts and back, with all of its gradients."""
    from npa_amd import experts as E
    from npa_amd import norm
    g = _gen(seed)
    x = _randn(g, rows, cols).to(dtype).requires_grad_(True)
    params = [1 + 0.1 * _randn(g, cols), 0.1 * _randn(g, cols), _randn(g, rows, choices).sigmoid()]
    params += [(_randn(g, experts, a, b) / b ** 0.5).to(dtype) for a, b in ((hidden, cols), (outs, hidden))]
    params += [_randn(g, experts, a).to(dtype) for a in (hidden, outs)]
    gamma, beta, weight, w1, w2, b1, b2 = (p.requires_grad_(True) for p in params)
    index, up = _index(rows, choices, experts, seed), _randn(g, rows, outs).to(dtype)

    def run():
        r = E.sort_rows(index, experts)
        z = norm.layer_norm(x, gamma, beta)
        y = E.combine(E.mlp(E.dispatch(z, r), w1, b1, w2, b2, r.offsets), weight, r)
        return [y.detach(), *torch.autograd.grad(y, [x, *params], up)]

    return run, x, index


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,experts,choices", [(100, 4, 1), (3000, 7, 2), (20000, 3, 1)])
def test_streams_and_graphs(rows, experts, choices, dtype):
    run, x, index = _mixture(rows, 66, 128, 18, experts, choices, dtype)
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
    for i in range(3):  # other rows and other choices every time
        with torch.no_grad():
            x.mul_(1.5)
            index.copy_(_index(rows, choices, experts, 50 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, run()))


def test_two_graphs():
    """Two captured passes replayed in turn and side by side keep to their own workspaces."""
    runs = [_mixture(2000, 66, 128, 18, 4, 2, F32, seed)[0] for seed in (1, 2)]
    want = [r() for r in runs]
    graphs, outs = [], []
    for r in runs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(r())
    sides = [torch.cuda.Stream() for _ in runs]
    for _ in range(3):
        for s, graph in zip(sides, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        for s in sides:
            torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        for out, ref in zip(outs, want):
            assert all(torch.equal(p, q) for p, q in zip(out, ref))


@pytest.mark.parametrize("choices", [1, 2])
def test_module_in_a_step(choices):
    """An automaton whose update rule is a norm and a mixture of experts, stepped and trained through step_euler; the
    gradients against torch's own modules on the same perception."""
    import types

    import npa_amd.sphops as sp
    from npa_amd import experts as E
    from npa_amd import norm
    from npa_amd.perceive import perceive
    from npa_amd.step import step_euler
    torch.manual_seed(0)
    C, N = 16, 700
    cols = 2 * C + 2 * C + 2
    rule = torch.nn.Sequential(norm.LayerNorm(cols), E.ExpertMlp(cols, 32, 2 + C, 3, choices)).cuda()
    model = types.SimpleNamespace(spatial_dims=2, eps0=0.1, alpha=0.5, model=rule, state_grad=True, density_grad=True,
                                  log_norm_grad=True, log_norm_density_grad=True, stopgrad_pos=True, stopgrad_state=False)
    grid = sp.HashGrid(dim=2, boundary="clamped", mode="grid", grid_size=[16, 16], eps=0.1, num_particles=N,
                       batch_size=1, max_particles_per_block=64)
    x = torch.rand(1, N, 2, device="cuda") * 1.2 - 0.6
    s = torch.randn(1, N, C, device="cuda")
    xs, ss, _ = step_euler(model, x, s, grid, update_prob=1.0)
    params = list(rule.parameters())
    grads = torch.autograd.grad(ss.square().sum(), params)
    z, x_bin, s_bin, _ = perceive(x, s, grid, 0.1, True, True, True, True, True, False)
    z, s_bin = z.detach().double(), s_bin.detach().double()
    ln, mix = rule[0], rule[1]
    wide = {p: p.detach().double().requires_grad_(True) for p in params}
    h = torch.nn.functional.layer_norm(z, (cols,), wide[ln.weight], wide[ln.bias], ln.eps)
    prob = torch.softmax(torch.nn.functional.linear(h, wide[mix.router.weight], wide[mix.router.bias]), -1)
    top = prob.topk(choices, -1)
    y = 0
    for j in range(choices):
        e = top.indices[0, :, j]
        a = torch.relu((wide[mix.w1][e] @ h[0, :, :, None])[..., 0] + wide[mix.b1][e])
        y = y + top.values[0, :, j, None] * ((wide[mix.w2][e] @ a[..., None])[..., 0] + wide[mix.b2][e])
    want = s_bin[0] + y[:, 2:]
    assert torch.allclose(ss[0].detach().double(), want.detach(), rtol=1e-4, atol=1e-4)
    for p, g in zip(params, grads):
        ref, = torch.autograd.grad(want.square().sum(), wide[p], retain_graph=True)
        assert (g.double() - ref).norm() <= 1e-3 * ref.norm(), p.shape


def test_module_in_16_bits():
    from npa_amd import experts as E
    mix = E.ExpertMlp(64, 96, 32, 6, 2, bias=False, device="cuda", dtype=BF16)
    x = torch.randn(5, 20, 64, device="cuda", dtype=BF16)
    y = mix(x)
    assert y.shape == (5, 20, 32) and y.dtype == BF16
    y.sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in mix.parameters())


def test_offsets_past_32_bits():
    from npa_amd import experts as E
    rows, cols = (1 << 20) + 5, 2056
    g = _gen(0)
    x = torch.randn(rows, cols, device="cuda", generator=g, dtype=BF16)
    assert x.numel() > 1 << 31
    index = torch.zeros(rows, 1, dtype=torch.int32, device="cuda")
    index[::2] = 1
    r = E.sort_rows(index, 2)
    z = E.dispatch(x, r)
    weight = torch.full((rows, 1), 2.0, device="cuda")
    back = E.combine(z, weight, r)
    for at in (slice(0, 50), slice(-50, None)):
        assert torch.equal(back[at], 2 * x[at])
    del back
    w = (torch.randn(2, 40, cols, device="cuda", generator=g) / 45).to(BF16)
    y = E.linear(z, w, None, r.offsets)
    for at, e in ((slice(0, 50), 0), (slice(-50, None), 1)):
        zd, wd = z[at].double(), w[e].double()
        _within("y", y[at], zd @ wd.T, (cols + 8) * 2 * U * (zd.abs() @ wd.abs().T))
    dy = torch.randn(rows, 40, device="cuda", generator=g).to(BF16).requires_grad_(True)
    wide = (torch.randn(2, cols, 40, device="cuda", generator=g) / 6).to(BF16)
    y = E.linear(dy, wide, None, r.offsets)
    assert y.numel() > 1 << 31
    for at, e in ((slice(0, 50), 0), (slice(-50, None), 1)):
        yd, wd = dy.detach()[at].double(), wide[e].double()
        _within("y", y.detach()[at], yd @ wd.T, 48 * 2 * U * (yd.abs() @ wd.abs().T))
    d, = torch.autograd.grad(y, dy, x)
    for at, e in ((slice(0, 50), 0), (slice(-50, None), 1)):
        xd, wd = x[at].double(), wide[e].double()
        _within("dx", d[at], xd @ wd, (cols + 8) * 2 * U * (xd.abs() @ wd.abs()))


def test_refusals():
    from npa_amd import experts as E
    index = _index(10, 2, 3)
    r = E.sort_rows(index, 3)
    x, res, w, b = (torch.randn(*s, device="cuda") for s in ((10, 4), (20, 4), (3, 5, 4), (3, 5)))
    weight = torch.rand(10, 2, device="cuda")
    host = E.Routing(*(t.cpu() for t in r))
    for call in (lambda: E.sort_rows(index.cpu(), 3), lambda: E.sort_rows(index.float(), 3),
                 lambda: E.sort_rows(index.short(), 3), lambda: E.dispatch(x.cpu(), r), lambda: E.dispatch(x.double(), r),
                 lambda: E.dispatch(x, host), lambda: E.combine(res, weight.double(), r),
                 lambda: E.combine(res, weight.to(BF16), r), lambda: E.combine(res, weight.cpu(), r),
                 lambda: E.linear(res, w.to(BF16), b, r.offsets), lambda: E.linear(res, w, b.to(BF16), r.offsets),
                 lambda: E.linear(res, w, b, r.offsets.long()), lambda: E.linear(res, w, b, r.offsets.cpu()),
                 lambda: E.linear(res.cpu(), w, b, r.offsets), lambda: E.linear(res, w.cpu(), b, r.offsets)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: E.sort_rows(torch.zeros((), dtype=torch.int32, device="cuda"), 3),
                 lambda: E.sort_rows(torch.zeros(2, 65, dtype=torch.int32, device="cuda"), 3),
                 lambda: E.sort_rows(index[:, :0], 3), lambda: E.dispatch(x[:9], r), lambda: E.dispatch(x[0], r),
                 lambda: E.combine(res[:19], weight, r), lambda: E.combine(res.view(20, 2, 2), weight, r),
                 lambda: E.combine(res, weight[:, :1], r), lambda: E.linear(res, w, b, r.offsets[:3]),
                 lambda: E.linear(res, w[:2], b, r.offsets), lambda: E.linear(res, w[:, :, :3], b, r.offsets),
                 lambda: E.linear(res, w[0], b, r.offsets), lambda: E.linear(res, w, b[:, :4], r.offsets),
                 lambda: E.linear(res.view(2, 10, 4), w, b, r.offsets), lambda: E.linear(res, w, b, r.offsets[:1]),
                 lambda: E.linear(res, w, b, r.offsets[::2]), lambda: E.linear(res, w[:, :0], b, r.offsets),
                 lambda: E.mlp(res, w, b, w, b, r.offsets), lambda: E.mlp(res, w, b, w[:, :, :3], None, r.offsets)):
        with pytest.raises(RuntimeError):
            call()
    for bad in (0, -1, 1025):
        with pytest.raises(ValueError):
            E.sort_rows(index, bad)
    for args in ((4, 8, 2, 3, 4), (4, 8, 2, 3, 0), (4, 8, 2, 1025, 1)):
        with pytest.raises(ValueError):
            E.ExpertMlp(*args)
