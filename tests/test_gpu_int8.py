"""Rows in 8 bits (npa_amd.int8): the row codes, layers as integer products, and
gradients from inputs kept in 8 bits.

The codes and integer layers are defined by float32 steps and exact sums, so
they are compared bit for bit with the same steps in torch.  Gradients are
compared with float64 at the kept rows: an fp32 sum of n products is within
(n + 8) 2^-24 of the sum of their absolute values (8: the roundings of the
scaled factor, its pieces and the joining of partial sums)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _codes(x, relu=False):
    """Codes and scales by the definition, in float32 on the CPU (numpy rounds half to even)."""
    v = x.detach().float().cpu().numpy().reshape(-1, x.shape[-1])
    if relu:
        v = np.where(v <= 0, np.float32(0), v)
    with np.errstate(all="ignore"):
        m = np.abs(v).max(1)
        fine = np.isfinite(m)
        m = np.maximum(np.where(fine, m, 0), np.float32(2.0 ** -100)).astype(np.float32)
        q = np.rint(v * (np.float32(127) / m)[:, None])
        if relu:
            q = np.where(v > 0, np.maximum(q, 1), 0)
        q = np.where(fine[:, None], q, 0).astype(np.int8)
        s = np.where(fine, m / np.float32(127), np.float32(np.nan)).astype(np.float32)
    return torch.from_numpy(q).cuda(), torch.from_numpy(s).cuda()


def _same(a, b):
    return torch.equal(torch.nan_to_num(a.float(), nan=12345.0), torch.nan_to_num(b.float(), nan=12345.0))


def _check_rows(x, relu=False, align=4):
    from npa_amd import int8
    r = int8.quantize_rows(x, relu=relu, align=align)
    q, s = _codes(x, relu)
    cols = x.shape[-1]
    assert r.shape == tuple(x.shape) and r.codes.shape == (q.shape[0], -(-cols // align) * align)
    assert torch.equal(r.codes[:, :cols], q) and not r.codes[:, cols:].any() and _same(r.scale, s)
    for dtype in (F32, BF16, F16):
        want = (q.float() * s[:, None]).to(dtype).reshape(x.shape)
        assert _same(int8.restore_rows(r, dtype), want)
    return r


# ------------------------------------------------------------------ rows

@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cols", [1, 2, 3, 4, 7, 31, 64, 83, 163, 256, 1000, 2049, 4097, 20000])
def test_rows_match_their_definition(cols, dtype):
    for rows in (1, 2, 65, 700):
        x = torch.randn(rows, cols, device="cuda", generator=_gen(cols + rows)).to(dtype)
        _check_rows(x)
        _check_rows(x, relu=True, align=16)


def test_rows_of_the_widest_and_of_many():
    _check_rows(torch.randn(3, 65536, device="cuda", generator=_gen(0)))
    _check_rows(torch.randn(300001, 19, device="cuda", generator=_gen(1)))
    _check_rows(torch.randn(70001, 66, device="cuda", generator=_gen(2)).to(BF16))


def test_special_rows():
    """Zeros, subnormals, the largest values, ties, and rows that are not finite, which touch no other row."""
    nan, inf, big = float("nan"), float("inf"), 3.0e38
    rows = [[0.0, -0.0, 0.0, 0.0, 0.0], [1e-45, -1e-40, 0.0, 1e-38, 0.0], [big, -big, 1e30, 0.0, 1.0],
            [127.0, 0.5, 1.5, -2.5, -0.5], [254.0, 1.0, 3.0, -5.0, 253.0], [1.0, nan, 2.0, 0.0, 0.0],
            [inf, 1.0, 0.0, 0.0, 2.0], [1.0, 2.0, -inf, 3.0, 4.0], [-1.0, -2.0, -3.0, -4.0, -5.0],
            [1e-20, 1.0, 0.0, 0.0, 0.0], [0.0, 0.0, 0.0, 0.0, 7.0]]
    x = torch.tensor(rows, device="cuda")
    r = _check_rows(x)
    assert r.codes[3, :5].tolist() == [127, 0, 2, -2, 0]
    assert torch.isnan(r.scale).tolist() == [False] * 5 + [True] * 3 + [False] * 3
    k = _check_rows(x, relu=True)
    fine = ~torch.isnan(r.scale)
    fine[7] = True  # its infinity is below zero
    assert torch.equal((k.codes[:, :5] > 0)[fine], (x > 0)[fine])
    wide = x.repeat(1, 300)  # the same values in rows of 1500
    assert torch.equal(_check_rows(wide).codes[:, :5], r.codes[:, :5])


def test_strides_alignments_and_leading_dimensions():
    g = _gen(3)
    base = torch.randn(67, 90, device="cuda", generator=g)
    for x in (base[:, :83], base[:, 1:84], base[::3, 2:], base.t(), base[:1].expand(9, 90), base[0], base[:, 5:6],
              base.reshape(67, 9, 10), base.reshape(67, 9, 10).transpose(0, 1), base.flatten()[1:1 + 66 * 90].view(66, 90)):
        _check_rows(x)
        _check_rows(x.to(BF16) if x.is_contiguous() else x)
    half = base.to(F16)
    for x in (half[:, 1:84], half[::2, 3:], half.flatten()[1:1 + 66 * 90].view(66, 90), half[:1].expand(5, 90)):
        _check_rows(x)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("cols", [63, 64, 65, 71, 72, 73, 95, 127, 128, 191, 255, 256, 383, 511, 767, 1023, 1535, 2047,
                                  3000, 4095, 6143, 6144, 6145, 8193])
def test_rows_at_odd_places(cols, dtype):
    """Rows of 2-byte values that start between words: all of them, every second
    one, a single one; the largest value first, last or not finite."""
    flat = torch.randn(1 + 9 * (cols + 1), device="cuda", generator=_gen(cols)).to(dtype)
    flat[0] = flat[-1] = 10000  # outside every row below
    for start, stride in ((1, cols + cols % 2), (0, cols + 1 - cols % 2), (1, cols + 1 - cols % 2)):
        x = torch.as_strided(flat, (8, cols), (stride, 1), start)
        _check_rows(x, relu=cols % 4 == 3)
        _check_rows(x[:1])
    x[2, 0], x[3, -1], x[4, cols // 2], x[5, 0], x[6, -1] = 77, -88, float("nan"), float("inf"), float("nan")
    _check_rows(x, align=16)
    _check_rows(x, relu=True)


def test_no_rows():
    from npa_amd import int8
    r = int8.quantize_rows(torch.empty(0, 83, device="cuda"))
    assert r.codes.shape == (0, 84) and int8.restore_rows(r).shape == (0, 83)
    dw, db = int8.weight_grad(r, torch.empty(0, 19, device="cuda"))
    assert not dw.any() and not db.any() and dw.shape == (19, 83)
    w = int8.quantize_rows(torch.randn(7, 83, device="cuda"), align=16)
    assert int8.linear(torch.empty(0, 83, device="cuda"), w).shape == (0, 7)
    assert int8.linear(torch.empty(3, 0, 83, device="cuda"), w).shape == (3, 0, 7)


# --------------------------------------------------------------- products

def _layer(q, s, w, bias):
    """The integer layer by its definition: exact sums, then float32 steps one at a time."""
    total = (q.double() @ w.codes[:, :w.shape[1]].double().T).float()
    y = total * (s[:, None] * w.scale)
    return y if bias is None else y + bias


def _check_linear(rows, cols, outs, dtype, bias=True, seed=0, ld=16):
    from npa_amd import int8
    g = _gen(seed + rows + cols)
    x = torch.randn(rows, cols, device="cuda", generator=g).to(dtype)
    w = int8.quantize_rows(torch.randn(outs, cols, device="cuda", generator=g), align=ld)
    b = torch.randn(outs, device="cuda", generator=g) if bias else None
    y = int8.linear(x, w, b)
    assert y.dtype == dtype and torch.equal(y, _layer(*_codes(x), w, b).to(dtype))
    return x, w, b, y


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows", [1, 2, 7, 16, 17, 32, 33, 64, 65, 100, 128, 129, 200, 256, 257, 600])
def test_linear_matches_its_definition(rows, dtype):
    for cols, outs in ((83, 128), (128, 19), (16, 16), (1, 1), (17, 300), (1000, 257), (513, 64)):
        _check_linear(rows, cols, outs, dtype, bias=outs != 300)


@pytest.mark.parametrize("rows,cols,outs,dtype", [(1, 4096, 4096, BF16), (1, 8192, 33, F32), (3, 20000, 130, F16),
                                                  (37, 2049, 8190, F16), (1, 65536, 5, F32), (300, 65536, 40, BF16),
                                                  (2048, 1024, 2048, BF16), (1111, 4100, 1030, F32),
                                                  (5000, 83, 128, F32), (100003, 66, 18, F32), (1, 16, 20000, F16)])
def test_linear_at_larger_sizes(rows, cols, outs, dtype):
    _check_linear(rows, cols, outs, dtype)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9])
def test_linear_of_single_tokens(rows):
    """Few rows of every length that shares out over a workgroup's threads and
    waves, and lengths and row counts past that."""
    for cols in (5, 64, 127, 129, 1000, 2048, 4095, 4097, 8192, 16383, 16384, 16385):
        _check_linear(rows, cols, 35, (F32, BF16, F16)[cols % 3])
    _check_linear(rows, 4096, 4096, BF16, ld=128)


@pytest.mark.parametrize("rows,outs", [(4097, 3333), (1500, 2008), (700, 131), (65600, 33)])
@pytest.mark.parametrize("cols", [70, 128, 200, 300, 400])
def test_linear_tiles(rows, cols, outs):
    """Ragged tiles of every size, channel counts that are no multiple of a
    store's, and even and odd numbers of steps."""
    _check_linear(rows, cols, outs, (F32, BF16, F16)[(rows + cols) % 3], bias=cols != 200)


@pytest.mark.parametrize("rows,cols", [(1, 32768), (1, 32769), (2, 16385), (6, 4095), (8, 4096), (8, 4097), (9, 1),
                                       (10, 83), (13, 1000), (15, 2047), (16, 2048), (16, 2049), (17, 64)])
def test_linear_of_a_few_tokens(rows, cols):
    """Rows that one launch holds and the first that it does not, in each type."""
    for dtype in (F32, BF16, F16):
        _check_linear(rows, cols, 37, dtype)


@pytest.mark.parametrize("rows,outs", [(17, 5), (64, 64), (65, 130), (190, 600)])
def test_linear_of_each_number_of_steps(rows, outs):
    """1 to 10 steps of 128 columns, whole and begun ones."""
    for steps in range(1, 11):
        _check_linear(rows, 128 * steps, outs, BF16)
        _check_linear(rows, 128 * steps - 127, outs, F32, bias=steps % 2 == 0)


def test_linear_extremes():
    """The largest sums (all codes 127, both signs), padded weights, rows that are not finite, strides."""
    from npa_amd import int8
    ones = torch.ones(3, 65536, device="cuda")
    ones[1] = -1
    w = int8.quantize_rows(torch.ones(4, 65536, device="cuda"), align=16)
    y = int8.linear(ones, w)
    assert torch.equal(y, _layer(*_codes(ones), w, None))
    _check_linear(40, 100, 50, F32, ld=64)
    x, w, b, y = _check_linear(130, 83, 40, F32, seed=5)
    bad = x.clone()
    bad[7, 3], bad[128, 82] = float("nan"), float("inf")
    got = int8.linear(bad, w, b)
    keep = torch.ones(130, dtype=torch.bool, device="cuda")
    keep[[7, 128]] = False
    assert torch.isnan(got[~keep]).all() and torch.equal(got[keep], y[keep])
    wide = torch.zeros(130, 100, device="cuda")
    wide[:, 9:92] = x
    assert torch.equal(int8.linear(wide[:, 9:92], w, b), y)
    assert torch.equal(int8.linear(x.reshape(10, 13, 83), w, b), y.reshape(10, 13, 40))
    assert torch.equal(int8.linear(x[5], w, b), y[5])
    assert torch.equal(int8.linear(x.t().contiguous().t(), w, b), y)


def test_int8_linear_module():
    from npa_amd import int8
    for bias in (True, False):
        layer = torch.nn.Linear(96, 40, bias=bias).cuda()
        m = int8.Int8Linear(layer)
        x = torch.randn(9, 96, device="cuda", generator=_gen(1))
        with torch.no_grad():
            y, ref = m(x), layer(x)
        # each factor is within half a code: |y - ref| <= (|x| sw + sx |w|) / 2 + ... summed over 96 products
        sx, sw = x.abs().amax(1) / 127, layer.weight.abs().amax(1) / 127
        bound = 0.5 * (x.abs().sum(1)[:, None] * sw + sx[:, None] * layer.weight.abs().sum(1) + 48 * sx[:, None] * sw)
        assert torch.all((y - ref).abs() <= bound * (1 + 1e-5))
        m2 = int8.Int8Linear(torch.nn.Linear(96, 40, bias=bias).cuda())
        m2.load_state_dict(m.state_dict())
        assert torch.equal(m2(x), y)


MLP_SHAPES = [(83, 19), (66, 18), (50, 14), (163, 35), (4, 4), (8, 8), (13, 33), (32, 32), (33, 5), (96, 64), (97, 9),
              (128, 33), (160, 16), (168, 64)]


def _mlp_case(rows, nin, nout, seed):
    from npa_amd import int8
    g = _gen(seed)
    z = torch.randn(rows, nin, device="cuda", generator=g)
    w1 = torch.randn(128, nin, device="cuda", generator=g) / nin ** 0.5
    w2 = torch.randn(nout, 128, device="cuda", generator=g) / 128 ** 0.5
    b1, b2 = torch.randn(128, device="cuda", generator=g), torch.randn(nout, device="cuda", generator=g)
    return z, int8.quantize_rows(w1, align=16), b1, int8.quantize_rows(w2, align=16), b2


def _mlp_ref(z, w1, b1, w2, b2):
    h = torch.relu(_layer(*_codes(z), w1, b1))
    return _layer(*_codes(h), w2, b2)


@pytest.mark.parametrize("shape", MLP_SHAPES)
def test_int8_mlp_matches_its_definition(shape):
    from npa_amd import int8
    for rows in (1, 31, 33, 65, 4097):
        case = _mlp_case(rows, *shape, rows)
        assert torch.equal(int8.mlp(*case), _mlp_ref(*case))
    z, w1, b1, w2, b2 = case
    assert torch.equal(int8.mlp(z, w1, None, w2, None), _mlp_ref(z, w1, None, w2, None))


def test_int8_mlp_many_rows_and_special_rows():
    from npa_amd import int8
    case = _mlp_case(300001, 83, 19, 1)
    y = int8.mlp(*case)
    assert torch.equal(y, _mlp_ref(*case))
    bad = case[0].clone()
    bad[40, 82], bad[41, 0], bad[300000, 5] = float("nan"), float("inf"), float("-inf")
    got = int8.mlp(bad, *case[1:])
    keep = torch.ones(300001, dtype=torch.bool, device="cuda")
    keep[[40, 41, 300000]] = False
    assert torch.isnan(got[~keep]).all() and torch.equal(got[keep], y[keep])
    zero = torch.zeros_like(case[0][:70])
    assert torch.equal(int8.mlp(zero, *case[1:]), _mlp_ref(zero, *case[1:]))
    assert torch.equal(int8.mlp(case[0][:98].reshape(2, 49, 83), *case[1:]).reshape(98, 19), y[:98])
    assert int8.mlp(case[0][:0], *case[1:]).shape == (0, 19)


def test_int8_mlp_module_in_and_out_of_the_kernels_shapes():
    from npa_amd import int8
    from npa_amd import mlp as M
    for sizes in ((83, 128, 19), (83, 64, 19), (200, 128, 19)):
        net = torch.nn.Sequential(torch.nn.Linear(sizes[0], sizes[1]), torch.nn.ReLU(),
                                  torch.nn.Linear(sizes[1], sizes[2], bias=False)).cuda()
        m = int8.Int8Mlp(net)
        assert m.fused == (sizes == (83, 128, 19))
        z = torch.randn(50, sizes[0], device="cuda", generator=_gen(2))
        with torch.no_grad():
            y, ref = M.mlp(m, z), net(z)
        assert ((y - ref).norm() < 0.03 * ref.norm()).item()  # two layers at 7 bits


# -------------------------------------------------------------- gradients

def _within(name, got, ref, bound):
    err = (got.double() - ref).abs()
    assert torch.all(err <= bound + 1e-30), f"{name}: {(err - bound).max().item():.3g} over its bound"


@pytest.mark.parametrize("cols,outs", [(1, 1), (4, 4), (19, 83), (83, 128), (128, 19), (163, 35), (33, 129), (300, 5),
                                       (256, 256), (1000, 130)])
@pytest.mark.parametrize("rows", [1, 31, 33, 200, 5003])
def test_weight_grad_matches_float64(rows, cols, outs):
    from npa_amd import int8
    g = _gen(rows + cols)
    x = torch.randn(rows, cols, device="cuda", generator=g) * torch.exp(3 * torch.randn(rows, 1, device="cuda", generator=g))
    dy = torch.randn(rows, outs, device="cuda", generator=g) / rows
    r = int8.quantize_rows(x)
    kept = r.codes[:, :cols].double() * r.scale.double()[:, None]
    dw, db = int8.weight_grad(r, dy)
    n = (rows + 8) * EPS
    _within("dW", dw, dy.double().T @ kept, n * (dy.double().abs().T @ kept.abs()))
    _within("db", db, dy.double().sum(0), n * dy.double().abs().sum(0))
    again = int8.weight_grad(r, dy, bias=False)
    assert torch.equal(again[0], dw) and again[1] is None


@pytest.mark.parametrize("rows,cols,outs", [(1 << 18, 83, 128), (300007, 128, 19), (8192, 1024, 1024), (70000, 300, 7)])
def test_weight_grad_of_many_rows(rows, cols, outs):
    """2-norms within 4e-6, several times what the roundings of long sums
    measure; a tile of 32 rows left out is off by (32 / rows)^(1/2), 1e-2."""
    from npa_amd import int8
    g = _gen(rows)
    r = int8.quantize_rows(torch.randn(rows, cols, device="cuda", generator=g))
    dy = torch.randn(rows, outs, device="cuda", generator=g)
    kept = r.codes[:, :cols].double() * r.scale.double()[:, None]
    dw, db = int8.weight_grad(r, dy)
    for got, ref in ((dw, dy.double().T @ kept), (db, dy.double().sum(0))):
        assert ((got.double() - ref).norm() <= 4e-6 * ref.norm()).item()


def test_gradients_of_sums_that_cancel():
    """Over 2^19 rows of random sign the errors of the matrix cores' sums, all of
    one sign, would add up to 4e-6 of db1; rounding alone leaves under 1e-6."""
    from npa_amd import int8
    from npa_amd import mlp as M
    net, g = _net(83, 19, True, 2)
    z = torch.randn(1 << 19, 83, device="cuda", generator=g)
    up = torch.randn(1 << 19, 19, device="cuda", generator=g)
    w1, b1, w2 = (t.detach().double() for t in (net[0].weight, net[0].bias, net[2].weight))
    zd = _kept(z)
    a = zd @ w1.T + b1
    up[(a.abs() < 1e-5).any(1)] = 0
    M.mlp(net, z, checkpoint="int8").backward(up)
    da = (up.double() @ w2) * (a > 0)
    for got, ref in ((net[0].weight.grad, da.T @ zd), (net[0].bias.grad, da.sum(0)),
                     (net[2].weight.grad, up.double().T @ a.clamp_min(0)),
                     (int8.weight_grad(int8.quantize_rows(z), up)[0], up.double().T @ zd)):
        assert ((got.double() - ref).norm() <= 1.5e-6 * ref.norm()).item()


def test_weight_grad_ranges():
    """Upstreams from 1e-30 to 1e30 a row, of one sign, and rows that are not finite."""
    from npa_amd import int8
    g = _gen(4)
    x = torch.randn(500, 40, device="cuda", generator=g)
    r = int8.quantize_rows(x)
    kept = r.codes[:, :40].double() * r.scale.double()[:, None]
    for size in (1e-30, 1e-12, 1e12, 1e30):
        dy = torch.rand(500, 24, device="cuda", generator=g) * size
        dw, db = int8.weight_grad(r, dy)
        _within("dW", dw, dy.double().T @ kept, 508 * EPS * (dy.double().T @ kept.abs()))
        _within("db", db, dy.double().sum(0), 508 * EPS * dy.double().sum(0))
    x[3, 5] = float("nan")
    dw, db = int8.weight_grad(int8.quantize_rows(x), dy)
    assert torch.isnan(dw).all() and torch.isfinite(db).all()


def _net(nin, nout, bias2, seed, hidden=128):
    g = _gen(seed)
    net = torch.nn.Sequential(torch.nn.Linear(nin, hidden), torch.nn.ReLU(),
                              torch.nn.Linear(hidden, nout, bias=bias2)).cuda()
    with torch.no_grad():
        for p in net.parameters():
            p.copy_(torch.randn(p.shape, device="cuda", generator=g) / max(p.shape[-1], 8) ** 0.5)
    return net, g


def _kept(z):
    q, s = _codes(z)
    return q.double() * s.double()[:, None]


@pytest.mark.parametrize("shape", MLP_SHAPES)
@pytest.mark.parametrize("rows", [1, 31, 33, 65, 5000])
def test_mlp_with_checkpoint_matches_float64(shape, rows):
    from npa_amd import mlp as M
    nin, nout = shape
    net, g = _net(nin, nout, rows % 2 == 1, rows + nin)
    z = torch.randn(rows, nin, device="cuda", generator=g)
    up = torch.randn(rows, nout, device="cuda", generator=g)
    w1, b1, w2 = (t.detach().double() for t in (net[0].weight, net[0].bias, net[2].weight))
    zd = _kept(z)
    a = zd @ w1.T + b1
    ea = (nin + 8) * EPS * (zd.abs() @ w1.abs().T + b1.abs())
    up[(a.abs() <= 2 * ea).any(1)] = 0  # within rounding of the ReLU's kink
    zr = z.clone().requires_grad_(True)
    y = M.mlp(net, zr, checkpoint="int8")
    # the forward takes z itself
    az, mz = z.double() @ w1.T + b1, z.double().abs() @ w1.abs().T + b1.abs()
    b2 = net[2].bias.detach().double() if net[2].bias is not None else torch.zeros(nout, device="cuda").double()
    _within("y", y.detach(), az.clamp_min(0) @ w2.T + b2, 136 * EPS * (az.clamp_min(0) @ w2.abs().T + b2.abs())
            + (nin + 8) * EPS * mz @ w2.abs().T)
    y.backward(up)
    h, ud, on = a.clamp_min(0), up.double(), (a > 0).double()
    da, eda = (ud @ w2) * on, (nout + 8) * EPS * (ud.abs() @ w2.abs()) * on
    _within("dz", zr.grad, da @ w1, 136 * EPS * (da.abs() @ w1.abs()) + eda @ w1.abs())
    n = (rows + 8) * EPS
    _within("dW1", net[0].weight.grad, da.T @ zd, n * (da.abs().T @ zd.abs()) + eda.T @ zd.abs())
    _within("db1", net[0].bias.grad, da.sum(0), n * da.abs().sum(0) + eda.sum(0))
    _within("dW2", net[2].weight.grad, ud.T @ h, n * (ud.abs().T @ h) + ud.abs().T @ ea)
    if net[2].bias is not None:
        _within("db2", net[2].bias.grad, ud.sum(0), n * ud.abs().sum(0))


@pytest.mark.parametrize("shape", [(150, 35), (165, 20), (112, 40)])
def test_mlp_with_checkpoint_at_more_widths(shape):
    test_mlp_with_checkpoint_matches_float64(shape, 65)
    test_mlp_with_checkpoint_matches_float64(shape, 9000)


@pytest.mark.parametrize("rows,shape", [(300001, (83, 19)), (300001, (163, 40)), (32769, (130, 32)), (100000, (66, 18))])
def test_mlp_with_checkpoint_many_rows(rows, shape):
    """2-norms within 4e-6; a row tile left out or read twice is off by (32 / rows)^(1/2), 1e-2."""
    from npa_amd import mlp as M
    nin, nout = shape
    net, g = _net(nin, nout, True, nin)
    z = torch.randn(rows, nin, device="cuda", generator=g)
    up = torch.randn(rows, nout, device="cuda", generator=g)
    w1, b1, w2 = (t.detach().double() for t in (net[0].weight, net[0].bias, net[2].weight))
    zd = _kept(z)
    a = zd @ w1.T + b1
    up[(a.abs() < 1e-5).any(1)] = 0
    zr = z.clone().requires_grad_(True)
    M.mlp(net, zr, checkpoint="int8").backward(up)
    h, ud = a.clamp_min(0), up.double()
    da = (ud @ w2) * (a > 0)
    pairs = [("dz", zr.grad, da @ w1), ("dW1", net[0].weight.grad, da.T @ zd), ("db1", net[0].bias.grad, da.sum(0)),
             ("dW2", net[2].weight.grad, ud.T @ h), ("db2", net[2].bias.grad, ud.sum(0))]
    for name, got, ref in pairs:
        assert ((got.double() - ref).norm() <= 4e-6 * ref.norm()).item(), name
    first = [p[1].clone() for p in pairs]
    net.zero_grad()
    zr.grad = None
    M.mlp(net, zr, checkpoint="int8").backward(up)
    again = [zr.grad, net[0].weight.grad, net[0].bias.grad, net[2].weight.grad, net[2].bias.grad]
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    last = rows - rows % 32
    assert torch.all((zr.grad[last - 32:].double() - pairs[0][2][last - 32:]).abs() <= 1e-5 * pairs[0][2].abs().max())


def test_mlp_with_checkpoint_against_differences():
    """Directional differences in float64 of sum(y * up) at the kept rows: the
    step of 1e-5 leaves 1e-9 of curvature (none away from kinks) and 1e-10 of
    rounding, the fp32 gradients 1e-5 of their norm."""
    from npa_amd import mlp as M
    net, g = _net(83, 19, True, 9)
    z = torch.randn(300, 83, device="cuda", generator=g)
    up = torch.randn(300, 19, device="cuda", generator=g)
    params = [p.detach().double() for p in net.parameters()]
    zd = _kept(z)
    up[((zd @ params[0].T + params[1]).abs() < 1e-2).any(1)] = 0
    keep = (up != 0).any(1)
    assert keep.sum() > 50

    def loss(zv, w1, b1, w2, b2):
        return ((torch.relu(zv @ w1.T + b1) @ w2.T + b2) * up.double()).sum()

    zr = z.clone().requires_grad_(True)
    y = M.mlp(net, zr, checkpoint="int8")
    grads = torch.autograd.grad(y, [zr, *net.parameters()], up)
    at = [zd, *params]
    for i, grad in enumerate(grads):
        d = torch.randn(at[i].shape, device="cuda", dtype=torch.float64, generator=g)
        d = d / d.norm()
        plus, minus = ([t + s * 1e-5 * d if j == i else t for j, t in enumerate(at)] for s in (1, -1))
        slope = (loss(*plus) - loss(*minus)) / 2e-5
        assert abs(slope - (grad.double() * d).sum()) <= 1e-5 * grad.double().norm() + 1e-7


def test_what_checkpoints_keep(monkeypatch):
    """The saved tensors are the codes, scales and weights; nothing is kept
    without a backward; other shapes and single layers keep codes too."""
    from npa_amd import int8
    from npa_amd import mlp as M
    net, g = _net(83, 19, True, 1)
    z = torch.randn(2, 500, 83, device="cuda", generator=g)
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        y = M.mlp(net, z.requires_grad_(True), checkpoint="int8")
    weights = {p.data_ptr() for p in net.parameters()}
    assert sum(t.numel() * t.element_size() for t in saved if t.data_ptr() not in weights) == 1000 * (84 + 4)
    y.sum().backward()
    calls, call = [], int8._lib.sphops_quantize_rows
    monkeypatch.setattr(int8._lib, "sphops_quantize_rows", lambda *a: calls.append(1) or call(*a))
    with torch.no_grad():
        M.mlp(net, z, checkpoint="int8")
    assert not calls
    with pytest.raises(ValueError):
        M.mlp(net, z, checkpoint="int4")
    for hidden, nout in ((64, 19), (256, 130)):  # layers of their own
        net, g = _net(83, nout, True, hidden, hidden)
        zr = torch.randn(700, 83, device="cuda", generator=g).requires_grad_(True)
        up = torch.randn(700, nout, device="cuda", generator=g)
        del calls[:]
        y = M.mlp(net, zr, checkpoint="int8")
        assert len(calls) == 2
        with torch.no_grad():
            a = net[0](zr)
            assert torch.allclose(y, net[2](torch.relu(a)), rtol=1e-5, atol=1e-5)
            up[(a.abs() <= 1e-5).any(1)] = 0
        y.backward(up)
        w1, w2 = net[0].weight.detach().double(), net[2].weight.detach().double()
        qh, sh = _codes(a, relu=True)
        da = (up.double() @ w2) * (a > 0)
        for got, ref in ((zr.grad, da @ w1), (net[0].weight.grad, da.T @ _kept(zr)), (net[0].bias.grad, da.sum(0)),
                         (net[2].weight.grad, up.double().T @ (qh.double() * sh.double()[:, None])),
                         (net[2].bias.grad, up.double().sum(0))):
            # a code on another side of a tie (torch's a here, the layer's there) moves one value by 1/127
            assert ((got.double() - ref).norm() <= 1e-4 * ref.norm()).item()
        with torch.no_grad():
            M.mlp(net, zr, checkpoint="int8")
        assert len(calls) == 2


def test_checkpoint_of_a_function():
    from npa_amd import int8
    g = _gen(6)
    x = torch.randn(40, 30, device="cuda", generator=g).requires_grad_(True)
    w = torch.randn(30, 30, device="cuda", generator=g).requires_grad_(True)
    up = torch.randn(40, 30, device="cuda", generator=g)

    def f(v, m):
        return torch.tanh(v @ m) * v

    y = int8.checkpoint(f, x, w)
    assert torch.equal(y.detach(), f(x, w).detach())
    y.backward(up)
    kept = int8.restore_rows(int8.quantize_rows(x)).requires_grad_(True)
    want = torch.autograd.grad(f(kept, w), [kept, w], up)
    assert torch.equal(x.grad, want[0]) and torch.equal(w.grad, want[1])
    fixed = x.detach()
    y = int8.checkpoint(f, fixed, w)
    assert torch.equal(torch.autograd.grad(y, w, up)[0], want[1])
    assert not int8.checkpoint(f, fixed, w.detach()).requires_grad


def test_checkpoint_of_a_function_under_autocast():
    """The second run is under the forward's autocast: the same gradients as autograd's there."""
    from npa_amd import int8
    g = _gen(8)
    x = torch.randn(40, 64, device="cuda", generator=g).requires_grad_(True)
    m = torch.randn(64, 32, device="cuda", generator=g).requires_grad_(True)
    up = torch.randn(40, 32, device="cuda", generator=g).to(BF16)
    f = lambda v, w: torch.tanh(v @ w)
    with torch.autocast("cuda", BF16):
        y = int8.checkpoint(f, x, m)
        kept = int8.restore_rows(int8.quantize_rows(x)).requires_grad_(True)
        ref = f(kept, m)
    assert y.dtype == BF16
    for got, want in zip(torch.autograd.grad(y, [x, m], up), torch.autograd.grad(ref, [kept, m], up)):
        assert got.dtype == F32 and torch.equal(got, want)


def test_special_rows_with_checkpoint():
    """A row that is not finite gives NaN where it reaches: its own dz stays the
    upstream's product or NaN, no other row's changes."""
    from npa_amd import mlp as M
    net, g = _net(83, 19, True, 3)
    z = torch.randn(99, 83, device="cuda", generator=g)
    up = torch.randn(99, 19, device="cuda", generator=g)
    grads = []
    for bad in (False, True):
        v = z.clone()
        if bad:
            v[40, 82], v[41, 0] = float("nan"), float("inf")
        v.requires_grad_(True)
        net.zero_grad()
        M.mlp(net, v, checkpoint="int8").backward(up)
        grads.append((v.grad, net[0].weight.grad.clone(), net[2].bias.grad.clone()))
    keep = torch.ones(99, dtype=torch.bool, device="cuda")
    keep[[40, 41]] = False
    assert torch.equal(grads[0][0][keep], grads[1][0][keep])
    assert torch.isnan(grads[1][1]).any() and torch.equal(grads[0][2], grads[1][2])


# ---------------------------------------------- streams, graphs, the path

def test_other_streams_and_graphs():
    from npa_amd import int8
    from npa_amd import mlp as M
    net, g = _net(83, 19, True, 8)
    z = torch.randn(3000, 83, device="cuda", generator=g)
    up = torch.randn(3000, 19, device="cuda", generator=g)
    w1, w2 = (int8.quantize_rows(m.weight, align=16) for m in (net[0], net[2]))
    b1, b2 = net[0].bias.detach(), net[2].bias.detach()

    def work(v):
        v = v.detach().requires_grad_(True)
        y = M.mlp(net, v, checkpoint="int8")
        grads = torch.autograd.grad(y, [v, *net.parameters()], up)
        with torch.no_grad():
            return [y.detach(), *grads, int8.mlp(v, w1, b1, w2, b2), int8.linear(v, w1, b1),
                    int8.linear(v[:1], w1, b1), *int8.weight_grad(int8.quantize_rows(v), up)]

    ref = work(z)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work(z)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    still = z.clone()
    with torch.cuda.stream(side):
        work(still)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work(still)
    for k in range(4):
        v = z * (1 + k)
        want = work(v)
        still.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, outs))


def test_refusals():
    from npa_amd import int8
    x = torch.randn(8, 32, device="cuda")
    w = int8.quantize_rows(torch.randn(16, 32, device="cuda"), align=16)
    r = int8.quantize_rows(x)
    bad = [(TypeError, lambda: int8.quantize_rows(x.double())), (TypeError, lambda: int8.quantize_rows(x.cpu())),
           (TypeError, lambda: int8.quantize_rows(x.int())), (RuntimeError, lambda: int8.quantize_rows(x[:, :0])),
           (RuntimeError, lambda: int8.quantize_rows(x.sum())),
           (RuntimeError, lambda: int8.quantize_rows(torch.empty(1, 65537, device="cuda"))),
           (ValueError, lambda: int8.quantize_rows(x, align=3)), (TypeError, lambda: int8.restore_rows(r, torch.float64)),
           (RuntimeError, lambda: int8.restore_rows(int8.Rows8(r.codes, r.scale, (8, 33)))),
           (RuntimeError, lambda: int8.restore_rows(int8.Rows8(r.codes[:, ::2], r.scale, (8, 16)))),
           (RuntimeError, lambda: int8.restore_rows(int8.Rows8(r.codes, r.scale[:7], (8, 32)))),
           (TypeError, lambda: int8.restore_rows(int8.Rows8(r.codes.int(), r.scale, (8, 32)))),
           (TypeError, lambda: int8.weight_grad(r, x.double())), (TypeError, lambda: int8.weight_grad(r, x.cpu())),
           (RuntimeError, lambda: int8.weight_grad(r, x[:7])),
           (RuntimeError, lambda: int8.linear(x[:, :31], w)), (TypeError, lambda: int8.linear(x.double(), w)),
           (TypeError, lambda: int8.linear(x, w, torch.zeros(16, device="cuda", dtype=torch.float16))),
           (RuntimeError, lambda: int8.linear(x, w, torch.zeros(15, device="cuda"))),
           (RuntimeError, lambda: int8.linear(x.clone().requires_grad_(True), w)),
           (RuntimeError, lambda: int8.linear(x[:, :20], int8.quantize_rows(torch.randn(16, 20, device="cuda")))),
           (RuntimeError, lambda: int8.mlp(x, w, None, w, None)),
           (TypeError, lambda: int8.Int8Mlp(torch.nn.Sequential(torch.nn.Linear(4, 4), torch.nn.GELU()).cuda())),
           (TypeError, lambda: int8.Int8Linear(torch.nn.Linear(4, 4)))]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
    assert int8.linear(x.clone().requires_grad_(True).detach(), w).shape == (8, 16)


def test_rollout_with_checkpoint_and_in_integers():
    """step_euler with its MLP's input in 8 bits: the same states, and weight
    gradients near those without (each input is within half of 1/127 of its
    row's largest, and the errors are independent); then an integer step, whose
    two layers are off by about 1% each."""
    import helpers as H
    import npa_amd.sphops as sp
    from npa_amd import int8, step
    from test_gpu_step import _Model
    c = H.random_case("int8", 2, 2000, 16, 3, 12, 0.15, False, "grid", uniform=False, sigma=0.3, seed=3)
    grid = sp.HashGrid(dim=3, boundary="clamped", mode="grid", grid_size=list(c.grid_size), eps=c.eps,
                       num_particles=c.N, batch_size=c.B, max_particles_per_block=c.maxp)
    torch.manual_seed(0)
    model = _Model(3, 16, hidden=128).cuda()
    x0, s0 = torch.from_numpy(c.x).cuda(), torch.from_numpy(c.s).cuda()
    runs = []
    for mode in (None, "int8"):
        model.zero_grad()
        x, s = x0, s0.clone().requires_grad_(True)
        leaf = s
        for _ in range(2):
            x, s, _ = step.step_euler(model, x, s, grid, update_prob=1.0, checkpoint=mode)
        s.square().mean().backward()
        runs.append((s.detach(), leaf.grad, [p.grad.clone() for p in model.model.parameters()]))
    assert torch.allclose(runs[0][0], runs[1][0], rtol=1e-4, atol=1e-5)
    for a, b in zip([runs[0][1], *runs[0][2]], [runs[1][1], *runs[1][2]]):
        assert ((a - b).norm() <= 0.05 * a.norm()).item()
    exact = model.model
    with torch.no_grad():
        _, se, _ = step.step_euler(model, x0, s0, grid, update_prob=1.0)
        model.model = int8.Int8Mlp(exact)
        _, sq, _ = step.step_euler(model, x0, s0, grid, update_prob=1.0)
        model.model = exact
    assert ((sq - se).norm() <= 0.02 * se.norm()).item()
