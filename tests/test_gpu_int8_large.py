"""Rows in 8 bits where byte and element offsets pass 32 bits: the first and last
rows of large calls against the definition (the sums over rows against a call
on each half)."""
import pytest
import torch

from test_gpu_int8 import _codes, _kept, _layer, _mlp_ref, _net

pytestmark = pytest.mark.gpu

ENDS = (slice(0, 70), slice(-70, None))


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def test_rows_past_32_bits():
    from npa_amd import int8
    x = torch.randn((1 << 22) + 3, 601, device="cuda", generator=_gen(0)).bfloat16()
    assert x.numel() > 1 << 31
    r = int8.quantize_rows(x)
    back = int8.restore_rows(r, torch.bfloat16)
    for at in ENDS:
        q, s = _codes(x[at])
        assert torch.equal(r.codes[at, :601], q) and torch.equal(r.scale[at], s)
        assert torch.equal(back[at], (q.float() * s[:, None]).bfloat16())


def test_linear_past_32_bits():
    from npa_amd import int8
    x = torch.randn((1 << 21) + 5, 40, device="cuda", generator=_gen(1)).half()
    w = int8.quantize_rows(torch.randn(1030, 40, device="cuda", generator=_gen(2)), align=16)
    y = int8.linear(x, w)
    assert y.numel() > 1 << 31
    for at in ENDS:
        assert torch.equal(y[at], _layer(*_codes(x[at]), w, None).half())


def test_weight_grad_past_32_bits():
    from npa_amd import int8
    rows = (1 << 21) + 64
    x = torch.randn(rows, 20, device="cuda", generator=_gen(3))
    dy = torch.randn(rows, 1030, device="cuda", generator=_gen(4))
    assert dy.numel() > 1 << 31
    dw, db = int8.weight_grad(int8.quantize_rows(x), dy)
    halves = [int8.weight_grad(int8.quantize_rows(x[at]), dy[at])
              for at in (slice(0, 1 << 20), slice(1 << 20, None))]
    assert ((dw - halves[0][0] - halves[1][0]).norm() <= 2e-6 * dw.norm()).item()
    assert ((db - halves[0][1] - halves[1][1]).norm() <= 2e-6 * db.norm()).item()


def test_mlp_past_32_bits():
    from npa_amd import int8
    from npa_amd import mlp as M
    rows = (1 << 22) + 33
    net, g = _net(163, 35, True, 5)
    z = torch.randn(rows, 163, device="cuda", generator=g)
    up = torch.randn(rows, 35, device="cuda", generator=g)
    assert z.numel() * 4 > 1 << 31
    w1, w2 = (int8.quantize_rows(m.weight, align=16) for m in (net[0], net[2]))
    b1, b2 = net[0].bias.detach(), net[2].bias.detach()
    with torch.no_grad():
        served = int8.mlp(z, w1, b1, w2, b2)
    z.requires_grad_(True)
    y = M.mlp(net, z, checkpoint="int8")
    (dz,) = torch.autograd.grad(y, z, up)
    d1, c1, d2 = (t.detach().double() for t in (net[0].weight, net[0].bias, net[2].weight))
    for at in ENDS:
        zr = z.detach()[at]
        assert torch.equal(served[at], _mlp_ref(zr, w1, b1, w2, b2))
        with torch.no_grad():
            assert torch.allclose(y[at], net(zr), rtol=1e-5, atol=1e-5)
        a = _kept(zr) @ d1.T + c1
        clear = ~(a.abs() < 1e-5).any(1)
        ref = ((up[at].double() @ d2) * (a > 0)) @ d1
        assert torch.all(((dz[at].double() - ref).abs() <= 1e-5 * ref.abs().max())[clear])
