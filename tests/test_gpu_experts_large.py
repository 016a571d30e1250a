"""Layers of experts whose rows or weights pass 2^31 values and more: first and last
rows against float64.  Bounds as everywhere: a float32 sum of n products is within
(n + 8) 2 u of the sum of their absolute values, u = 2^-24, and rounded once more."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF16 = torch.bfloat16


def _within(name, got, ref, size, n):
    limit = (n + 8) * 2 * U * size * (1 + 2.0 ** -8) + 2.0 ** -8 * ref.abs() + torch.finfo(got.dtype).tiny
    err = (got.double() - ref).abs()
    assert (err <= limit).all(), f"{name}: {(err / limit).nan_to_num(1e30).max().item():.3g} bounds off"


def test_results_past_36_billion_values():
    """Nine million rows of 4096 outputs."""
    from npa_amd import experts as E
    g = torch.Generator(device="cuda").manual_seed(0)
    rows, cols, outs = 9_000_003, 8, 4096
    x = torch.randn(rows, cols, device="cuda", generator=g, dtype=BF16)
    w = torch.randn(2, outs, cols, device="cuda", generator=g, dtype=BF16)
    half = rows // 2
    offsets = torch.tensor([0, half, rows - 5], dtype=torch.int32, device="cuda")
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = E.linear(x, w, None, offsets)
    xd, wd = x.detach().double(), w.detach().double()
    for at, e in ((slice(0, 300), 0), (slice(half - 300, half), 0), (slice(half, half + 300), 1), (slice(-305, -5), 1)):
        _within("y", y.detach()[at], xd[at] @ wd[e].T, xd[at].abs() @ wd[e].abs().T, cols)
    assert not y[-5:].any()
    up = torch.randn(1, outs, device="cuda", generator=g, dtype=BF16)
    dx, dw = torch.autograd.grad(y, [x, w], up.expand(rows, outs))
    ud = up.double()
    for at, e in ((slice(0, 300), 0), (slice(-305, -5), 1)):
        ref = (ud @ wd[e]).expand(300, cols)
        _within("dx", dx[at], ref, (ud.abs() @ wd[e].abs()).expand(300, cols), outs)
    for at, e in ((slice(0, half), 0), (slice(half, rows - 5), 1)):
        _within("dW", dw[e], ud.T * xd[at].sum(0), ud.T.abs() * xd[at].abs().sum(0), half)


@pytest.mark.parametrize("cols", [8192, 8191])
@pytest.mark.parametrize("slots", [200, 1500])
def test_weights_past_32_bits(slots, cols):
    """40 experts of 8192 outputs: weights and their gradients are 2.7e9 values."""
    from npa_amd import experts as E
    g = torch.Generator(device="cuda").manual_seed(1)
    n, outs = 40, 8192
    w = torch.randn(n, outs, cols, device="cuda", generator=g, dtype=BF16)
    assert w.numel() > 1 << 31
    x = torch.randn(slots, cols, device="cuda", generator=g, dtype=BF16)
    first = slots // 4
    at = [0, *[first] * (n - 2), first + 7, slots - 3]  # the first expert, the last two
    offsets = torch.tensor(at, dtype=torch.int32, device="cuda")
    x.requires_grad_(True)
    w.requires_grad_(True)
    dy = torch.randn(slots, outs, device="cuda", generator=g, dtype=BF16)
    y = E.linear(x, w, None, offsets)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    for e in (0, 1, n - 2, n - 1):
        s = slice(at[e], at[e + 1])
        xd, ud, wd = x.detach()[s].double(), dy[s].double(), w.detach()[e].double()
        _within("y", y.detach()[s], xd @ wd.T, xd.abs() @ wd.abs().T, cols)
        _within("dx", dx[s], ud @ wd, ud.abs() @ wd.abs(), outs)
        _within("dW", dw[e], ud.T @ xd, ud.abs().T @ xd.abs(), at[e + 1] - at[e])
    assert not y[-3:].any() and not dx[-3:].any()
