"""Gradients of functions and layers that keep rows in 8 bits, as autograd sees them."""
import pytest
import torch

from test_gpu_int8 import _gen, _net

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("needs_x", [True, False])
def test_checkpoint_of_a_module(needs_x):
    from npa_amd import int8
    g = _gen(1)
    net = torch.nn.Sequential(torch.nn.Linear(40, 24), torch.nn.Tanh()).cuda()
    x = torch.randn(70, 40, device="cuda", generator=g).requires_grad_(needs_x)
    up = torch.randn(70, 24, device="cuda", generator=g)
    int8.checkpoint(net, x).backward(up)
    kept = int8.restore_rows(int8.quantize_rows(x)).requires_grad_(True)
    want = torch.autograd.grad(net(kept), [*net.parameters(), kept], up)
    for p, ref in zip(net.parameters(), want):
        assert torch.equal(p.grad, ref)
    assert torch.equal(x.grad, want[-1]) if needs_x else x.grad is None


@pytest.mark.parametrize("hidden,nout", [(128, 19), (64, 19), (256, 130)])
def test_second_derivatives_are_right_or_refused(hidden, nout):
    """Of layers with codes only dx is differentiated again, which is linear in the
    upstream and the weights; the fused MLP's gradients and weight gradients raise."""
    from npa_amd import mlp as M
    net, g = _net(83, nout, True, hidden, hidden)
    x = torch.randn(300, 83, device="cuda", generator=g).requires_grad_(True)

    def penalty(y):
        (dx,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        return dx.square().sum()

    y = M.mlp(net, x, checkpoint="int8")
    if hidden == 128:
        with pytest.raises(RuntimeError, match="no second derivative"):
            (penalty(y) + net(x).sum()).backward()
    else:  # each value of the saved rows is within 1/254 of its row's largest
        got = torch.autograd.grad(penalty(y), list(net.parameters()))
        for a, b in zip(got, torch.autograd.grad(penalty(net(x)), list(net.parameters()))):
            assert ((a - b).norm() <= 0.02 * b.norm()).item()
    y = M.mlp(net, x, checkpoint="int8")
    dw = torch.autograd.grad(y.sum(), net[0].weight, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="no second derivative"):
        dw.square().sum().backward()
    first, again = (torch.autograd.grad(M.mlp(net, x, checkpoint="int8").sum(), list(net.parameters()), create_graph=c)
                    for c in (True, False))
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("hidden,nout", [(128, 19), (64, 19), (256, 130)])
def test_second_derivatives_without_a_checkpoint(hidden, nout):
    """The same of the float32 layers: a Linear's dx is differentiated again, what a kernel computes raises."""
    from npa_amd import mlp as M
    net, g = _net(83, nout, True, hidden, hidden)
    x = torch.randn(300, 83, device="cuda", generator=g).requires_grad_(True)

    def penalty(y):
        (dx,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        return dx.square().sum()

    if nout <= 64:
        with pytest.raises(RuntimeError, match="no second derivative"):
            (penalty(M.mlp(net, x)) + net(x).sum()).backward()
    else:
        got = torch.autograd.grad(penalty(M.mlp(net, x)), list(net.parameters()))
        for a, b in zip(got, torch.autograd.grad(penalty(net(x)), list(net.parameters()))):
            assert ((a - b).norm() <= 1e-5 * b.norm()).item()
    dw = torch.autograd.grad(M.mlp(net, x).sum(), net[0].weight, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="no second derivative"):
        dw.square().sum().backward()
    first, again = (torch.autograd.grad(M.mlp(net, x).sum(), list(net.parameters()), create_graph=c)
                    for c in (True, False))
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_widths_that_no_codes_are_kept_of():
    """Rows past the widest that is kept run as they do without a checkpoint."""
    from npa_amd import mlp as M
    layer = torch.nn.Linear(70000, 65).cuda().requires_grad_(False)
    a = torch.randn(3, 70000, device="cuda", generator=_gen(2)).requires_grad_(True)
    grads = []
    for mode in (None, "int8"):
        for net in (layer, torch.nn.Sequential(torch.nn.ReLU(), layer)):
            y = M.mlp(net, a, checkpoint=mode)
            grads.append((y.detach(), *torch.autograd.grad(y, a, torch.ones_like(y))))
    assert all(torch.equal(p, q) for i in (0, 1) for p, q in zip(grads[i], grads[i + 2]))
    with pytest.raises(RuntimeError):  # the layer's own weight gradient ends at 32768 features, with and without
        M.mlp(layer.requires_grad_(True), a).sum().backward()
    with pytest.raises(RuntimeError):
        M.mlp(layer, a, checkpoint="int8").sum().backward()
