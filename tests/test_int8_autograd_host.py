"""What npa_amd.int8.checkpoint differentiates, without a GPU: the two calls that
put rows into 8 bits and back are replaced by ones that keep the rows as they
are, so gradients equal those of the function itself."""
import pytest
import torch

from npa_amd import int8


@pytest.fixture(autouse=True)
def rows_as_they_are(monkeypatch):
    monkeypatch.setattr(int8, "_check_rows", lambda x, what: None)
    monkeypatch.setattr(int8, "quantize_rows",
                        lambda x: int8.Rows8(x.detach().clone(), torch.ones(1), tuple(x.shape)))
    monkeypatch.setattr(int8, "restore_rows", lambda r, dtype: r.codes.clone())


def _block(seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(6, 6), torch.nn.Tanh(), torch.nn.Linear(6, 6, bias=False))


@pytest.mark.parametrize("needs_x", [True, False])
def test_a_modules_parameters_get_their_gradients(needs_x):
    net = _block()
    for function in (net, net.forward):
        x = torch.randn(5, 6).requires_grad_(needs_x)
        net.zero_grad()
        int8.checkpoint(function, x).square().sum().backward()
        ref = torch.autograd.grad(net(x).square().sum(), list(net.parameters()) + ([x] if needs_x else []))
        for got, want in zip([p.grad for p in net.parameters()] + ([x.grad] if needs_x else []), ref):
            assert torch.allclose(got, want, rtol=1e-6, atol=0)


def test_blocks_in_a_row_all_learn():
    blocks = [_block(i) for i in range(3)]
    x = torch.randn(5, 6)
    v = x
    for b in blocks:
        v = int8.checkpoint(b, v)
    v.sum().backward()
    assert all(p.grad is not None and p.grad.any() for b in blocks for p in b.parameters())


def test_frozen_parameters_and_given_ones():
    net = _block()
    net[0].weight.requires_grad_(False)
    x, w = torch.randn(5, 6).requires_grad_(True), torch.randn(6, 6).requires_grad_(True)
    int8.checkpoint(net, x).sum().backward()
    assert net[0].weight.grad is None and net[0].bias.grad is not None

    y = int8.checkpoint(net, x).sum()
    net[2].weight.requires_grad_(False)  # between forward and backward
    net.zero_grad()
    y.backward()
    assert net[2].weight.grad is None and net[0].bias.grad is not None

    class Scaled(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.gain = torch.nn.Parameter(torch.tensor(2.0))

        def forward(self, v, m):
            return self.gain * (v @ m)

    scaled = Scaled()
    int8.checkpoint(scaled, x, w).sum().backward()
    ref = torch.autograd.grad((2.0 * (x @ w)).sum(), w)[0]
    assert torch.allclose(w.grad, ref) and scaled.gain.grad is not None


@pytest.mark.parametrize("needs_x", [True, False])
def test_gradients_of_captured_tensors_are_not_lost_silently(needs_x):
    """A tensor that the function reads besides its arguments, leaf or not: the call raises where its gradient would be lost."""
    net, w = _block(), torch.randn(6, 6).requires_grad_(True)
    made = w * 2
    for function in (lambda v: net(v), lambda v: v @ w, lambda v: v @ made):
        x = torch.randn(5, 6).requires_grad_(needs_x)
        y = int8.checkpoint(function, x)
        if needs_x:
            with pytest.raises(RuntimeError, match="int8.checkpoint"):
                y.sum().backward()
        else:  # nothing is kept: the function ran as it is
            y.sum().backward(retain_graph=True)
    assert w.grad is None or not needs_x
    fixed = torch.randn(6, 6)
    x = torch.randn(5, 6).requires_grad_(True)
    int8.checkpoint(lambda v: v @ fixed, x).sum().backward()
    assert torch.allclose(x.grad, torch.ones(5, 6) @ fixed.T)


def test_second_derivatives_are_refused():
    """A gradient penalty beside another loss raises instead of losing its terms, also where the upstream is a constant."""
    net, x = _block(), torch.randn(5, 6).requires_grad_(True)
    for upstream in (lambda y: y.sum(), lambda y: y.square().sum()):
        (dx,) = torch.autograd.grad(upstream(int8.checkpoint(net, x)), x, create_graph=True)
        with pytest.raises(RuntimeError, match="no second derivative"):
            (dx.square().sum() + net(x).sum()).backward()
    # the first derivative alone is as ever
    got = torch.autograd.grad(int8.checkpoint(net, x).sum(), list(net.parameters()), create_graph=True)
    for a, b in zip(got, torch.autograd.grad(net(x).sum(), list(net.parameters()))):
        assert torch.allclose(a, b)
