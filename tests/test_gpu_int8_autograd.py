"""Gradients of functions and layers that keep rows in 8 bits, as autograd sees them."""
import pytest
import torch

from test_gpu_int8 import _gen

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
