"""npa_amd.mlp.mlp under autocast: the layers' own 16-bit products, trained too."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes", [(40, 96, 70, 9), (40, 128, 18), (33, 50), (20, 30, 100)])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_layers_under_autocast(sizes, kind, checkpoint):
    from npa_amd import mlp
    torch.manual_seed(0)
    layers = []
    for i, o in zip(sizes[:-1], sizes[1:]):
        layers += [torch.nn.Linear(i, o), torch.nn.ReLU()]
    module = torch.nn.Sequential(*layers[:-1]).cuda()
    z, up = torch.randn(90, sizes[0], device="cuda"), torch.randn(90, sizes[-1], device="cuda")
    leaves = [z.requires_grad_(True), *module.parameters()]
    out = []
    for run in (lambda t: mlp.mlp(module, t, checkpoint), module):
        with torch.autocast("cuda", kind):
            y = run(z)
        assert y.dtype == kind
        out.append([y.detach(), *torch.autograd.grad((y.float() * up).sum(), leaves)])
    for p, q in zip(*out):
        assert torch.equal(p, q)


def test_relu_and_layer_in_one_kernel_stay_float32():
    from npa_amd import mlp
    torch.manual_seed(0)
    module = torch.nn.Sequential(torch.nn.ReLU(), torch.nn.Linear(64, 18)).cuda()
    a = torch.randn(90, 64, device="cuda", requires_grad=True)
    want = mlp.mlp(module, a)
    with torch.autocast("cuda", torch.bfloat16):
        y = mlp.mlp(module, a)
    assert torch.equal(y, want)
    grads = torch.autograd.grad(y.square().sum(), [a, *module.parameters()])
    assert all(torch.equal(p, q) for p, q in zip(grads, torch.autograd.grad(want.square().sum(), [a, *module.parameters()])))
