"""float32 tensors give the same results whatever torch's default type is."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _randn(g, *shape):
    return torch.randn(*shape, dtype=torch.float32, device="cuda", generator=g)


def _norm(g):
    from npa_amd import norm
    leaves = [_randn(g, 70, 83), _randn(g, 83), _randn(g, 83)]
    return leaves, lambda x, w, b: norm.layer_norm(x, w, b)


def _combine(g):
    from npa_amd import experts as E
    r = E.sort_rows(torch.randint(-1, 4, (50, 2), device="cuda", generator=g), 4)
    return [_randn(g, 100, 40), _randn(g, 50, 2)], lambda results, weight: E.combine(results, weight, r)


def _experts(hidden):
    def make(g):
        from npa_amd import experts as E
        offsets = torch.tensor([0, 30, 30, 77], dtype=torch.int32, device="cuda")
        leaves = [_randn(g, 80, 66), _randn(g, 3, hidden, 66), _randn(g, 3, hidden), _randn(g, 3, 18, hidden),
                  _randn(g, 3, 18)]
        return leaves, lambda *t: E.mlp(*t, offsets)
    return make


def _layers(checkpoint):
    def make(g):
        from npa_amd import mlp
        layers = torch.nn.Sequential(torch.nn.Linear(40, 128), torch.nn.ReLU(), torch.nn.Linear(128, 70),
                                     torch.nn.ReLU(), torch.nn.Linear(70, 9)).to("cuda", torch.float32)
        with torch.no_grad():
            for p in layers.parameters():
                p.copy_(0.1 * _randn(g, *p.shape))
        return [_randn(g, 60, 40), *layers.parameters()], lambda z, *_: mlp.mlp(layers, z, checkpoint)
    return make


def _mlp_rows(g):
    from npa_amd import mlp
    layers = torch.nn.Sequential(torch.nn.Linear(40, 128), torch.nn.ReLU(), torch.nn.Linear(128, 9)).to("cuda", torch.float32)
    with torch.no_grad():
        for p in layers.parameters():
            p.copy_(0.1 * _randn(g, *p.shape))
    return [_randn(g, 60, 40), *layers.parameters()], lambda z, *_: mlp.mlp(layers, z)


def _module(g):
    from npa_amd import experts as E
    mix = E.ExpertMlp(20, 128, 8, 3, 2, device="cuda", dtype=torch.float32)
    with torch.no_grad():
        for p in mix.parameters():
            p.copy_(_randn(g, *p.shape))
    return [_randn(g, 90, 20), *mix.parameters()], lambda x, *_: mix(x)


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64])
@pytest.mark.parametrize("make", [_norm, _combine, _experts(128), _experts(36), _layers(None), _mlp_rows, _module])
def test_results_do_not_depend_on_the_default_type(make, default):
    def run():
        g = torch.Generator(device="cuda").manual_seed(7)
        leaves, f = make(g)
        leaves = [t.requires_grad_(True) for t in leaves]
        y = f(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, _randn(g, *y.shape))]

    want = run()
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        got = run()
    finally:
        torch.set_default_dtype(before)
    for p, q in zip(got, want):
        assert p.dtype == torch.float32 and torch.equal(p, q)
