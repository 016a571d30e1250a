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


def _int8(g):
    from npa_amd import int8
    w = int8.quantize_rows(_randn(g, 30, 83), align=16)
    dy = _randn(g, 70, 12)

    def run(x):
        r = int8.quantize_rows(x)
        assert r.scale.dtype == torch.float32
        with torch.no_grad():
            out = [int8.linear(x, w), *int8.weight_grad(r, dy), r.codes.float(), r.scale]
        return torch.cat([t.flatten() for t in out]) + int8.restore_rows(r).sum() + 0 * x.sum()

    return [_randn(g, 70, 83)], run


def _step(dim):
    """A step of an automaton, perception and splatted image with it."""
    def make(g):
        import types

        import npa_amd.sphops as sp
        from npa_amd.splatting import splat_particles_batch
        from npa_amd.step import step_euler
        C, N = 8, 400
        cols = 2 * C + dim * C + dim
        rule = torch.nn.Sequential(torch.nn.Linear(cols, 128), torch.nn.ReLU(), torch.nn.Linear(128, dim + C))
        rule = rule.to("cuda", torch.float32)
        with torch.no_grad():
            for p in rule.parameters():
                p.copy_(0.1 * _randn(g, *p.shape))
        model = types.SimpleNamespace(spatial_dims=dim, eps0=0.1, alpha=0.5, model=rule, state_grad=True,
                                      density_grad=True, log_norm_grad=True, log_norm_density_grad=True,
                                      stopgrad_pos=False, stopgrad_state=False)
        x = 1.2 * torch.rand(1, N, dim, dtype=torch.float32, device="cuda", generator=g) - 0.6

        def run(s, *_):
            grid = sp.HashGrid(dim=dim, boundary="periodic", mode="grid", grid_size=[16] * dim, eps=0.1, num_particles=N,
                               batch_size=1, max_particles_per_block=64)
            at = grid.wrap_positions(x)
            at = torch.cat([at, torch.zeros_like(at[..., :1])], -1) if dim == 3 else at  # rows of 4 in 3D
            xs, ss, _ = step_euler(model, at, s, grid, update_prob=1.0)
            out = [xs.flatten(), ss.flatten()]
            if dim == 2:
                out.append(splat_particles_batch(xs, ss.sigmoid(), img_size=32).flatten())
            return torch.cat(out)

        return [_randn(g, 1, N, C), *rule.parameters()], run
    return make


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64])
@pytest.mark.parametrize("make", [_norm, _combine, _experts(128), _experts(36), _layers(None), _mlp_rows, _module,
                                  _layers("int8"), _int8, _step(2), _step(3)])
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
