"""ExpertMlp under autocast, where a layer before it gives 16-bit rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hidden", [128, 48])
def test_experts_between_layers(hidden, kind):
    from npa_amd import experts as E
    torch.manual_seed(0)
    first, last = torch.nn.Linear(12, 20, device="cuda"), torch.nn.Linear(8, 3, device="cuda")
    mix = E.ExpertMlp(20, hidden, 8, 4, 2, device="cuda")
    x, up = torch.randn(5, 30, 12, device="cuda"), torch.randn(5, 30, 3, device="cuda")
    params = [*first.parameters(), *mix.parameters(), *last.parameters()]

    def parts(h):
        """The module from its pieces: the router as autocast runs it, the experts in float32."""
        assert h.dtype == kind
        weight, index = torch.softmax(torch.nn.functional.linear(h, mix.router.weight, mix.router.bias).float(),
                                      -1).topk(2, dim=-1)
        r = E.sort_rows(index, 4)
        return E.combine(E.mlp(E.dispatch(h.float(), r), mix.w1, mix.b1, mix.w2, mix.b2, r.offsets), weight, r)

    out = []
    for middle in (mix, parts):
        with torch.autocast("cuda", kind):
            y = last(middle(first(x)))
        assert y.dtype == kind
        out.append([y.detach(), *torch.autograd.grad((y.float() * up).sum(), params)])
    for p, q in zip(*out):
        assert torch.isfinite(p).all() and torch.equal(p, q)


def test_float32_rows_train_under_autocast():
    from npa_amd import experts as E
    torch.manual_seed(0)
    mix = E.ExpertMlp(20, 48, 8, 4, 1, device="cuda")
    x = torch.randn(40, 20, device="cuda", requires_grad=True)
    with torch.autocast("cuda", torch.bfloat16):
        y = mix(x)
    assert y.dtype == torch.float32
    for g in torch.autograd.grad(y.square().sum(), [x, *mix.parameters()]):
        assert torch.isfinite(g).all()


def test_other_types_are_refused_without_autocast():
    from npa_amd import experts as E
    mix = E.ExpertMlp(20, 48, 8, 4, 1, device="cuda")
    for kind in (torch.bfloat16, torch.float64):
        with pytest.raises((TypeError, RuntimeError)):
            mix(torch.randn(40, 20, device="cuda").to(kind))
