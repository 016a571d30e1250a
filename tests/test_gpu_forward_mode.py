"""Operators without a forward-mode derivative refuse tensors that hold tangents:
the results would have none."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def _calls():
    """Name, the call, its tensors."""
    from npa_amd import experts as E
    from npa_amd import norm
    randn = lambda *s: torch.randn(*s, dtype=torch.float32, device="cuda")
    r = E.sort_rows(torch.tensor([[0, 2], [1, 1], [2, -1], [0, 0]], device="cuda"), 3)
    mlp = [randn(8, 6), randn(3, 128, 6), randn(3, 128), randn(3, 5, 128), randn(3, 5)]
    small = [randn(8, 6), randn(3, 10, 6), None, randn(3, 5, 10), None]
    return [("layer_norm", lambda *t: norm.layer_norm(*t), [randn(4, 6), randn(6), randn(6)]),
            ("dispatch", lambda x: E.dispatch(x, r), [randn(4, 6)]),
            ("combine", lambda results, weight: E.combine(results, weight, r), [randn(8, 6), torch.rand(4, 2, device="cuda")]),
            ("linear", lambda *t: E.linear(*t, r.offsets), [randn(8, 6), randn(3, 5, 6), randn(3, 5)]),
            ("mlp of 128", lambda *t: E.mlp(*t, r.offsets), mlp), ("mlp", lambda *t: E.mlp(*t, r.offsets), small)]


@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(grad):
    for name, call, tensors in _calls():
        want = call(*tensors)
        for i, t in enumerate(tensors):
            if t is None:
                continue
            with torch.set_grad_enabled(grad), forward_ad.dual_level():
                dual = [forward_ad.make_dual(u, torch.ones_like(u)) if j == i else u for j, u in enumerate(tensors)]
                with pytest.raises(RuntimeError, match="forward AD|forward-mode|jvp"):
                    call(*dual)
                    pytest.fail(f"{name} lost the tangent of its tensor {i}")
                assert torch.equal(call(*tensors), want)  # none of these holds one


def test_integer_layers_refuse_tangents():
    from npa_amd import int8
    w = [int8.quantize_rows(torch.randn(*s, device="cuda"), align=16) for s in ((128, 20), (8, 128))]
    z = torch.randn(10, 20, device="cuda")
    for call in (lambda t: int8.linear(t, w[0]), lambda t: int8.mlp(t, w[0], None, w[1], None)):
        want = call(z)
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(forward_ad.make_dual(z, z))
            assert torch.equal(call(z), want)


def test_transforms_are_refused():
    for _, call, tensors in _calls():
        first, rest = tensors[0], tensors[1:]
        with pytest.raises(RuntimeError):
            torch.func.jvp(lambda x: call(x, *rest), (first,), (torch.ones_like(first),))
