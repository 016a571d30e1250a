"""Buffers that kernels write float32 into are float32 whatever torch's default
type is: every allocation of the package names its type."""
import ast
import os

import pytest
import torch

import npa_amd
from npa_amd import experts as E
from npa_amd import norm

ROOT = os.path.dirname(npa_amd.__file__)


@pytest.fixture(params=[torch.bfloat16, torch.float64])
def other_default(request):
    before = torch.get_default_dtype()
    torch.set_default_dtype(request.param)
    yield
    torch.set_default_dtype(before)


@pytest.mark.parametrize("module", ["norm.py", "experts.py", "mlp.py", "int8.py", "step.py", "perceive.py",
                                    "splatting.py", "sphops/sph.py", "sphops/sph_hip.py"])
def test_allocations_name_their_type(module):
    with open(os.path.join(ROOT, module)) as f:
        tree = ast.parse(f.read())
    for node in ast.walk(tree):
        if (isinstance(node, ast.Call) and isinstance(node.func, ast.Attribute)
                and getattr(node.func.value, "id", None) == "torch"
                and node.func.attr in ("empty", "zeros", "ones", "full", "tensor")):
            names = [k.arg for k in node.keywords]
            assert "dtype" in names or None in names, f"{module}:{node.lineno}"  # None: **kwargs


def test_buffers_of_norm_and_experts(other_default, monkeypatch):
    """What the entry points are given, with the library's calls left out."""
    types, empty = [], torch.empty

    def recorded(*args, **kwargs):
        types.append(empty(*args, **kwargs).dtype)
        return empty(*args, **kwargs)

    monkeypatch.setattr(E._rows, "call", lambda *args: None)
    monkeypatch.setattr(torch, "empty", recorded)
    f32 = dict(dtype=torch.float32)
    x, w = torch.zeros(6, 8, **f32).requires_grad_(True), torch.ones(8, **f32).requires_grad_(True)
    norm._LayerNorm.apply(x, w, w, 1e-5).backward(torch.zeros(6, 8, **f32))
    slot = torch.zeros(6, 1, dtype=torch.int32)
    weight = torch.ones(6, 1, **f32).requires_grad_(True)
    E._Combine.apply(x, weight, slot, slot.flatten()).backward(torch.zeros(6, 8, **f32))
    params = [torch.ones(*s, **f32).requires_grad_(True) for s in ((2, 128, 8), (2, 128), (2, 4, 128), (2, 4))]
    offsets = torch.tensor([0, 3, 6], dtype=torch.int32)
    E._FusedMlp.apply(x, *params, offsets).backward(torch.zeros(6, 4, **f32))
    E._Mlp.apply(x, *params, offsets).backward(torch.zeros(6, 4, **f32))
    # stats, results, gradients, the mask's words and workspaces' bytes
    assert set(types) == {torch.float32, torch.int32, torch.uint8}
