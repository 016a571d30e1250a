"""npa_amd.norm and npa_amd.experts without a GPU: refusals of tensors that are
not on one, and the C entry points' own checks, which come before a launch."""
import ctypes

import pytest
import torch

from npa_amd import experts as E
from npa_amd import norm
from npa_amd.sphops import _native

lib = _native.lib


def test_host_tensors_are_refused():
    x, w = torch.randn(4, 8), torch.randn(2, 3, 8)
    index, offsets = torch.zeros(4, 1, dtype=torch.int32), torch.tensor([0, 2, 4], dtype=torch.int32)
    routing = E.Routing(offsets, index, index.flatten())
    for call in (lambda: norm.layer_norm(x), lambda: norm.LayerNorm(8)(x), lambda: E.sort_rows(index, 2),
                 lambda: E.dispatch(x, routing), lambda: E.combine(x, None, routing),
                 lambda: E.linear(x, w, None, offsets), lambda: E.mlp(x, w, None, w, None, offsets)):
        with pytest.raises(TypeError):
            call()


def test_modules_hold_what_torchs_hold():
    assert {k: v.shape for k, v in norm.LayerNorm(8).state_dict().items()} == {
        k: v.shape for k, v in torch.nn.LayerNorm(8).state_dict().items()}
    mix = E.ExpertMlp(6, 10, 4, 3, 2)
    assert [tuple(p.shape) for p in (mix.w1, mix.b1, mix.w2, mix.b2, mix.router.weight)] == [
        (3, 10, 6), (3, 10), (3, 4, 10), (3, 4), (3, 6)]
    assert mix.w1.abs().max() <= 6 ** -0.5 and mix.b2.abs().max() <= 10 ** -0.5
    for args in ((4, 8, 2, 3, 4), (4, 8, 2, 3, 0), (4, 8, 2, 1025, 1)):
        with pytest.raises(ValueError):
            E.ExpertMlp(*args)


def _fails(status, text):
    assert status == -1
    assert text in lib.sphops_last_error().decode()


def test_entry_points_check_their_arguments():
    p = ctypes.c_void_p(4096)  # never read: every call fails before a launch
    odd = ctypes.c_void_p(4097)
    _fails(lib.sphops_layer_norm(p, 3, 8, p, p, 1, p, p, 1, 8, 1e-5, None), "element type")
    _fails(lib.sphops_layer_norm(p, 0, 8, p, p, 1, p, p, 1, 0, 1e-5, None), "values")
    _fails(lib.sphops_layer_norm(p, 0, 8, p, p, 1, p, p, 1, 65537, 1e-5, None), "values")
    _fails(lib.sphops_layer_norm(p, 0, 8, p, p, 1, p, p, -1, 8, 1e-5, None), "rows")
    _fails(lib.sphops_layer_norm(p, 0, -8, p, p, 1, p, p, 2, 8, 1e-5, None), "row_stride")
    _fails(lib.sphops_layer_norm(None, 0, 8, p, p, 1, p, p, 1, 8, 1e-5, None), "null")
    _fails(lib.sphops_layer_norm(p, 1, 8, odd, p, 0, p, p, 1, 8, 1e-5, None), "aligned")
    _fails(lib.sphops_layer_norm(p, 0, 8, p, p, 1, p, ctypes.c_void_p(4100), 1, 8, 1e-5, None), "8-byte")
    _fails(lib.sphops_layer_norm_backward(p, 8, p, 8, 0, p, 1, None, p, p, p, 1, 8, p, None), "null")
    _fails(lib.sphops_layer_norm_backward(p, 8, p, -8, 0, p, 1, p, p, p, p, 2, 8, p, None), "strides")
    assert lib.sphops_layer_norm_workspace_bytes(0, -1, 8) == -1
    assert lib.sphops_layer_norm_workspace_bytes(3, 1, 8) == -1
    _fails(lib.sphops_sort_rows(p, 0, 4, 0, 3, p, p, p, p, None), "choices")
    _fails(lib.sphops_sort_rows(p, 0, 4, 65, 3, p, p, p, p, None), "choices")
    _fails(lib.sphops_sort_rows(p, 0, 1 << 30, 2, 3, p, p, p, p, None), "2^30")
    _fails(lib.sphops_sort_rows(p, 0, 4, 1, 1025, p, p, p, p, None), "experts")
    _fails(lib.sphops_sort_rows(p, 0, 4, 1, 3, None, p, p, p, None), "null")
    _fails(lib.sphops_sort_rows(p, 0, 1 << 20, 1, 3, p, p, p, None, None), "null")
    assert lib.sphops_sort_rows_workspace_bytes(1, 0, 3) == -1
    _fails(lib.sphops_dispatch_rows(p, 0, 8, p, None, None, 1, 1, 8, None), "null")
    _fails(lib.sphops_dispatch_rows(p, 0, 8, p, p, p, 1, 1, 0, None), "values")
    _fails(lib.sphops_combine_rows(p, 5, p, p, p, 1, 1, 8, None), "element type")
    _fails(lib.sphops_combine_rows(p, 0, p, None, p, 1, 1, 8, None), "null")
    _fails(lib.sphops_combine_rows_backward(p, 0, 8, None, p, p, p, p, p, 1, 1, 8, None), "null")
    _fails(lib.sphops_expert_linear(p, 0, 8, p, p, p, p, 4, 0, 8, 8, 0, p, None), "not supported")
    _fails(lib.sphops_expert_linear(p, 0, 8, p, p, p, p, 4, 2, 0, 8, 0, p, None), "not supported")
    _fails(lib.sphops_expert_linear(p, 0, 8, p, p, None, p, 4, 2, 8, 8, 0, p, None), "null")
    _fails(lib.sphops_expert_linear(p, 0, 8, p, p, p, p, 1 << 16, 2, 1024, 1024, 0, None, None), "null")
    _fails(lib.sphops_expert_linear(p, 0, 8, p, p, p, p, 4, 2, 8, 8, 0, ctypes.c_void_p(4100), None), "16-byte")
    _fails(lib.sphops_expert_linear_backward(p, 8, p, 0, 8, p, None, p, p, p, p, -4, 2, 8, 8, p, None), "not supported")
    _fails(lib.sphops_expert_linear_backward(p, 8, p, 0, 8, p, None, None, p, p, p, 4, 2, 8, 8, p, None), "null")
    _fails(lib.sphops_expert_linear_backward(p, 8, p, 0, 8, p, None, p, p, p, p, 4, 2, 8, 8, ctypes.c_void_p(4100), None),
           "16-byte")
    assert lib.sphops_expert_linear_workspace_bytes(0, 4, 1025, 8, 8) == -1
    assert lib.sphops_expert_linear_backward_workspace_bytes(3, 4, 2, 8, 8) == -1
    _fails(lib.sphops_expert_mlp_forward(p, p, p, p, p, p, p, p, 4, 2, 8, 64, 8, None), "not supported")
    _fails(lib.sphops_expert_mlp_forward(p, p, p, p, p, None, p, p, 4, 2, 8, 128, 8, None), "null")
    _fails(lib.sphops_expert_mlp_forward(p, p, p, p, p, p, p, ctypes.c_void_p(4100), 4, 2, 8, 128, 8, None), "8-byte")
    _fails(lib.sphops_expert_mlp_input_grad(p, p, p, None, p, p, 4, 2, 8, 128, 8, None), "null")
    _fails(lib.sphops_expert_mlp_weight_grad(p, p, p, p, p, p, p, p, p, p, 4, 2, 8, 128, 8, None, None), "null")
    assert lib.sphops_expert_mlp_workspace_bytes(4, 2, 8, 128, 65) == -1
    # no part of the rows' sums is longer than 8192 rows
    for rows in (1, 1 << 20, 1 << 27):
        partial = 4 * (128 * 83 + 128 + 19 * 128 + 19)
        size = lib.sphops_expert_mlp_workspace_bytes(rows, 3, 83, 128, 19)
        assert size % partial == 0 and size // partial - 3 >= rows // 8192
