"""npa_amd.int8 without a GPU: refusals of tensors that are not on one, and the C
entry points' own checks, which come before anything is launched."""
import ctypes

import pytest
import torch

from npa_amd import int8
from npa_amd import mlp as M
from npa_amd.sphops import _native

lib = _native.lib


def test_host_tensors_are_refused():
    x = torch.randn(4, 8)
    saved = int8.Rows8(torch.zeros(4, 8, dtype=torch.int8), torch.ones(4), (4, 8))
    for call in (lambda: int8.quantize_rows(x), lambda: int8.restore_rows(saved), lambda: int8.weight_grad(saved, x),
                 lambda: int8.linear(x, saved), lambda: int8.mlp(x, saved, None, saved, None),
                 lambda: int8.checkpoint(torch.tanh, x), lambda: int8.Int8Linear(torch.nn.Linear(4, 4))):
        with pytest.raises(TypeError):
            call()


def test_unknown_checkpoint_is_refused():
    with pytest.raises(ValueError):
        M.mlp(torch.nn.Linear(4, 4), torch.randn(2, 4), checkpoint="fp8")


def _fails(status, text):
    assert status == -1
    assert text in lib.sphops_last_error().decode()


def test_entry_points_check_their_arguments():
    p = ctypes.c_void_p(4096)  # never read: every call fails before a launch
    odd = ctypes.c_void_p(4098)
    _fails(lib.sphops_quantize_rows(p, 3, 8, p, 8, p, 1, 8, 0, None), "element type")
    _fails(lib.sphops_quantize_rows(p, 0, 8, p, 6, p, 1, 8, 0, None), "ld")
    _fails(lib.sphops_quantize_rows(p, 0, 9, p, 10, p, 1, 9, 0, None), "ld")
    _fails(lib.sphops_quantize_rows(p, 0, 0, p, 4, p, 1, 0, 0, None), "values")
    _fails(lib.sphops_quantize_rows(p, 0, 65537, p, 65540, p, 1, 65537, 0, None), "values")
    _fails(lib.sphops_quantize_rows(p, 0, 8, p, 8, p, -1, 8, 0, None), "rows")
    _fails(lib.sphops_quantize_rows(p, 0, 8, odd, 8, p, 1, 8, 0, None), "aligned")
    _fails(lib.sphops_quantize_rows(None, 0, 8, p, 8, p, 1, 8, 0, None), "null")
    _fails(lib.sphops_restore_rows(p, 8, p, None, 0, 1, 8, None), "null")
    _fails(lib.sphops_rows8_weight_grad(p, 8, p, p, None, None, 1, 8, 8, p, None), "null")
    _fails(lib.sphops_rows8_weight_grad(p, 8, p, p, p, None, 1, 8, 0, p, None), "not supported")
    _fails(lib.sphops_linear8(p, 0, 8, p, 24, p, None, p, 1, 8, 8, p, None), "multiple of 16")
    _fails(lib.sphops_linear8(p, 0, 8, ctypes.c_void_p(4100), 16, p, None, p, 1, 8, 8, p, None), "16-byte")
    _fails(lib.sphops_linear8(p, 0, 8, p, 16, p, None, p, 1, 8, 0, p, None), "not supported")
    _fails(lib.sphops_mlp8_forward(p, p, 16, p, None, p, 128, p, None, p, 1, 8, 64, 8, None), "not supported")
    _fails(lib.sphops_mlp8_forward(p, p, 16, p, None, p, 112, p, None, p, 1, 8, 128, 8, None), "multiple of 16")
    _fails(lib.sphops_mlp_rows8_forward(p, p, None, p, None, p, 32, p, p, 1, 8, 128, 8, None), "rounded up")
    _fails(lib.sphops_mlp_rows8_backward(p, 8, p, p, p, None, p, p, None, None, None, None, 1, 200, 128, 8, p, None),
           "not supported")
    assert lib.sphops_linear8_workspace_bytes(1, 0, 4) == -1
    assert lib.sphops_rows8_weight_grad_workspace_bytes(-1, 4, 4) == -1
    assert lib.sphops_mlp_rows8_workspace_bytes(1, 8, 64, 8) == -1


def test_weight_gradient_chunks_are_bounded():
    """No chunk of a weight gradient, each one chain of sums in 32 bits, is
    longer than 8192 rows: the workspace holds a partial sum per chunk."""
    for nin, nout in ((4, 4), (83, 19), (163, 35), (300, 700)):
        for rows in (1, 65, 1 << 20, (1 << 25) + 1):
            partial = 4 * (nin * nout + nout)
            size = lib.sphops_rows8_weight_grad_workspace_bytes(rows, nin, nout)
            assert size % partial == 0 and size // partial >= -(-rows // 8192)
            if nin <= 168 and nout <= 64:
                partial = 4 * (128 * nin + 128 + 128 * nout + nout)
                size = lib.sphops_mlp_rows8_workspace_bytes(rows, nin, 128, nout)
                assert size % partial == 0 and size // partial >= -(-rows // 8192)
