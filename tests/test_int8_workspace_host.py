"""The 8-bit entry points' check of their workspace, which comes before anything is launched."""
import ctypes

from npa_amd.sphops import _native

lib = _native.lib


def test_workspaces_that_are_not_aligned_are_refused():
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4100)  # never read: every call fails before a launch
    calls = {"weight gradient": lambda w: lib.sphops_rows8_weight_grad(p, 8, p, p, p, None, 1, 8, 8, w, None),
             "integer layer": lambda w: lib.sphops_linear8(p, 0, 8, p, 16, p, None, p, 1, 8, 8, w, None),
             "MLP": lambda w: lib.sphops_mlp_rows8_backward(p, 8, p, p, p, None, p, p, None, None, None, None, 1, 8, 128,
                                                            8, w, None)}
    for name, call in calls.items():
        assert call(odd) == -1, name
        assert "workspace must be 16-byte aligned" in lib.sphops_last_error().decode(), name
        assert call(None) == -1, name
        assert "null buffer" in lib.sphops_last_error().decode(), name
