"""Which layers of experts the library takes: all whose launches have fewer than 2^32
threads, counted for the kernels of the rows' type."""
import pytest

from npa_amd.sphops import _native

lib = _native.lib
F32, BF16, F16 = 0, 1, 2


def _takes(kind, slots, experts, cols, outs):
    forward = lib.sphops_expert_linear_workspace_bytes(kind, slots, experts, cols, outs) >= 0
    assert forward == (lib.sphops_expert_linear_backward_workspace_bytes(kind, slots, experts, cols, outs) >= 0)
    return forward


@pytest.mark.parametrize("kind,slots,experts,cols,outs", [
    (BF16, 9_000_000, 2, 8, 4096), (F16, 30_000_000, 8, 4096, 1024), (BF16, 120_000_000, 8, 1024, 1000),
    (F32, 60_000_000, 4, 1024, 4096), (F32, (1 << 30) - (1 << 18), 4, 128, 128), (BF16, (1 << 30) - (1 << 18), 4, 64, 100),
    (BF16, 16384, 64, 8192, 8192), (F32, 4096, 64, 4096, 14336), (F16, 32, 1024, 4096, 4096)])
def test_large_layers_are_taken(kind, slots, experts, cols, outs):
    assert _takes(kind, slots, experts, cols, outs)


@pytest.mark.parametrize("kind,slots,experts,cols,outs", [
    (BF16, 1 << 30, 2, 4096, 8), (BF16, 1 << 25, 2, 8, 4096), (F16, 1 << 25, 2, 4097, 8), (F32, 1 << 26, 2, 4096, 8),
    (BF16, (1 << 30) + 1, 2, 8, 8), (BF16, 100, 1024, 65536, 65536)])
def test_launches_of_2_32_threads_are_refused(kind, slots, experts, cols, outs):
    assert not _takes(kind, slots, experts, cols, outs)
