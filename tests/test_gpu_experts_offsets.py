"""The experts' entry points on offsets that no sort gives: whatever they hold,
nothing outside the call's buffers is written.  Each buffer stands inside a
larger one whose pattern on either side has to stay."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
_KIND = {F32: 0, BF16: 1, F16: 2}


class _Guarded:
    """A call's buffer inside a larger one, with a pattern on either side."""

    def __init__(self, nbytes):
        self.room, self.nbytes = 1 << 20, nbytes
        self.all = torch.full((nbytes + 2 * self.room,), 0x5a, dtype=torch.uint8, device="cuda")
        self.ptr = self.all.data_ptr() + self.room

    def check(self, name):
        assert (self.all[:self.room] == 0x5a).all() and (self.all[self.room + self.nbytes:] == 0x5a).all(), name


def _raw_layer(at, slots, experts, cols, outs, dtype, fused=False):
    """The C entry points of a layer (or of the fused MLP of `cols` inputs and `outs` outputs) on the given offsets:
    nothing outside what they are given changes."""
    from npa_amd.sphops import _native
    lib, kind, size = _native.lib, _KIND[dtype], torch.finfo(dtype).bits // 8
    offsets = torch.tensor(at, dtype=torch.int32, device="cuda")
    ones = lambda *s: torch.ones(*s, dtype=dtype, device="cuda")
    x, dy, stream = ones(slots, cols), ones(slots, outs), torch.cuda.current_stream().cuda_stream
    buffers = {}

    def room(name, nbytes):
        buffers[name] = _Guarded(nbytes)
        return buffers[name].ptr

    if fused:
        w1, w2 = ones(experts, 128, cols), ones(experts, outs, 128)
        size_w = lib.sphops_expert_mlp_workspace_bytes(slots, experts, cols, 128, outs)
        mask = room("mask", 16 * slots)
        _native.check(lib.sphops_expert_mlp_forward(x.data_ptr(), w1.data_ptr(), None, w2.data_ptr(), None, offsets.data_ptr(),
                                                    room("y", slots * outs * 4), mask, slots, experts, cols, 128, outs,
                                                    stream))
        _native.check(lib.sphops_expert_mlp_input_grad(dy.data_ptr(), w1.data_ptr(), w2.data_ptr(), mask, offsets.data_ptr(),
                                                       room("dz", slots * cols * 4), slots, experts, cols, 128, outs, stream))
        _native.check(lib.sphops_expert_mlp_weight_grad(
            x.data_ptr(), dy.data_ptr(), w1.data_ptr(), None, w2.data_ptr(), offsets.data_ptr(), room("dw1", w1.numel() * 4),
            room("db1", experts * 512), room("dw2", w2.numel() * 4), room("db2", experts * outs * 4), slots, experts, cols,
            128, outs, room("workspace", size_w), stream))
    else:
        w = ones(experts, outs, cols)
        forward = lib.sphops_expert_linear_workspace_bytes(kind, slots, experts, cols, outs)
        backward = lib.sphops_expert_linear_backward_workspace_bytes(kind, slots, experts, cols, outs)
        _native.check(lib.sphops_expert_linear(x.data_ptr(), kind, cols, w.data_ptr(), None, offsets.data_ptr(),
                                               room("y", slots * outs * size), slots, experts, cols, outs, 1,
                                               room("workspace", forward), stream))
        _native.check(lib.sphops_expert_linear_backward(
            dy.data_ptr(), outs, x.data_ptr(), kind, cols, w.data_ptr(), None, offsets.data_ptr(),
            room("dx", slots * cols * size), room("dw", w.numel() * size), room("db", experts * outs * size), slots, experts,
            cols, outs, room("workspace backward", backward), stream))
    torch.cuda.synchronize()
    for name, b in buffers.items():
        b.check(name)


def _wild(slots, experts, seed):
    rng = np.random.default_rng(seed)
    yield [0, slots] * ((experts + 1) // 2) + [0] * ((experts + 1) % 2)
    yield [slots, 0] * ((experts + 1) // 2) + [slots] * ((experts + 1) % 2)
    yield list(range(experts, -1, -1))
    yield rng.integers(-2 ** 31, 2 ** 31, experts + 1).tolist()
    yield rng.integers(-slots, 2 * slots, experts + 1).tolist()
    yield [0] + sorted(rng.integers(0, slots + 1, experts).tolist())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("slots,experts,cols,outs", [
    (500, 8, 4096, 128),     # cut tiles, more of them than sorted rows have
    (2000, 3, 4096, 128), (1200, 19, 4096, 120), (300, 15, 1001, 33),
    (500, 8, 128, 4096),     # the same in the input gradient
    (2000, 3, 1030, 600),    # operands laid out first
    (3000, 40, 72, 56),      # weight gradients in chunks
    (700, 60, 600, 40),      # few rows an expert
    (20000, 5, 264, 72)])
def test_offsets_that_no_sort_gives_leave_no_buffer(slots, experts, cols, outs, dtype):
    for at in _wild(slots, experts, slots):
        _raw_layer(at, slots, experts, cols, outs, dtype)


@pytest.mark.parametrize("slots,experts,cols,outs", [(500, 8, 20, 16), (40000, 6, 83, 19), (3000, 300, 168, 64)])
def test_fused_mlp_offsets_that_no_sort_gives_leave_no_buffer(slots, experts, cols, outs):
    for at in _wild(slots, experts, slots):
        _raw_layer(at, slots, experts, cols, outs, F32, fused=True)
