"""ExpertMlp as programs call it: captured into a graph, on another stream, on a
single row, on none, on rows that are not finite."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _mix(cols, hidden, outs, experts, choices, dtype=F32):
    from npa_amd import experts as E
    torch.manual_seed(cols)
    return E.ExpertMlp(cols, hidden, outs, experts, choices, device="cuda", dtype=dtype)


@pytest.mark.parametrize("rows,cols,hidden,outs,experts,choices,dtype", [
    (700, 66, 128, 18, 8, 1, F32), (3000, 66, 128, 18, 4, 2, F32), (300, 40, 48, 16, 70, 3, F32),
    (2000, 64, 256, 64, 8, 2, BF16), (40, 512, 1024, 512, 16, 2, BF16), (900, 20, 128, 8, 1024, 1, F32)])
def test_streams_and_graphs(rows, cols, hidden, outs, experts, choices, dtype):
    mix = _mix(cols, hidden, outs, experts, choices, dtype)
    g = torch.Generator(device="cuda").manual_seed(1)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)
    x, up = randn(rows, cols).requires_grad_(True), randn(rows, outs)
    leaves = [x, *mix.parameters()]

    def run():
        y = mix(x)
        return [y.detach(), *torch.autograd.grad(y, leaves, up)]

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    del got, want
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(4):  # other rows, and with them other experts, every time
        with torch.no_grad():
            x.copy_(randn(rows, cols))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, run()))


def test_single_rows_and_none():
    mix = _mix(20, 128, 8, 5, 5)
    x = torch.randn(6, 20, device="cuda")
    y = mix(x)
    assert y.shape == (6, 8) and mix(x[0]).shape == (8,)
    # one row and six may run in other kernels: float32 sums of 20 and 128 products
    assert torch.allclose(mix(x[0]), y[0], rtol=1e-5, atol=1e-5) and torch.allclose(mix(x[:1])[0], y[0], rtol=1e-5, atol=1e-5)
    none = mix(x[:0])
    assert none.shape == (0, 8)
    for p in torch.autograd.grad(none.sum(), list(mix.parameters())):
        assert not p.any()


def test_rows_that_are_not_finite():
    mix = _mix(20, 48, 8, 4, 2)
    x = torch.randn(200, 20, device="cuda")
    bad = x.clone()
    bad[3, 4], bad[77, 0], bad[199, 19] = float("nan"), float("inf"), float("-inf")
    fine = [i for i in range(200) if i not in (3, 77, 199)]
    with torch.no_grad():
        y, want = mix(bad), mix(x)
    assert not torch.isfinite(y[[3, 77, 199]]).all(1).any()
    assert torch.allclose(y[fine], want[fine], rtol=1e-5, atol=1e-5)
