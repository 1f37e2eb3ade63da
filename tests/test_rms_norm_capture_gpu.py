"""A backward pass captured into a graph while an eager graph of the same leaves, made on the default stream, is alive: refused on the host, before
autograd's engine makes the default stream wait for the capture."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _in_capture(side, f):
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.capture_begin()
        try:
            return graph, f()
        finally:
            graph.capture_end()


def test_an_eager_graph_of_the_same_leaves():
    from od_wscl_amd import layers
    assert torch.cuda.current_stream().cuda_stream == torch.cuda.default_stream().cuda_stream
    x, w = torch.randn(6, 40, device="cuda", requires_grad=True), torch.ones(40, device="cuda", requires_grad=True)
    dy, side = torch.randn(6, 40, device="cuda"), torch.cuda.Stream()
    want = torch.autograd.grad(layers.rms_norm(x, w), (x, w), dy)
    alive = layers.rms_norm(x, w)

    def refused():
        y = layers.rms_norm(x, w)
        with pytest.raises(RuntimeError, match="default stream"):
            torch.autograd.grad(y, (x, w), dy)
    _in_capture(side, refused)
    torch.cuda.synchronize()
    # what does not reach the leaf that the eager graph holds is not refused
    v = w.detach().clone().requires_grad_(True)
    graph, (dw,) = _in_capture(side, lambda: torch.autograd.grad(layers.rms_norm(x, v), (v,), dy))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(dw, want[1])
    # an input that was computed on the default stream
    z = x * 1.0
    _in_capture(side, lambda: pytest.raises(RuntimeError, torch.autograd.grad, layers.rms_norm(z, v), (z,), dy).match("default stream"))
    torch.cuda.synchronize()
    for a, b in zip(torch.autograd.grad(alive, (x, w), dy), want):              # eager as ever
        assert torch.equal(a, b)


def test_captured_once_the_eager_graph_is_gone():
    from od_wscl_amd import layers
    x, w = torch.randn(6, 40, device="cuda", requires_grad=True), torch.ones(40, device="cuda", requires_grad=True)
    dy, side = torch.randn(6, 40, device="cuda"), torch.cuda.Stream()
    layers.rms_norm(x, w).backward(dy)
    torch.cuda.synchronize()
    graph, got = _in_capture(side, lambda: torch.autograd.grad(layers.rms_norm(x, w), (x, w), dy))
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(6, 40, generator=torch.Generator().manual_seed(k)))
        a, b = (t.detach().clone().requires_grad_(True) for t in (x, w))
        want = torch.autograd.grad(layers.rms_norm(a, b), (a, b), dy)
        graph.replay()
        torch.cuda.synchronize()
        for u, v in zip(got, want):
            assert torch.equal(u, v)
