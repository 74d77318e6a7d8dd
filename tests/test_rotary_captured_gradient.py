"""The rotation with its gradient captured into a HIP graph, replayed with new rows and positions."""
import pytest
import torch

from fgw_amd.operators.mha.rotary import Rotary, apply_rotary


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_replays_of_a_captured_gradient(dtype):
    r = Rotary(64, interleaved=True)
    x = torch.randn(33, 6, 64, device="cuda").to(dtype).requires_grad_()
    grad, pos = torch.randn(33, 6, 64, device="cuda").to(dtype), torch.arange(33, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # (no eager graph of x outlives its call)
        torch.autograd.grad(apply_rotary(x, pos, r), x, grad)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = apply_rotary(x, pos, r)
        dx, = torch.autograd.grad(out, x, grad)
    for i in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(33, 6, 64, device="cuda"))
        grad.copy_(torch.randn(33, 6, 64, device="cuda"))
        pos.add_(1000 * i)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.detach(), apply_rotary(x.detach(), pos, r))
        assert torch.equal(dx, apply_rotary(grad, pos, r, inverse=True))
