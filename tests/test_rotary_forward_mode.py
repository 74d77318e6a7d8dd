"""Forward-mode derivatives of the rotation: the map is linear, so a tangent is rotated as its rows are."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from fgw_amd.operators.mha.rotary import Rotary, apply_rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_tangent_is_the_rotated_tangent(inverse, requires_grad):
    r = Rotary(32, scaling=dict(kind="yarn", factor=4.0, original=4096))
    x, t = (torch.randn(5, 3, 48, device="cuda") for _ in range(2))
    x.requires_grad_(requires_grad)
    pos = torch.tensor([0, 1, 77, 4000, 100001], device="cuda")
    with fwd.dual_level():
        out = fwd.unpack_dual(apply_rotary(fwd.make_dual(x, t), pos, r, inverse=inverse))
        assert torch.equal(out.primal, apply_rotary(x.detach(), pos, r, inverse=inverse))
        assert torch.equal(out.tangent, apply_rotary(t, pos, r, inverse=inverse))
        assert fwd.unpack_dual(apply_rotary(t, pos, r)).tangent is None


def test_tangents_at_any_stride_and_without_gradients():
    r, pos = Rotary(16), torch.arange(6, dtype=torch.int32, device="cuda")
    x = torch.randn(6, 4, 16, device="cuda")
    one = torch.randn(6, 1, 16, device="cuda")
    for t in (one.expand(6, 4, 16), torch.randn(6, 16, 4, device="cuda").transpose(1, 2),
              torch.randn(6 * 4 * 16 + 1, device="cuda")[1:].view(6, 4, 16)):
        with torch.no_grad(), fwd.dual_level():
            out = fwd.unpack_dual(apply_rotary(fwd.make_dual(x, t), pos, r))
            assert torch.equal(out.tangent, apply_rotary(t.contiguous().clone(), pos, r))


def test_tangent_of_the_gradient():
    """Forward over reverse: of |rotated x|^2 / 2, whose gradient is x itself (s = 1)."""
    r, pos = Rotary(16), torch.arange(6, dtype=torch.int32, device="cuda")
    x, t = (torch.randn(6, 2, 16, device="cuda") for _ in range(2))
    with fwd.dual_level():
        dual = fwd.make_dual(x.requires_grad_(), t)
        g, = torch.autograd.grad(apply_rotary(dual, pos, r).square().sum() / 2, dual, create_graph=True)
        torch.testing.assert_close(fwd.unpack_dual(g).tangent, t, rtol=0, atol=2e-6)


def test_an_output_in_place_of_a_dual_tensor_is_refused():
    r, pos = Rotary(16), torch.arange(6, dtype=torch.int32, device="cuda")
    x = torch.randn(6, 4, 16, device="cuda")
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(ValueError, match="gradient"):
            apply_rotary(dual, pos, r, out=torch.empty_like(x))
        with pytest.raises(ValueError, match="gradient"):
            apply_rotary(torch.randn_like(x), pos, r, out=dual)
