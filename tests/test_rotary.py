"""Rotary positions against a plain 64-bit form: layouts, scalings, types, strides, far and negative
positions, the gradient, and what is refused."""
import math

import pytest
import torch

from fgw_amd.operators.mha import rotary as R
from tests import kv_oracle as K

SCALINGS = [None, dict(kind="linear", factor=4.0), dict(kind="base", factor=8.0),
            dict(kind="yarn", factor=16.0, original=4096), dict(kind="yarn", factor=4.0, original=8192, attention=0.9),
            dict(kind="bands", factor=8.0, original=8192, low=1.0, high=4.0)]


# ---- frequencies (CPU) -------------------------------------------------------------------------

@pytest.mark.parametrize("scaling", SCALINGS, ids=lambda s: s["kind"] if s else "none")
@pytest.mark.parametrize("dim,base", [(16, 10000.0), (48, 500000.0), (128, 10000.0)])
def test_frequencies_are_those_of_the_formulas(dim, base, scaling):
    got, s = R.rotary_frequencies(dim, base, scaling)
    want, t = K.frequencies(dim, base, scaling)
    torch.testing.assert_close(torch.tensor(got, dtype=torch.float64), want, rtol=1e-14, atol=0)
    assert s == pytest.approx(t, rel=1e-14)


def test_turns_are_the_frequencies_as_fractions_of_a_turn():
    r = R.Rotary(64, base=1e6, device="cpu")
    for turn, w in zip(r.turns.tolist(), R.rotary_frequencies(64, 1e6)[0]):
        assert (turn % 2**64) / 2**64 == pytest.approx(w / (2 * math.pi), rel=1e-15)


def test_yarn_keeps_fast_pairs_and_divides_slow_ones():
    w, s = R.rotary_frequencies(128, scaling=dict(kind="yarn", factor=4.0, original=4096))
    plain, _ = R.rotary_frequencies(128)
    assert w[0] == plain[0] and w[-1] == plain[-1] / 4 and s == 0.1 * math.log(4.0) + 1


@pytest.mark.parametrize("args,message", [
    (dict(dim=0), "multiple of 16"), (dict(dim=24), "multiple of 16"), (dict(dim=64, base=1.0), "above 1"),
    (dict(dim=64, base=math.nan), "above 1"), (dict(dim=64, scaling=dict(kind="other", factor=2.0)), "kind"),
    (dict(dim=64, scaling=dict(kind="linear")), "takes factor"),
    (dict(dim=64, scaling=dict(kind="linear", factor=0.0)), "positive"),
    (dict(dim=64, scaling=dict(kind="yarn", factor=2.0)), "takes factor, original"),
    (dict(dim=64, scaling=dict(kind="linear", factor=2.0, low=1.0)), "takes factor"),
    (dict(dim=64, scaling=dict(kind="bands", factor=2.0, original=4096, low=4.0, high=4.0)), "above low"),
])
def test_frequency_refusals(args, message):
    with pytest.raises(ValueError, match=message):
        R.Rotary(args.pop("dim"), device="cpu", **args)


def test_rows_on_the_cpu_are_refused():
    r = R.Rotary(64, device="cpu")
    with pytest.raises(ValueError, match="GPU"):
        R.apply_rotary(torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int32), r)
    with pytest.raises(TypeError, match="Rotary"):
        R.apply_rotary(torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int32), r.turns)


# ---- rows (GPU) --------------------------------------------------------------------------------

def _rows(t, h, d, dtype, seed=0):
    return torch.randn(t, h, d, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _check(got, x, pos, dim, **options):
    want, bound = K.rotate_exact(x, pos, dim, **options)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= bound).all()), float((err - bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("t,h,d,dim,interleaved", [
    (1, 1, 16, 16, False), (1, 3, 64, 64, True), (7, 12, 80, 48, False), (33, 5, 128, 128, True),
    (129, 8, 128, 64, False), (1000, 32, 128, 128, False), (3000, 40, 96, 32, True), (5, 2, 256, 256, False),
    (2, 1, 1024, 1024, True)])
def test_rotation_matches_the_64_bit_form(dtype, t, h, d, dim, interleaved):
    x = _rows(t, h, d, dtype)
    pos = torch.randint(0, 100000, (t,), generator=torch.Generator().manual_seed(1))
    r = R.Rotary(dim, interleaved=interleaved)
    for inverse in (False, True):
        got = R.apply_rotary(x.cuda(), pos.to(torch.int32).cuda(), r, inverse=inverse)
        assert got.is_contiguous() and got.dtype == dtype
        _check(got, x, pos, dim, interleaved=interleaved, inverse=inverse)


@pytest.mark.gpu
@pytest.mark.parametrize("scaling", SCALINGS, ids=lambda s: s["kind"] if s else "none")
def test_scalings_at_far_and_negative_positions(scaling):
    # The oracle's angle p w has an error of p w 2^-53: below the bound up to 2^26 positions.
    x = _rows(8, 3, 64, torch.float32)
    pos = torch.tensor([0, 1, -1, 4095, -70000, 1 << 20, (1 << 26) - 1, -(1 << 26)])
    r = R.Rotary(64, base=500000.0, scaling=scaling)
    for dt in (torch.int32, torch.int64):
        _check(R.apply_rotary(x.cuda(), pos.to(dt).cuda(), r), x, pos, 64, base=500000.0, scaling=scaling)


@pytest.mark.gpu
def test_positions_past_32_bits_turn_modulo_a_turn():
    """2^32 further is the angle of 2^32 positions further, from exact integers."""
    x = _rows(2, 1, 16, torch.float32)
    r = R.Rotary(16)
    pos = torch.tensor([(1 << 40) + 12345, (1 << 62) + 1])
    got = R.apply_rotary(x.cuda(), pos.cuda(), r).cpu().double()
    for i, p in enumerate(pos.tolist()):
        for j, turn in enumerate(r.turns.tolist()):
            t = (turn * p % 2**64) / 2**64 * 2 * math.pi
            a, b = float(x[i, 0, j]), float(x[i, 0, j + 8])
            limit = (abs(a) + abs(b)) * 5 * 2.0 ** -24
            assert abs(float(got[i, 0, j]) - (a * math.cos(t) - b * math.sin(t))) <= limit
            assert abs(float(got[i, 0, j + 8]) - (b * math.cos(t) + a * math.sin(t))) <= limit


@pytest.mark.gpu
def test_strided_rows_in_place_and_given_outputs():
    fused = _rows(9, 7, 64, torch.bfloat16).cuda()
    pos = torch.arange(9, dtype=torch.int32).cuda()
    r = R.Rotary(32)
    want = R.apply_rotary(fused[:, 2:5].contiguous(), pos, r)
    assert torch.equal(R.apply_rotary(fused[:, 2:5], pos, r), want)
    heads_first = fused[:, 2:5].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(R.apply_rotary(heads_first, pos, r), want)
    out = torch.full((9, 3, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    got = R.apply_rotary(fused[:, 2:5], pos, r, out=out[:, :, :64])
    assert got.data_ptr() == out.data_ptr() and torch.equal(out[:, :, :64], want)
    assert bool((out[:, :, 64:] == 7.0).all())
    keep = fused.clone()
    R.apply_rotary(fused[:, 2:5], pos, r, out=fused[:, 2:5])
    assert torch.equal(fused[:, 2:5], want)
    assert torch.equal(fused[:, :2], keep[:, :2]) and torch.equal(fused[:, 5:], keep[:, 5:])


@pytest.mark.gpu
def test_no_rows():
    r = R.Rotary(32)
    got = R.apply_rotary(torch.empty(0, 4, 64, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), r)
    assert got.shape == (0, 4, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_is_the_formulas_and_the_differences(interleaved):
    x = _rows(5, 3, 48, torch.float32).cuda()
    grad = _rows(5, 3, 48, torch.float32, seed=3)
    pos = torch.tensor([0, 1, 77, 4000, 100001])
    scaling = dict(kind="yarn", factor=4.0, original=4096)
    r = R.Rotary(32, interleaved=interleaved, scaling=scaling)
    leaf = x.clone().requires_grad_()
    R.apply_rotary(leaf, pos.cuda(), r).backward(grad.cuda())
    # The transpose of the linear map, from its columns in 64 bits.
    eye = torch.eye(48, dtype=torch.float64)
    for i in range(5):
        cols, _ = K.rotate_exact(eye.reshape(1, 48, 48).float(), pos[i:i + 1], 32, interleaved=interleaved,
                                 scaling=scaling)
        want = grad[i].double() @ cols[0].T  # row j of cols is the map of unit vector j
        _, bound = K.rotate_exact(grad[i:i + 1], pos[i:i + 1], 32, interleaved=interleaved, scaling=scaling)
        assert bool(((leaf.grad[i].cpu().double() - want).abs() <= bound[0]).all())
    # Differences: the map is linear, so a step of any size gives its derivative; fp32 sums of a few
    # hundred terms each side, each off by at most 2^-21 of its size.
    step = _rows(5, 3, 48, torch.float32, seed=4)
    with torch.no_grad():
        diff = (R.apply_rotary(x + step.cuda(), pos.cuda(), r) - R.apply_rotary(x, pos.cuda(), r)).cpu().double()
    left, right = (diff * grad.double()).sum(), (step.double() * leaf.grad.cpu().double()).sum()
    size = (grad.double().abs() * 8).sum()
    assert abs(float(left - right)) <= 2.0 ** -21 * float(size)


@pytest.mark.gpu
def test_gradient_through_expanded_rows_and_twice():
    r = R.Rotary(16)
    pos = torch.arange(6, dtype=torch.int32).cuda()
    one = torch.randn(6, 1, 16, device="cuda", requires_grad=True)
    R.apply_rotary(one.expand(6, 4, 16), pos, r).sum().backward()  # one head to four, grad expanded
    ones = torch.ones(6, 4, 16, device="cuda")
    torch.testing.assert_close(one.grad, R.apply_rotary(ones, pos, r, inverse=True).sum(1, keepdim=True))
    x = torch.randn(6, 2, 16, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(R.apply_rotary(x, pos, r).square().sum(), x, create_graph=True)
    second, = torch.autograd.grad(g.sum(), x)  # of |x|^2: 2 in every place, after two rotations
    torch.testing.assert_close(second, torch.full_like(x, 2.0), rtol=0, atol=2e-6)


@pytest.mark.gpu
def test_gradient_that_starts_at_any_element():
    r = R.Rotary(16)
    pos = torch.arange(6, dtype=torch.int32).cuda()
    x = torch.randn(6, 2, 16, device="cuda", requires_grad=True)
    weights = torch.randn(1 + 6 * 2 * 16, device="cuda")
    flat = torch.cat([torch.zeros(1, device="cuda"), R.apply_rotary(x, pos, r).flatten()])
    flat.backward(weights)  # the rotation's gradient is a view of it, 4 bytes on
    assert torch.equal(x.grad, R.apply_rotary(weights[1:].view(6, 2, 16).clone(), pos, r, inverse=True))


@pytest.mark.gpu
def test_replays_of_a_captured_rotation():
    r = R.Rotary(64)
    x, pos = _rows(9, 4, 64, torch.bfloat16).cuda(), torch.arange(9, dtype=torch.int32).cuda()
    out = torch.empty_like(x)
    R.apply_rotary(x, pos, r, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        R.apply_rotary(x, pos, r, out=out)
    for i in range(3):
        x.copy_(_rows(9, 4, 64, torch.bfloat16, seed=i))
        pos.add_(100 * i)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, R.apply_rotary(x, pos, r))


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    r = R.Rotary(32)
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    wide = torch.zeros(4, 2, 72, dtype=torch.bfloat16, device="cuda")
    for args, message in [
            ((x[0], pos, r), "rows"), ((x.double(), pos, r), "FP16, BF16 or FP32"),
            ((x, pos.float(), r), "int32 or int64"), ((x, pos[:3], r), "positions must be"),
            ((x, pos.cpu(), r), "same GPU"), ((x.transpose(1, 2), pos, r), "last dim"),
            ((wide[:, :, 4:68], pos, r), "16-byte"), ((x[:, :, :16], pos, r), "at most the head dim"),
            ((x[:, :, :40], pos, r), "divisible by 16"), ((x, pos, R.Rotary(32, device="cpu")), "on the GPU of")]:
        with pytest.raises(ValueError, match=message):
            R.apply_rotary(*args)
    for out, message in [(torch.empty_like(x)[:3], "does not match"), (x.float(), "does not match"),
                         (torch.empty(4, 1, 64, dtype=x.dtype, device="cuda").expand(4, 2, 64), "overlap")]:
        with pytest.raises(ValueError, match=message):
            R.apply_rotary(x, pos, r, out=out)
    leaf = x.float().requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        R.apply_rotary(leaf, pos, r, out=torch.empty_like(x.float()))
