"""Attention weight over a table of more than 2^29 keys: every key counts once in a row's normalisation, however
many splits the row has."""
import pytest
import torch

from fgw_amd.operators.mha import eviction as E


@pytest.mark.gpu
def test_a_row_of_nine_million_blocks():
    """The same few pages over and over, so a key weighs as much as all of its copies.

    One K/V head has 512 splits of 17579 blocks of 64 keys. A row's sum takes an addition for each 32 of them to a
    running sum and one a split: 2^-24 each; scores as in eviction_oracle."""
    new, d, page, pages, length = 64, 16, 1 << 16, 4, 9_000_000 * 64
    dtype, gen = torch.bfloat16, torch.Generator().manual_seed(3)
    q = torch.randn(new, 1, d, generator=gen).to(dtype)
    k = torch.randn(pages * page, 1, d, generator=gen).to(dtype)
    width = -(-length // page)
    table = (torch.arange(width, dtype=torch.int32) % pages).view(1, width).cuda()
    scores = torch.zeros(1, 1, width * page, device="cuda")
    E.add_weights(scores, q.cuda(), k.cuda(), table, torch.tensor([length], dtype=torch.int32, device="cuda"),
                  torch.tensor([0, new], dtype=torch.int32, device="cuda"), page, new)

    period = pages * page
    x = q[:, 0].double().cuda() @ k[:, 0].double().cuda().T * d ** -0.5
    weight = x.exp()
    seen = length - new + 1 + torch.arange(new, device="cuda")           # keys of each row
    whole, rest = seen // period, seen % period
    below = torch.arange(period, device="cuda")[None] < rest[:, None]
    total = weight.sum(1) * whole + (weight * below).sum(1)
    p = weight / total[:, None]
    size = float((q[:, 0].double().abs() @ k[:, 0].double().abs().T).amax()) * d ** -0.5
    unit = 2.0 ** -24
    off = unit * (2 * (d + 8) * size + 17579 * 2 + 512 + 16 + 4 * (size + 21) + new / 8 + 32) + 2.0 ** -20
    want = p.sum(0)
    periods = (length - new) // period
    got = scores[0, 0, :periods * period].view(periods, period)
    for part in got.split(256):
        assert bool(((part.double() - want).abs() <= off * want).all())
    for j in range(new):                                                 # the new tokens' own keys
        key = length - new + j
        own = float(p[j:, key % period].sum())
        assert abs(float(scores[0, 0, key]) - own) <= off * own, j
    assert not bool(scores[0, 0, length:].any())
