"""Attention weight of many rows over wide tables: what a call asks for is bounded, and sums that are taken a range
of keys at a time are those of one range."""
import ctypes

import pytest
import torch

from fgw_amd import _lib
from fgw_amd.operators.mha import eviction as E
from tests import eviction_oracle as X
from tests.test_attention_weight import _args

BOUND = 256 << 20  # or the pool's bytes


def _need(**changes):
    lib = _lib.load()
    lib.fgw_kv_weights_workspace.restype = ctypes.c_int64
    return 4 * lib.fgw_kv_weights_workspace(ctypes.byref(_args(**changes)))


@pytest.mark.parametrize("tokens,batch,last,heads,keys", [
    (64 * 300, 64, 300, 32, 1 << 20), (2 * 4096, 2, 4096, 32, 1 << 20), (8 * 600, 8, 600, 32, 131072),
    (131072, 1, 131072, 64, 131072), (4 * 131072, 4, 131072, 64, 131072), (1100, 1, 1100, 8, 1 << 30)])
def test_partial_sums_are_bounded(tokens, batch, last, heads, keys):
    sizes = dict(tokens=tokens, batch=batch, last=last, heads=heads, kv_heads=8, dim=128, page_size=64,
                 width=keys // 64, scores_stride=keys)
    # Beside the sums: L of a row for each of its splits, at most 512 items more than tiles of 256 rows.
    statistics = 4 * 256 * 8 * (tokens * (heads // 8) // 256 + batch + 64) + 16 * batch
    for pool in (64 << 20, 1 << 30):
        assert 0 < _need(pool_rows=pool // 2048, **sizes) <= max(BOUND, pool) + statistics


def test_requests_of_one_part_have_no_places_for_sums():
    """One request of 3 parts among 1000 of a few rows each."""
    sizes = dict(tokens=3072 + 999, batch=1000, last=3072, heads=8, kv_heads=8, dim=128, page_size=64, width=1024,
                 scores_stride=65536, pool_rows=65536)
    assert _need(**sizes) <= 4 * 8 * 65536 * 2 * (4071 // 1024) + 4 * 256 * 8 * (4071 // 256 + 1000 + 64) + 16 * 1000


@pytest.mark.gpu
def test_a_range_of_keys_at_a_time():
    """64 K/V heads, two requests of two parts and one of one: 2^28 bytes are places for the sums of 262144 keys.
    The same bits as with a pool that is large enough for all of them, and one head against the 64-bit form."""
    heads, d, page, dtype, gen = 64, 16, 64, torch.bfloat16, torch.Generator().manual_seed(11)
    news, lens = [1100, 1030, 3], [300000, 1030, 270000]
    pages, width = 40, 300000 // page + 60
    q = torch.randn(sum(news), heads, d, generator=gen).to(dtype).cuda()
    k = torch.randn(pages * page, heads, d, generator=gen).to(dtype).cuda()
    table = torch.randint(0, pages, (3, width), generator=gen, dtype=torch.int32)
    cu = torch.tensor([0, 1100, 2130, 2133], dtype=torch.int32)
    ints = [x.cuda() for x in (table, torch.tensor(lens, dtype=torch.int32), cu)]
    start = torch.rand(3, heads, width * page, generator=gen).cuda()
    got, whole = start.clone(), start.clone()
    E.add_weights(got, q, k, *ints, page, 1100, decay=0.5)
    large = torch.zeros(8000 * page, heads, d, dtype=dtype, device="cuda")  # 1 GiB
    large[:pages * page] = k
    E.add_weights(whole, q, large, *ints, page, 1100, decay=0.5)
    assert torch.equal(got.view(torch.int32), whole.view(torch.int32))
    for h in (41,):
        want, bound = X.weights_exact(start[:, h:h + 1].cpu(), q[:, h:h + 1].cpu(), k[:, h:h + 1].cpu(), table, ints[1].cpu(),
                                      cu, page, 1100, decay=0.5)
        assert bool(((got[:, h:h + 1].cpu().double() - want).abs() <= bound).all())
