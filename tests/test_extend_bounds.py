"""Sizes that a caller of the C entry may give: splits and workspace of the attention of new tokens stay
those of the card (host code, which runs without a GPU). Lengths past the table."""
import ctypes

import pytest
import torch

from fgw_amd import _lib
from fgw_amd.operators.mha import paged_extend as P
from tests import kv_oracle as K
from tests.test_paged_extend import _cache, _extend_args, _queries


def _workspace(**changes):
    lib = _lib.load()
    floats, counters = ctypes.c_int64(), ctypes.c_int64()
    assert lib.fgw_kv_extend_workspace(ctypes.byref(_extend_args(**changes)), ctypes.byref(floats),
                                       ctypes.byref(counters)) == 0
    return floats.value, counters.value


@pytest.mark.parametrize("sizes", [
    dict(dim=256, width=1 << 20, tokens=1, batch=1, max_new=1, kv_heads=1),
    dict(dim=128, width=1 << 20, tokens=64, batch=64, max_new=1),
    dict(dim=128, width=1 << 20, tokens=200, batch=1, max_new=200, kv_heads=1),
    dict(dim=256, width=1 << 20, tokens=200, batch=3, max_new=200, kv_heads=2),
])
def test_more_compute_units_than_the_card_has_split_no_further(sizes):
    want = _workspace(num_cus=256, **sizes)
    assert want[0] > 0
    for units in (257, 1024, 1 << 17, 2**31 - 1):
        assert _workspace(num_cus=units, **sizes) == want
    assert _workspace(num_cus=64, **sizes)[0] < want[0]
    # A launch's partials lie within the 2^31 bytes of a buffer, with room for both kernels.
    assert 4 * want[0] < 1 << 27


@pytest.mark.gpu
@pytest.mark.parametrize("new,length,window", [(4, 66, None), (4, 66, 8), (1, 70, None), (70, 130, 20)])
def test_a_length_past_the_table_in_the_write_and_in_the_attention(new, length, window):
    """The write goes by the length as given and leaves out what has no place; the attention takes the
    table's capacity for the length."""
    capacity, dtype = 64, torch.bfloat16
    kc, vc, table, full, cu = _cache([new], [capacity], 2, 64, 16, dtype, poison=False)
    k, v = (_queries(new, 2, 64, dtype, seed) for seed in (1, 2))
    q = _queries(new, 4, 64, dtype)
    dev = [x.cuda() for x in (kc, vc, table)]
    lens = torch.tensor([length], dtype=torch.int32)
    P.mha_paged_append(q.cuda(), k.cuda(), v.cuda(), *dev, lens.cuda(), cu.cuda(), 16)
    for j in range(new):
        pos = length - new + j
        if 0 <= pos < capacity:
            row = int(table[0, pos // 16]) * 16 + pos % 16
            kc[row], vc[row] = k[j], v[j]
    assert torch.equal(dev[0].cpu(), kc) and torch.equal(dev[1].cpu(), vc)
    kernel = P.build_extend_kernel(4, 2, 64, 16, dtype, 0, window=window)
    got = kernel(q.cuda(), *dev, lens.cuda(), cu.cuda(), new)
    assert torch.equal(got, kernel(q.cuda(), *dev, full.cuda(), cu.cuda(), new))
    want, bound = K.extend_exact(q, kc, vc, table, full, cu, 16, window=window or 0)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())
