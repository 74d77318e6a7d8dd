"""Sizes that a caller of the C entry may give: splits and workspace of the attention of new tokens stay
those of the card. Host code: runs where there is no GPU."""
import ctypes

import pytest

from fgw_amd import _lib
from tests.test_paged_extend import _extend_args


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
