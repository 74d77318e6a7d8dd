"""Attention weight where queries or keys hold infinities: a key whose score is minus infinity weighs nothing, a
row that sees a score of plus infinity is NaN, as after a softmax, and nothing else changes."""
import math

import pytest
import torch

from tests import eviction_oracle as X
from tests.test_attention_weight import _cache, _queries, _run


def _relative(q, k, used, g, length, scale):
    """Largest relative error of a sum: eviction_oracle's, with the largest score of any row and finite key."""
    d, unit = q.shape[-1], 2.0 ** -24
    finite = lambda x: torch.where(x.isfinite(), x, 0.0).double().abs().flatten(0, 1)
    s = float((finite(q) @ finite(k).T).amax()) * scale
    return unit * (2 * (d + 8) * s + length / 32 + 16 + 4 * (s + math.log(length) + 1) + g * used / 8 + 34) + 2.0 ** -20


# (new tokens, keys before them, query heads, K/V heads, D, page): scores kept, whole and split, 32 rows and 64;
# two passes with rows that leave a tile part empty, split, in parts, at D 256.
SHAPES = {"one": (1, 90, 1, 1, 64, 16), "kept": (3, 300, 4, 1, 64, 16), "kept_split": (2, 9000, 8, 2, 128, 64),
          "kept_tall": (11, 700, 8, 2, 128, 16), "kept_wide": (16, 700, 4, 1, 256, 16), "rows_50": (50, 300, 1, 1, 64, 16),
          "rows_99": (33, 1000, 3, 1, 96, 48), "full_tiles": (64, 500, 2, 2, 128, 64), "parts": (1100, 40, 1, 1, 64, 16),
          "rows_wide": (67, 400, 1, 1, 256, 16)}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("what", ["minus", "plus_in_one_row", "two_keys", "query", "new_key"])
@pytest.mark.parametrize("name", SHAPES)
def test_infinities(name, what, dtype):
    new, before, hq, hk, d, page = SHAPES[name]
    length = new + before
    k, table, lens, cu = _cache([new], [length], hk, d, page, dtype)
    k = torch.where(k.isfinite(), k, 0.0)
    q = _queries(new, hq, d, dtype)
    row_of = lambda pos: int(table[0, pos // page]) * page + pos % page
    if what == "query":  # scores of both infinities
        q[new // 2, -1, 5] = math.inf
    else:
        q[:, :, 5] = -q[:, :, 5].abs() - 0.125
        k[row_of(length - 1 if what == "new_key" else before // 2), -1, 5] = math.inf
    if what == "plus_in_one_row":
        q[new // 2, -1, 5] = 0.5
    if what == "two_keys":  # minus and plus infinity in the same rows
        k[row_of(0), -1, 5] = -math.inf
    cache = (k, table, lens, cu)
    scores = torch.zeros(1, hk, table.shape[1] * page)
    want, _ = X.weights_exact(scores, q, *cache, page, new)
    lost = torch.isnan(want)
    assert bool(lost.any()) == (what not in ("minus", "new_key"))
    print(name, what, dtype, flush=True)
    got = _run(scores, q, cache, page, new).cpu().double()
    assert torch.equal(torch.isnan(got), lost)
    off = ((got - want).abs() - (_relative(q, k, new, hq // hk, length, d ** -0.5) * want + 1e-30 * new))[~lost]
    assert bool((off <= 0).all()), float(off.max())
