"""Attention weight of many rows where a program of the second and of the third kernel takes several items, one after
the other through the same LDS; rows of samples that hold the same pages."""
import pytest
import torch

from tests import eviction_oracle as X
from tests.test_attention_weight import _cache, _check, _queries, _run, _scores
from tests.test_shared_prefix import _cache as _samples

CUS = 256


def _items(news, lens, group, part):
    """(blocks of 256 keys that some row of a part sees, of all parts; blocks of the requests with several parts), of a
    K/V head."""
    columns = sums = 0
    for n, length in zip(news, lens):
        rows = n * group
        parts = -(-rows // part)
        for c in range(parts):
            hi = length - n + (min((c + 1) * part, rows) - 1) // group + 1
            columns += max(0, -(-hi // 256))
        sums += -(-length // 256) if parts > 1 else 0
    return columns, sums


# (new tokens, lens, query heads, K/V heads, D, page, rows of a part): more items than programs, two to a CU of the
# second kernel (one above D 128), four of the third.
CASES = {
    "dim_64": ([1500, 1, 1300], [1500, 40, 3000], 16, 16, 64, 16, 256),
    "dim_128": ([1100, 1000, 70], [2900, 2000, 333], 16, 8, 128, 64, 512),
    "dim_96": ([700, 650], [2500, 3000], 24, 12, 96, 48, 512),
    "dim_256": ([900, 17, 1100], [1900, 300, 2500], 4, 4, 256, 64, 256),
    "dim_192": ([800, 500], [3000, 1200], 8, 8, 192, 16, 256),
    "sums": ([600, 600, 600], [2000, 1000, 1400], 64, 64, 16, 16, 512),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", CASES)
def test_more_items_than_programs(name):
    news, lens, hq, hk, d, page, part = CASES[name]
    columns, sums = _items(news, lens, hq // hk, part)
    assert (4 * CUS < sums * hk) if name == "sums" else (CUS * (1 if d > 128 else 2) < columns * hk)
    dtype = torch.float16 if d == 96 else torch.bfloat16
    cache = _cache(news, lens, hk, d, page, dtype)
    q = _queries(sum(news), hq, d, dtype)
    scores = _scores(cache, hk, page)
    print(name, columns * hk, sums * hk, flush=True)
    _check(_run(scores, q, cache, page, max(news), decay=0.5), scores, q, cache, page, max(news), name, decay=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 5, 30])
def test_samples_on_the_same_pages(new):
    """Three groups of samples, the whole pages of a prefix in every row of its group."""
    members, prefixes, hk, d, page = [9, 20, 3], [1500, 2300, 100], 4, 128, 16
    keys = [new + 13 * i for i in range(32)]
    k, _, table, lens, cu = _samples(members, prefixes, [new] * 32, keys, hk, d, page, torch.bfloat16)
    cache = (k, table, lens, cu)
    q = _queries(32 * new, 16, d, torch.bfloat16)
    scores = _scores(cache, hk, page)
    _check(_run(scores, q, cache, page, new), scores, q, cache, page, new, new)
