"""Attention over shared prefixes for requests of few rows holds its weights in as many bits as without sharing:
two numbers of the input type, whatever the number of rows of a group.

With p as hi + lo, lo the rest of p beside hi, p is off by half^2 p at most (half = eps / 2 of the type), where
kv_oracle's bound has half p; A, the sum of p |v|, is what the oracle gives for |v|."""
import pytest
import torch

from fgw_amd.operators.mha import paged_extend as P
from fgw_amd.operators.mha import shared_prefix as S
from tests import kv_oracle as K
from tests.test_shared_prefix import _cache, _offsets, _queries


def _check(got, q, cache, page, dtype, label):
    want, bound = K.extend_exact(q, *cache, page)
    k, v, table, lens, cu = cache
    size, _ = K.extend_exact(q, k, v.abs(), table, lens, cu, page)
    half = torch.finfo(dtype).eps / 2
    err, allowed = (got.cpu().double() - want).abs(), bound - (half - half * half) * size
    print(label, "largest error, of its bound: %.3f" % float((err / allowed).max()), flush=True)
    assert bool((err <= allowed).all()), label


# (members, prefixes, new tokens, keys behind the prefix, query heads, K/V heads, D, page): groups of up to 64 rows of a
# K/V head, of some hundred, of more than 2048.
CASES = {
    "60_rows": ([15], [900], [1] * 15, [1 + i for i in range(15)], 8, 2, 128, 16),
    "68_rows": ([17], [900], [1] * 17, [1 + i for i in range(17)], 8, 2, 128, 16),
    "256_rows": ([64], [3000], [1] * 64, [1 + 5 * i for i in range(64)], 8, 2, 128, 64),
    "dim_64": ([36], [1500], [2] * 36, [2 + 3 * i for i in range(36)], 12, 2, 64, 16),
    "dim_32": ([50], [700], [1] * 50, [1 + 3 * i for i in range(50)], 8, 2, 32, 8),
    "dim_80": ([18], [801], [5] * 18, [5 + 9 * i for i in range(18)], 8, 2, 80, 48),
    "dim_256": ([20], [800], [2] * 20, [2 + 13 * i for i in range(20)], 8, 1, 256, 64),
    "dim_192_groups": ([11, 30], [300, 650], [3] * 41, [3 + 7 * (i % 9) for i in range(41)], 8, 2, 192, 7),
    "2100_rows": ([70], [600], [15] * 70, [15 + i for i in range(70)], 4, 2, 128, 64),
    "2304_rows_dim_64": ([72], [500], [8] * 72, [8 + i % 30 for i in range(72)], 4, 1, 64, 16),
    "2304_rows_ragged_pages": ([72, 72], [333, 90], [4] * 144, [4 + i % 30 for i in range(144)], 16, 2, 96, 7),
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("name", CASES)
def test_weights_are_held_in_two_numbers(name, dtype):
    members, prefixes, news, keys, hq, hk, d, page = CASES[name]
    cache = _cache(members, prefixes, news, keys, hk, d, page, dtype)
    q = _queries(sum(news), hq, d, dtype)
    dev = [x.cuda() for x in cache]
    kernel = S.build_shared_kernel(hq, hk, d, page, dtype, 0, always=True)
    got = kernel(q.cuda(), *dev, _offsets(members).cuda(), torch.tensor(prefixes, dtype=torch.int32).cuda(), max(news))
    _check(got, q, cache, page, dtype, "shared")
    _check(P.build_extend_kernel(hq, hk, d, page, dtype, 0)(q.cuda(), *dev, max(news)), q, cache, page, dtype, "alone")
