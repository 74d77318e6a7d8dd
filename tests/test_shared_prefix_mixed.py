"""Samples that share a prefix beside other requests of the same call: what those have does not keep the samples from
sharing. Whether they share shows in their rows of the table, which are not read there."""
import pytest
import torch

from fgw_amd.operators.mha import shared_prefix as S
from tests.test_shared_prefix import _cache, _compare, _offsets, _queries


@pytest.mark.gpu
@pytest.mark.parametrize("first", [True, False])
def test_samples_share_beside_a_prompt(first):
    """40 samples of 3000 keys save 490 MB of reading, and a prompt of 600 tokens is in a group of its own, or in none."""
    hq, hk, d, page = 16, 8, 128, 64
    members, prefixes = ([1, 40], [5, 3000]) if first else ([40], [3000])
    news = [600] + [1] * 40 if first else [1] * 40 + [600]
    keys = [700] + [1 + i for i in range(40)] if first else [1 + i for i in range(40)] + [700]
    cache = _cache(members, prefixes, news, keys, hk, d, page, torch.bfloat16)
    q = _queries(sum(news), hq, d, torch.bfloat16)
    broken = [x.clone() for x in cache]
    samples = slice(2, 41) if first else slice(1, 40)
    broken[2][samples, :3000 // page] = -1
    got = S.build_shared_kernel(hq, hk, d, page, "bfloat16", 0)(
        q.cuda(), *[x.cuda() for x in broken], _offsets(members).cuda(), torch.tensor(prefixes, dtype=torch.int32).cuda(), 600)
    _compare(got, q, cache, page, first)
