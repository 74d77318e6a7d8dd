"""Shared prefixes with infinities in a key: tokens with a score of plus infinity are NaN, ones with minus infinity
give the key no weight, others are as without it, whether the prefix or a request's own keys hold it."""
import math

import pytest
import torch

from fgw_amd.operators.mha import shared_prefix as S
from tests import kv_oracle as K
from tests.test_shared_prefix import _cache, _offsets, _queries


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["prefix", "own"])
@pytest.mark.parametrize("members,new,d,page", [(3, 1, 128, 16), (20, 2, 64, 64), (9, 2, 192, 16), (40, 1, 96, 48), (2, 150, 128, 64)])
def test_an_infinite_key(members, new, d, page, where):
    """The oracle's bound, without the infinity, of which the part for the weights is doubled: a key's weight is far below
    a half here, so without it the others' weights grow by less than that."""
    hq, hk, dtype, prefix = 8, 2, torch.bfloat16, 400
    keys = [new + 20 + 7 * i for i in range(members)]
    cache = _cache([members], [prefix], [new] * members, keys, hk, d, page, dtype)
    q = _queries(members * new, hq, d, dtype, std=1.0)
    clean, bound = K.extend_exact(q, *cache, page)
    k, v, table, lens, cu = [x.clone() for x in cache]
    pos, rows = (130, range(members)) if where == "prefix" else (prefix + 5, [1])
    for b in rows:  # (a key of the prefix may lie in copies of its last page)
        k[int(table[b, pos // page]) * page + pos % page, 1, 3] = math.inf
    broken = (k, v, table, lens, cu)
    want, _ = K.extend_exact(q, *broken, page)
    sees = torch.zeros(members * new, hq, dtype=torch.bool)
    sees[slice(None) if where == "prefix" else slice(new, 2 * new), hq // 2:] = True
    lost = (sees & (q[:, :, 3] > 0))[..., None].expand(want.shape)
    assert bool(lost.any()) and bool((sees[..., None] & ~lost).any())
    half = torch.finfo(dtype).eps / 2
    allowed = half * want.abs() + 2 * (bound - half * clean.abs())
    got = S.build_shared_kernel(hq, hk, d, page, dtype, 0, always=True)(
        q.cuda(), *[x.cuda() for x in broken], _offsets([members]).cuda(),
        torch.tensor([prefix], dtype=torch.int32).cuda(), new).cpu().double()
    assert torch.equal(torch.isnan(got), lost)
    assert bool(((got - want).abs() <= allowed)[~lost].all())
