"""Attention of new tokens where what a token sees is not a number: it comes out as NaN, in whole tiles
and in split ones alike."""
import math

import pytest
import torch

from fgw_amd.operators.mha import paged_extend as P
from tests import kv_oracle as K

# (new tokens, cached tokens, query heads, K/V heads, D): few rows whole and split (by the last
# program of a tile and, captured, by a second launch), long tiles whole and split, wide ones alike.
SHAPES = {"few": (2, 60, 4, 2, 128), "few_split": (2, 9000, 4, 2, 128), "few_split_tall": (5, 9000, 16, 2, 64),
          "long": (300, 300, 4, 2, 128), "long_split": (150, 9000, 4, 2, 64), "wide_split": (150, 9000, 2, 1, 192)}


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("what", ["query", "key", "infinite_key", "value"])
@pytest.mark.parametrize("name", SHAPES)
def test_not_a_number_reaches_the_tokens_that_see_it(name, what, captured):
    new, length, hq, hk, d = SHAPES[name]
    page, dtype = 16, torch.bfloat16
    width = -(-length // page)
    gen = torch.Generator().manual_seed(7)
    q, k, v = (torch.randn(n, h, d, generator=gen).to(dtype).cuda() for n, h in (
        (new, hq), (width * page, hk), (width * page, hk)))
    table = torch.arange(width, dtype=torch.int32, device="cuda").view(1, width)
    lens, cu = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([length], [0, new]))
    kernel = P.build_extend_kernel(hq, hk, d, page, dtype, 0)
    kept, cache = q.cpu(), [x.cpu() for x in (k, v, table, lens, cu)]
    assert bool(kernel(q, k, v, table, lens, cu, new).isfinite().all())
    # The last K/V head: a key that all tokens see (in one of many splits), or the last token's query.
    at = (length - new) * 2 // 3
    if what == "query":
        q[-1, -1, 3] = math.nan
    elif what == "value":
        v[at, -1, :] = math.nan
    else:
        k[at, -1, 5] = math.nan if what == "key" else math.inf
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = kernel(q, k, v, table, lens, cu, new)
        graph.replay()
    else:
        out = kernel(q, k, v, table, lens, cu, new)
    hit = torch.zeros(new, hq, dtype=torch.bool)
    if what == "query":
        hit[-1, -1] = True
    else:
        hit[:, hq - hq // hk:] = True
    rest = ~hit
    if what == "infinite_key":  # a score of +infinity is NaN after the softmax, one of -infinity weighs nothing
        hit &= q[:, :, 5].cpu() > 0
    assert bool(out.cpu()[hit].isnan().all())
    # (A row beside them may have another exponent reference, so other roundings.)
    want, bound = K.extend_exact(kept, *cache, page)
    assert bool(((out.cpu().double() - want).abs() <= bound)[rest].all())
