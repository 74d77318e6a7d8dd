"""Attention of new tokens: results that must be the same bits, a request's alone and in a batch where
its tile is whole in both, and a captured call's and an eager one's, whose splits are joined by
different programs."""
import pytest
import torch

from fgw_amd.operators.mha import paged_extend as P
from tests.test_paged_extend import _cache, _queries

pytestmark = pytest.mark.gpu

# Keys that are never split: rounds of 128 for few rows (four at D <= 64, else three), one split of
# four 64-key blocks for many.
BATCHES = {
    "few": (128, 8, 2, [1, 4, 1, 2], [384, 300, 5, 129], 384),
    "few_narrow": (64, 4, 4, [1, 2, 17, 0, 3], [512, 33, 400, 9, 3], 512),
    "few_tall": (96, 16, 1, [1, 8, 3], [250, 384, 64], 384),
    "few_wide": (256, 4, 2, [2, 1, 9], [384, 31, 200], 384),
    "long": (128, 8, 2, [100, 1, 64], [256, 200, 64], 256),
    "long_narrow": (64, 4, 1, [40, 200, 33], [256, 256, 33], 256),
    "long_wide": (192, 2, 2, [130, 3, 140], [256, 190, 141], 256),
}


@pytest.mark.parametrize("window", [None, 50])
@pytest.mark.parametrize("name", BATCHES)
def test_a_request_alone_and_in_a_batch(name, window):
    d, hq, hk, news, lens, most = BATCHES[name]
    assert max(lens) <= most
    k, v, table, lens, cu = [x.cuda() for x in _cache(news, lens, hk, d, 16, torch.bfloat16)]
    q = _queries(sum(news), hq, d, torch.bfloat16).cuda()
    kernel = P.build_extend_kernel(hq, hk, d, 16, "bfloat16", 0, window=window)
    whole = kernel(q, k, v, table, lens, cu, max(news))
    at = 0
    for b, n in enumerate(news):
        if n:
            own = torch.tensor([0, n], dtype=torch.int32, device="cuda")
            alone = kernel(q[at:at + n], k, v, table[b:b + 1], lens[b:b + 1], own, n)
            assert torch.equal(alone, whole[at:at + n]), (name, b)
        at += n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("d", [16, 32, 48, 64, 80, 128, 192, 256])
@pytest.mark.parametrize("hq,hk,news", [(1, 1, [1, 1]), (8, 2, [1, 2, 1]), (9, 1, [1, 1, 2]), (16, 1, [2, 1]), (4, 4, [31, 5]),
                                        (4, 1, [8, 3, 33]), (8, 2, [40, 1, 3])])
def test_captured_and_eager(hq, hk, news, d, dtype):
    lens = [5000, 300, 1700][:len(news)]
    k, v, table, lens, cu = [x.cuda() for x in _cache(news, lens, hk, d, 16, dtype)]
    q = _queries(sum(news), hq, d, dtype).cuda()
    kernel = P.build_extend_kernel(hq, hk, d, 16, dtype, 0)
    eager = kernel(q, k, v, table, lens, cu, max(news))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernel(q, k, v, table, lens, cu, max(news))
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        assert torch.equal(kernel(q, k, v, table, lens, cu, max(news)), eager)
