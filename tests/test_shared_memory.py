"""What the cache operators write must share no memory with what they read: the rule that tells views
of one buffer apart, on the CPU against sets of addresses, and the calls that it refuses."""
import random

import pytest
import torch

from fgw_amd import _lib
from fgw_amd.operators.mha import cache_pages as C, paged_extend as P
from fgw_amd.operators.mha.rotary import Rotary, apply_rotary

shares = _lib.load_kv_module().shares_memory


def _elements(x):
    at = torch.full((1,), x.storage_offset(), dtype=torch.int64)
    for n, s in zip(x.shape, x.stride()):
        at = (at[:, None] + torch.arange(n) * s).flatten()
    return set(at.tolist())


@pytest.mark.parametrize("seed", range(8))
def test_views_taken_for_apart_share_no_element(seed):
    rng = random.Random(seed)
    buffer = torch.zeros(4000, dtype=torch.bfloat16)
    told = touching = 0
    for _ in range(1500):
        views = []
        d, token = rng.choice((1, 4, 8)), rng.choice((8, 16, 24, 48, 96))
        for _ in range(2):
            sizes = (rng.randint(1, 6), rng.randint(1, 5), d)
            strides = (rng.choice((token, token, rng.randint(0, 60))), rng.choice((d, 2 * d, 3 * d, rng.randint(0, 90))), 1)
            views.append(buffer.as_strided(sizes, strides, rng.randint(0, 200)))
        common = bool(_elements(views[0]) & _elements(views[1]))
        assert shares(views[0], views[1]) == shares(views[1], views[0])
        if common:
            assert shares(*views), [(x.shape, x.stride(), x.storage_offset()) for x in views]
        touching += common
        told += not shares(*views)
    assert told > 100 and touching > 100


def test_views_of_one_buffer_side_by_side():
    fused = torch.zeros(5, 8, 16, dtype=torch.float16)
    thirds = torch.zeros(5, 4, 3, 16)
    first = torch.zeros(8, 5, 16)
    apart = [
        (fused[:, :4], fused[:, 4:6]), (fused[:, 4:6], fused[:, 6:8]), (fused[:, :4], fused[:, 4:8]),
        (fused[:1, :4], fused[:1, 4:6]), (fused[:, 2:3], fused[:, 7:8]), (fused[:3], fused[3:]),
        (fused[..., :8], fused[..., 8:]), (thirds[:, :, 0], thirds[:, :, 1]), (thirds[:, :, 2], thirds[:, :, 0]),
        (first[:4].transpose(0, 1), first[4:].transpose(0, 1)), (fused, thirds), (fused[:0], fused), (fused, fused[2:2]),
    ]
    for a, b in apart:
        assert not shares(a, b) and not shares(b, a)
    for a, b in [(fused, fused), (fused[:, :4], fused[:, 3:5]), (fused[1:4], fused[:, :1]), (fused[:, :4], fused[1:, :4]),
                 (thirds[:, :, 0], thirds[:, 1, 0:2]), (fused[..., :9], fused[..., 8:]), (fused.view(-1)[7:8], fused[:, :1])]:
        assert shares(a, b) and shares(b, a)


# ---- refused on the host before any launch -----------------------------------------------------

@pytest.fixture
def step():
    """Five tokens of two requests, 4 + 2 + 2 heads of one projection, and a pool of 8 pages."""
    fused = torch.randn(5, 8, 64, device="cuda").to(torch.bfloat16)
    buffer = torch.zeros(2, 8 * 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    lens, cu = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([40, 9], [0, 3, 5]))
    return fused, buffer, (table, lens, cu)


@pytest.mark.gpu
def test_append_refuses_outputs_over_its_inputs(step):
    fused, (kc, vc), meta = step
    q, k, v = fused[:, :4], fused[:, 4:6], fused[:, 6:8]
    rotary = Rotary(64)
    kept = fused.clone()
    in_pool = kc.view(-1, 4, 64)[:5]
    for bad in (fused[:, 4:8], in_pool, vc.view(-1, 4, 64)[20:25], fused.flatten()[:5 * 4 * 64 + 1024][1024:].view(5, 4, 64)):
        for r in (rotary, None):
            with pytest.raises(ValueError, match="share memory|memory apart"):
                P.mha_paged_append(q, k, v, kc, vc, *meta, 16, rotary=r, q_out=bad)
    with pytest.raises(ValueError, match="share memory"):
        P.mha_paged_append(in_pool, k, v, kc, vc, *meta, 16)
    for rows in (kc[3:8], vc[60:65]):
        with pytest.raises(ValueError, match="share memory"):
            P.mha_paged_append(q, rows, v, kc, vc, *meta, 16)
        with pytest.raises(ValueError, match="share memory"):
            P.mha_paged_append(q, k, rows, kc, vc, *meta, 16, rotary=rotary)
    with pytest.raises(ValueError, match="share memory"):
        table = kc.view(torch.int32).view(-1)[:8].view(2, 4)
        P.mha_paged_append(q, k, v, kc, vc, table, *meta[1:], 16)
    assert torch.equal(fused, kept) and not kc.any() and not vc.any()


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["heads", "thirds"])
def test_append_takes_views_side_by_side_and_q_itself(step, layout):
    fused, (kc, vc), meta = step
    rotary = Rotary(64)
    if layout == "heads":
        q, k, v = fused[:, :2], fused[:, 4:6], fused[:, 6:8]
        spare = fused[:, 2:4]
    else:
        fused = torch.randn(5, 2, 4, 64, device="cuda").to(torch.bfloat16)
        q, k, v, spare = fused.unbind(2)
    want = P.mha_paged_append(q.clone(), k.clone(), v.clone(), kc, vc, *meta, 16, rotary=rotary)
    keys, values = kc.clone(), vc.clone()
    for out in (spare, q):
        kc.zero_()
        vc.zero_()
        P.mha_paged_append(q, k, v, kc, vc, *meta, 16, rotary=rotary, q_out=out)
        assert torch.equal(out, want) and torch.equal(kc, keys) and torch.equal(vc, values)


@pytest.mark.gpu
def test_attention_and_rotation_refuse_outputs_over_their_inputs(step):
    fused, (kc, vc), meta = step
    q = fused[:, :4].contiguous()
    kernel = P.build_extend_kernel(4, 2, 64, 16, "bfloat16", 0)
    for pool in (kc, vc):
        with pytest.raises(ValueError, match="share memory"):
            kernel(q, kc, vc, *meta, 3, pool.view(-1, 4, 64)[1:6])
        with pytest.raises(ValueError, match="share memory"):
            P.mha_paged_extend(q, kc, vc, *meta, 16, out=pool.view(-1, 4, 64)[-5:])
    pos = torch.zeros(1280, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        apply_rotary(fused, pos[:5], Rotary(64), out=pos.view(torch.bfloat16).view(5, 8, 64))


@pytest.mark.gpu
def test_books_lists_and_pools_must_be_apart():
    pages, rows, width, page = 8, 4, 6, 4
    books = C.new_books(pages, rows, width)
    refs, table, lens = books
    pools = [torch.zeros(pages * page, 8, device="cuda") for _ in range(2)]
    ids = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
    buffer = torch.zeros(pages * page + page, 8, device="cuda")
    within = buffer.view(torch.int32).view(-1)
    table2 = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
    calls = [
        lambda: C.reserve_rows(*books, table[0, :4], page), lambda: C.reserve_rows(*books, refs[2:6], page),
        lambda: C.reserve_rows(refs, table2, table2.view(-1)[:rows], ids, page),
        lambda: C.reserve_rows(table2.view(-1)[:pages], table2, lens, ids, page),
        lambda: C.free_rows(*books, table[1], page), lambda: C.free_rows(*books, lens, page),
        lambda: C.fork_rows(pools, *books, ids[:2], table[0, 2:4], page), lambda: C.fork_rows(pools, *books, lens, ids, page),
        lambda: C.fork_rows([buffer[:-page], buffer[page:]], *books, ids[:1], ids[1:2], page),
        lambda: C.fork_rows([pools[0], buffer[:-page]], *books, within[5:6], ids[1:2], page),
        lambda: C.compact_pages([buffer[1:1 - page], pools[0], buffer[:-page]], *books, page),
        lambda: C.compact_pages([buffer[:-page]], within[:pages], table, lens, page),
        lambda: C.copy_pages([buffer[:-page]], within[:2], ids[:2], page),
        lambda: C.copy_pages([buffer[page:], buffer[:-page]], ids[:1], ids[1:2], page),
    ]
    for call in calls:
        with pytest.raises(ValueError, match="share memory"):
            call()
    assert not refs.any() and not lens.any() and bool((table == -1).all())
    # Neighbours in one buffer, parts of one pool's layers, and one pool twice are taken.
    layers = torch.randn(2, 2, pages * page, 8, device="cuda")
    want = layers.clone()
    want.view(4, pages, -1)[:, 5] = want.view(4, pages, -1)[:, 2]
    C.copy_pages([*layers[0], *layers[1], layers[0, 0]], ids[2:3], ids[2:3] + 3, page)
    assert torch.equal(layers, want)
    assert C.reserve_rows(*books, ids, page).tolist() == [0, 0] and lens.tolist() == [0, 1, 2, 3]
    assert C.reserve_rows(*books, lens, page).tolist() == [0, 0] and lens.tolist() == [0, 2, 4, 6]
