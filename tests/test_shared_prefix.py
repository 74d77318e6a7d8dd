"""Attention of new tokens where groups of requests share a prefix: against the 64-bit form over each
request's own row, at the sizes where the two passes and their join can go wrong; graphs, refusals."""
import ctypes
import math

import pytest
import torch

from fgw_amd import _lib
from fgw_amd.operators.mha import shared_prefix as S
from tests import kv_oracle as K


def _offsets(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32)


def _cache(members, prefixes, news, keys, hk, d, page, dtype, seed=0, spare=1):
    """Rows as forks leave them: the whole pages of a prefix in every row of its group, the rest of it in a
    page of each row's own with the same contents. keys: of each request behind its group's prefix (of
    requests in no group: all). Rows that no live token holds are NaN."""
    gen = torch.Generator().manual_seed(seed)
    group = [g for g, m in enumerate(members) for _ in range(m)]
    group += [-1] * (len(news) - len(group))
    lens = [(prefixes[g] if g >= 0 else 0) + n for g, n in zip(group, keys)]
    width = max(1, max(-(-n // page) for n in lens)) + spare
    need = sum(-(-n // page) for n in lens) + sum(p // page + 1 for p in prefixes) + 4
    ids = torch.randperm(need, generator=gen).tolist()
    k = torch.randn(need * page, hk, d, generator=gen).to(dtype)
    v = torch.randn(need * page, hk, d, generator=gen).to(dtype)
    common = [[ids.pop() for _ in range(p // page)] for p in prefixes]
    table, live, seen = [], torch.zeros(need * page, dtype=torch.bool), {}
    for b, (g, n) in enumerate(zip(group, lens)):
        row = (common[g] if g >= 0 else [])[:-(-n // page)]
        row = row + [ids.pop() for _ in range(-(-n // page) - len(row))]
        if g >= 0 and prefixes[g] % page and len(row) > len(common[g]):
            at, rest = row[len(common[g])] * page, prefixes[g] % page
            if g in seen:
                k[at:at + rest], v[at:at + rest] = k[seen[g]:seen[g] + rest], v[seen[g]:seen[g] + rest]
            else:
                seen[g] = at
        table.append(row + [-1] * (width - len(row)))
        pos = torch.arange(n)
        live[torch.tensor(row + [0])[pos // page] * page + pos % page] = True
    k[~live] = math.nan
    v[~live] = math.nan
    return (k, v, torch.tensor(table, dtype=torch.int32), torch.tensor(lens, dtype=torch.int32), _offsets(news))


def _queries(t, hq, d, dtype, seed=5, std=2.0):
    return (torch.randn(t, hq, d, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def _compare(got, q, cache, page, label, **options):
    want, bound = K.extend_exact(q, *cache, page, **options)
    rows = int(cache[4][-1])
    err = (got.cpu().double()[:rows] - want[:rows]).abs()
    assert bool((err <= bound[:rows]).all()), (label, float((err - bound[:rows]).max()))


# (members of each group, prefixes, new tokens, keys behind the prefix, query heads, K/V heads, D, page)
CASES = {
    "two": ([2], [40], [1, 1], [3, 9], 4, 2, 64, 16),
    "whole_pages": ([3], [64], [1, 1, 1], [1, 1, 17], 8, 2, 128, 16),
    "own_token_only": ([4], [333], [1] * 4, [1] * 4, 8, 2, 128, 16),
    "long_prefix_split": ([5], [5000], [1] * 5, [1, 70, 128, 129, 300], 8, 2, 128, 64),
    "groups_ragged": ([2, 5, 3], [100, 31, 700], [1] * 10, [4, 1, 9, 2, 300, 33, 1, 1, 1, 64], 12, 4, 64, 16),
    "empty_requests": ([3, 2], [50, 20], [0, 2, 0, 1, 0], [7, 8, 1, 4, 2], 6, 3, 96, 8),
    "empty_group": ([2, 2, 2], [50, 60, 70], [1, 1, 0, 0, 3, 1], [1, 2, 1, 1, 3, 1], 4, 4, 128, 16),
    "alone_in_group": ([1, 3, 1], [90, 40, 70], [1, 2, 1, 2, 5], [5, 9, 4, 2, 6], 8, 2, 80, 16),
    "behind_the_groups": ([2], [300], [1, 1, 1, 4], [1, 3, 200, 4], 8, 1, 64, 32),
    "one_token_prefix": ([3], [1], [1, 2, 3], [1, 9, 40], 4, 1, 32, 16),
    "dim_16": ([3], [77], [1, 5, 2], [1, 9, 40], 4, 2, 16, 16),
    "dim_192": ([3], [400], [1, 1, 2], [3, 200, 40], 8, 2, 192, 64),
    "dim_256_small_pages": ([2], [131], [2, 1], [3, 20], 4, 2, 256, 7),
    "one_token_pages": ([3], [37], [1, 1, 2], [1, 2, 9], 2, 2, 64, 1),
    "rows_on_a_border": ([8], [500], [4] * 8, [4, 5, 6, 7, 100, 9, 10, 11], 8, 2, 128, 16),   # 128 rows a head
    "rows_past_a_border": ([11], [500], [3] * 11, [3 + 7 * i for i in range(11)], 8, 2, 128, 16),
    "long_tiles": ([70], [1000], [1] * 70, [1 + i % 90 for i in range(70)], 16, 2, 128, 64),
    "long_tiles_split_own": ([40, 30], [2000, 777], [1] * 70, [1 + (i % 7) * 900 for i in range(70)], 8, 1, 128, 16),
    "long_tiles_dim_64": ([36], [1500], [2] * 36, [2 + 3 * i for i in range(36)], 12, 2, 64, 128),
    "long_tiles_dim_96": ([9], [600], [5] * 9, [5 + 11 * i for i in range(9)], 16, 2, 96, 48),
    "wide_tiles": ([20], [800], [2] * 20, [2 + 13 * i for i in range(20)], 8, 1, 256, 64),
    "prompts": ([3], [500], [150, 200, 40], [150, 260, 40], 8, 2, 128, 64),
    "prompts_dim_64": ([2, 2], [300, 64], [300, 70, 33, 150], [301, 70, 90, 150], 4, 1, 64, 16),
    "prompts_wide": ([2], [200], [150, 90], [160, 90], 4, 2, 192, 64),
    "prompts_split_own": ([2], [200], [140, 90], [4000, 90], 2, 1, 128, 16),
    "many_groups": ([2] * 70, [5 + 3 * (i % 40) for i in range(70)], [1] * 140, [1 + i % 50 for i in range(140)], 4, 2, 64, 16),
    "many_in_one": ([150], [90], [1 + i % 2 for i in range(150)], [2 + i % 30 for i in range(150)], 2, 1, 128, 16),
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("name", CASES)
def test_matches_the_64_bit_form(name, dtype):
    members, prefixes, news, keys, hq, hk, d, page = CASES[name]
    cache = _cache(members, prefixes, news, keys, hk, d, page, dtype)
    q = _queries(sum(news), hq, d, dtype)
    print(name, dtype, flush=True)
    kernel = S.build_shared_kernel(hq, hk, d, page, dtype, 0, always=True)
    got = kernel(q.cuda(), *[x.cuda() for x in cache], _offsets(members).cuda(),
                 torch.tensor(prefixes, dtype=torch.int32).cuda(), max(news))
    _compare(got, q, cache, page, name)


# (members, prefixes, new tokens, keys behind, heads, K/V heads, D, page): what is read without sharing, on both
# sides of the rule.
SIZES = {
    "short": ([4], [200], [1] * 4, [1, 2, 3, 4], 8, 2, 128, 16),
    "long_enough": ([40], [3000], [1] * 40, [1 + i for i in range(40)], 16, 8, 128, 64),
    "together_long_enough": ([14] * 3, [2900] * 3, [1] * 42, [1 + i for i in range(42)], 8, 8, 128, 16),
    "too_short_for_the_capacity": ([40], [90], [1] * 40, [1] * 39 + [4000], 16, 8, 128, 64),
    "many_groups": ([2] * 70, [900] * 70, [1] * 140, [1 + i % 9 for i in range(140)], 8, 8, 64, 16),
    "many_groups_long_enough": ([2] * 70, [1900] * 70, [1] * 140, [1 + i % 9 for i in range(140)], 8, 8, 64, 64),
    "many_rows": ([3], [1500], [200, 190, 180], [200, 190, 180], 4, 1, 128, 64),
    "many_rows_in_one_group": ([2, 40], [1500, 3000], [150, 140] + [1] * 40, [150, 140] + [1] * 40, 8, 8, 128, 64),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", SIZES)
def test_shared_where_that_is_faster_gives_the_same(name):
    members, prefixes, news, keys, hq, hk, d, page = SIZES[name]
    cache = _cache(members, prefixes, news, keys, hk, d, page, torch.bfloat16)
    q = _queries(sum(news), hq, d, torch.bfloat16)
    print(name, flush=True)
    got = S.build_shared_kernel(hq, hk, d, page, "bfloat16", 0)(
        q.cuda(), *[x.cuda() for x in cache], _offsets(members).cuda(), torch.tensor(prefixes, dtype=torch.int32).cuda(), max(news))
    _compare(got, q, cache, page, name)


@pytest.mark.gpu
def test_the_prefix_is_read_through_the_first_request():
    """Its row alone counts there: entries of the other rows in the prefix are not looked at."""
    cache = _cache([4], [320], [1] * 4, [1, 5, 40, 2], 2, 128, 16, torch.bfloat16)
    q = _queries(4, 8, 128, torch.bfloat16)
    broken = [x.clone() for x in cache]
    broken[2][1:, :20] = -1
    kernel = S.build_shared_kernel(8, 2, 128, 16, "bfloat16", 0, always=True)
    got = kernel(q.cuda(), *[x.cuda() for x in broken], _offsets([4]).cuda(), torch.tensor([320], dtype=torch.int32).cuda(), 1)
    _compare(got, q, cache, 16, "first row")


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [0, -5, 20, 100])
def test_prefixes_that_not_every_request_reaches(prefix):
    """None, a part, all of what is shared; the last request's new tokens begin within it."""
    members, news, keys = [4], [2, 1, 60, 3], [30, 1, 70, -20]
    cache = _cache(members, [100], news, keys, 2, 64, 16, torch.float16)
    q = _queries(sum(news), 8, 64, torch.float16)
    kernel = S.build_shared_kernel(8, 2, 64, 16, "float16", 0, always=True)
    got = kernel(q.cuda(), *[x.cuda() for x in cache], _offsets(members).cuda(),
                 torch.tensor([prefix], dtype=torch.int32).cuda(), max(news))
    _compare(got, q, cache, 16, prefix)


@pytest.mark.gpu
def test_a_first_request_that_ends_early_shares_less():
    """The first request has 37 keys before its token: the others share those alone."""
    cache = _cache([3], [37], [1, 1, 1], [1, 80, 200], 2, 128, 16, torch.bfloat16)
    q = _queries(3, 8, 128, torch.bfloat16)
    kernel = S.build_shared_kernel(8, 2, 128, 16, "bfloat16", 0, always=True)
    got = kernel(q.cuda(), *[x.cuda() for x in cache], _offsets([3]).cuda(), torch.tensor([64], dtype=torch.int32).cuda(), 1)
    _compare(got, q, cache, 16, "early")


@pytest.mark.gpu
def test_offsets_of_groups_that_say_nothing():
    """Groups past the batch, falling offsets and no group at all: every request reads its own keys."""
    cache = _cache([2], [90], [1, 2], [5, 6], 2, 64, 16, torch.bfloat16)
    dev = [x.cuda() for x in cache]
    q = _queries(3, 4, 64, torch.bfloat16)
    kernel = S.build_shared_kernel(4, 2, 64, 16, "bfloat16", 0, always=True)
    for first, prefixes in (([0], []), ([0, 3], [90]), ([2, 0], [90]), ([-1, 2], [90]), ([0, 0, 0], [90, 90]), ([0, 1, 2], [90, 90])):
        print(first, flush=True)
        got = kernel(q.cuda(), *dev, torch.tensor(first, dtype=torch.int32).cuda(),
                     torch.tensor(prefixes, dtype=torch.int32).cuda(), 2)
        _compare(got, q, cache, 16, first)


@pytest.mark.gpu
@pytest.mark.parametrize("always", [True, False])
def test_a_group_whose_offsets_run_out_of_q(always):
    """Its requests within q read their keys themselves, as without groups; other groups share."""
    news = [1, 2, 1, 1]
    cache = _cache([2, 2], [300, 90], news, [4, 6, 7, 9], 2, 64, 16, torch.bfloat16)
    q = _queries(5, 4, 64, torch.bfloat16)
    dev = [x.cuda() for x in cache]
    first, prefixes = _offsets([2, 2]).cuda(), torch.tensor([300, 90], dtype=torch.int32).cuda()
    kernel = S.build_shared_kernel(4, 2, 64, 16, "bfloat16", 0, always=always)
    want, bound = K.extend_exact(q, *cache, 16)
    for cu, rows in (([0, 1, 3, 4, 9], 4), ([0, 1, 9, 9, 9], 1)):
        print(cu, flush=True)
        dev[4] = torch.tensor(cu, dtype=torch.int32).cuda()
        got = kernel(q.cuda(), *dev, first, prefixes, 2).cpu().double()
        assert bool(((got - want).abs()[:rows] <= bound[:rows]).all()), cu


@pytest.mark.gpu
def test_rows_behind_the_last_request_are_left_and_strides_are_taken():
    cache = _cache([3], [200], [1, 2, 1], [1, 2, 50], 2, 128, 16, torch.bfloat16)
    fused = _queries(7, 12, 128, torch.bfloat16)
    fused[4:] = math.nan
    q = fused.cuda()[:, 2:10]
    out = torch.full((7, 8, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    kernel = S.build_shared_kernel(8, 2, 128, 16, "bfloat16", 0, softmax_scale=0.25, always=True)
    got = kernel(q, *[x.cuda() for x in cache], _offsets([3]).cuda(), torch.tensor([200], dtype=torch.int32).cuda(), 2, out)
    assert got.data_ptr() == out.data_ptr() and bool((out[4:] == 7.0).all())
    _compare(out, fused[:4, 2:10], cache, 16, "padded", scale=0.25)


@pytest.mark.gpu
def test_pages_outside_the_pool_read_as_zeros():
    k, v, table, lens, cu = _cache([2], [128], [1, 1], [40, 9], 2, 64, 16, torch.bfloat16)
    table[:, 3], table[0, 9] = -1, 10**6
    q = _queries(2, 4, 64, torch.bfloat16)
    kernel = S.build_shared_kernel(4, 2, 64, 16, "bfloat16", 0, always=True)
    got = kernel(q.cuda(), *[x.cuda() for x in (k, v, table, lens, cu)], _offsets([2]).cuda(),
                 torch.tensor([128], dtype=torch.int32).cuda(), 1)
    _compare(got, q, (k, v, table, lens, cu), 16, "outside")


@pytest.mark.gpu
@pytest.mark.parametrize("news", [[1, 1, 2], [40, 50, 30]])
def test_pools_past_four_gib(news):
    """Rows whose offsets pass 32 bits: the same bits as in small pools."""
    page, large = 64, 50000  # pages of 128 KB
    k, v, table, lens, cu = [x.cuda() for x in _cache([3], [700], news, [n + 70 for n in news], 8, 128, page, torch.bfloat16)]
    q = _queries(sum(news), 16, 128, torch.bfloat16).cuda()
    first, prefixes = _offsets([3]).cuda(), torch.tensor([700], dtype=torch.int32).cuda()
    kernel = S.build_shared_kernel(16, 8, 128, page, "bfloat16", 0, always=True)
    near = kernel(q, k, v, table, lens, cu, first, prefixes, max(news))
    pools = [torch.zeros(large * page, 8, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for x, y in zip(pools, (k, v)):
        x[-y.shape[0]:] = y
    far = kernel(q, *pools, torch.where(table < 0, -1, table + large - k.shape[0] // page).to(torch.int32), lens, cu, first,
                 prefixes, max(news))
    assert torch.equal(near, far)


@pytest.mark.gpu
def test_nan_of_a_key_reaches_the_rows_that_see_it():
    """A NaN among the shared keys: every row of the group is NaN; among one request's own: its rows."""
    for where in ("prefix", "own"):
        k, v, table, lens, cu = _cache([3], [300], [1, 1, 1], [1, 20, 40], 2, 128, 16, torch.bfloat16)
        pos, b = (130, 0) if where == "prefix" else (310, 1)
        k[int(table[b, pos // 16]) * 16 + pos % 16, 0, 5] = math.nan
        q = _queries(3, 4, 128, torch.bfloat16)
        kernel = S.build_shared_kernel(4, 2, 128, 16, "bfloat16", 0, always=True)
        got = kernel(q.cuda(), *[x.cuda() for x in (k, v, table, lens, cu)], _offsets([3]).cuda(),
                     torch.tensor([300], dtype=torch.int32).cuda(), 1)
        bad = torch.isnan(got).all(-1).cpu()
        want = torch.zeros(3, 4, dtype=torch.bool)
        want[slice(None) if where == "prefix" else slice(1, 2), :2] = True
        assert torch.equal(bad, want), where


@pytest.mark.gpu
def test_captured_and_replayed_after_groups_changed():
    """One graph, replayed with other lengths, tables, groups and prefixes in the same tensors."""
    hq, hk, d, page = 8, 2, 128, 16
    layouts = [([4, 4], [500, 90], [1] * 8, [1, 2, 70, 4, 300, 6, 7, 8]),
               ([6, 2], [300, 200], [1] * 8, [9, 8, 7, 6, 5, 4, 3, 200]),
               ([1, 7], [30, 450], [1] * 8, [1, 1, 1, 1, 60, 61, 62, 63])]
    kernel = S.build_shared_kernel(hq, hk, d, page, "bfloat16", 0, always=True)
    caches = [_cache(*x, hk, d, page, torch.bfloat16, seed=i) for i, x in enumerate(layouts)]
    width = max(c[2].shape[1] for c in caches)
    rows = max(c[0].shape[0] for c in caches)

    def padded(c):
        k, v = (torch.cat([x, torch.zeros(rows - x.shape[0], hk, d, dtype=x.dtype)]) for x in c[:2])
        table = torch.cat([c[2], torch.full((8, width - c[2].shape[1]), -1, dtype=torch.int32)], 1)
        return k, v, table, c[3], c[4]

    caches = [padded(c) for c in caches]
    q = _queries(8, hq, d, torch.bfloat16)
    dev = [x.cuda() for x in caches[0]]
    meta = [_offsets(layouts[0][0]).cuda(), torch.tensor(layouts[0][1], dtype=torch.int32).cuda()]
    qd, out = q.cuda(), torch.zeros(8, hq, d, dtype=torch.bfloat16, device="cuda")
    for _ in range(2):
        kernel(qd, *dev, *meta, 1, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernel(qd, *dev, *meta, 1, out)
    for turn in (0, 1, 2, 1, 0):
        for x, y in zip(dev, caches[turn]):
            x.copy_(y)
        meta[0].copy_(_offsets(layouts[turn][0]))
        meta[1].copy_(torch.tensor(layouts[turn][1], dtype=torch.int32))
        eager = kernel(qd, *dev, *meta, 1)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        _compare(out, q, caches[turn], page, turn)
        _compare(eager, q, caches[turn], page, turn)


@pytest.mark.gpu
def test_two_calls_at_once_on_two_streams():
    cache = _cache([6], [3000], [1] * 6, [1 + 40 * i for i in range(6)], 1, 128, 16, torch.bfloat16)
    dev = [x.cuda() for x in cache]
    meta = [_offsets([6]).cuda(), torch.tensor([3000], dtype=torch.int32).cuda()]
    kernel = S.build_shared_kernel(8, 1, 128, 16, "bfloat16", 0, always=True)
    qs = [_queries(6, 8, 128, torch.bfloat16, seed=s) for s in (1, 2)]
    qd = [x.cuda() for x in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    outs = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i] = kernel(qd[i], *dev, *meta, 1)
    torch.cuda.synchronize()
    for i in range(2):
        _compare(outs[i], qs[i], cache, 16, i)


@pytest.mark.gpu
def test_one_call_checks_its_metadata():
    cache = [x.cuda() for x in _cache([2], [40], [1, 1], [3, 9], 2, 64, 16, torch.bfloat16)]
    q = _queries(2, 4, 64, torch.bfloat16)
    groups, prefixes = _offsets([2]).cuda(), torch.tensor([40], dtype=torch.int32).cuda()
    got = S.mha_paged_shared(q.cuda(), *cache, groups, prefixes, 16, always=True)
    _compare(got, q, [x.cpu() for x in cache], 16, "one call")
    k, v, table, lens, cu = cache

    def ints(*x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    for changes, message in [
            (dict(lens=lens + 10000), "table capacity"), (dict(cu=ints(0, 2, 1)), "cu_seqlens must run"),
            (dict(groups=ints(0, 3)), "cu_groups must run"), (dict(groups=ints(1, 2)), "cu_groups must run"),
            (dict(prefixes=ints(-1)), "must not be negative"), (dict(groups=ints(0, 1, 2)), "metadata shape"),
            (dict(prefixes=prefixes.long()), "int32"), (dict(prefixes=prefixes.cpu()), "same GPU"),
            (dict(groups=groups[None]), "metadata shape")]:
        a = dict(table=table, lens=lens, cu=cu, groups=groups, prefixes=prefixes, **{})
        a.update(changes)
        with pytest.raises(ValueError, match=message):
            S.mha_paged_shared(q.cuda(), k, v, *a.values(), 16)


@pytest.mark.gpu
def test_tensor_refusals():
    cache = [x.cuda() for x in _cache([2], [40], [1, 1], [3, 9], 2, 64, 16, torch.bfloat16)]
    k, v, table, lens, cu = cache
    q = _queries(2, 4, 64, torch.bfloat16).cuda()
    groups, prefixes = _offsets([2]).cuda(), torch.tensor([40], dtype=torch.int32).cuda()
    kernel = S.build_shared_kernel(4, 2, 64, 16, "bfloat16", 0, always=True)
    whole = torch.zeros(2 * 4 * 64 + 16, dtype=torch.bfloat16, device="cuda")
    out, inside = whole[:512].view(2, 4, 64), whole[508:512].view(torch.int32)[:1]
    for args, message in [
            ((q, k, v, table, lens, cu, groups[:0], prefixes[:0], 1), "metadata"),
            ((q, k, v, table, lens, cu, groups, prefixes[:0], 1), "metadata"),
            ((q, k, v, table, lens, cu, groups.long(), prefixes, 1), "int32"),
            ((q, k, v, table, lens, cu, groups, prefixes.cpu(), 1), "same GPU"),
            ((q.half(), k, v, table, lens, cu, groups, prefixes, 1), "FP16/BF16"),
            ((q, k, v, table, lens, cu, groups, prefixes, 0), "max_new"),
            ((q, k, v, table, lens, cu, groups, inside, 1, out), "out must not"),
            ((q, k, v, table, lens, cu, groups, prefixes, 1, q), "out must not")]:
        with pytest.raises(ValueError, match=message):
            kernel(*args)
    with pytest.raises(ValueError, match="requires a gradient"):
        kernel(q, k, v, table, lens, cu, groups, prefixes, 1, out.clone().requires_grad_())


@pytest.mark.parametrize("args,options,message", [
    ((8, 3, 64, 16, "bfloat16", 0), {}, "multiple of the K/V heads"),
    ((8, 2, 72, 16, "bfloat16", 0), {}, "divisible by 16"), ((8, 2, 64, 0, "bfloat16", 0), {}, "page size"),
    ((8, 2, 64, 16, "float32", 0), {}, "FP16/BF16"), ((8, 2, 64, 16, "bfloat16", 0), dict(softmax_scale=0.0), "scale")])
def test_build_refusals(args, options, message):
    with pytest.raises(ValueError, match=message):
        S.build_shared_kernel(*args, **options)


class _Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("token_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class _Extend(ctypes.Structure):
    _fields_ = [("q", _Rows)] + [(n, ctypes.c_void_p) for n in (
        "out", "k_cache", "v_cache", "block_table", "cache_seqlens", "cu_seqlens", "workspace", "counters")] + [
        ("pool_rows", ctypes.c_int64)] + [(n, ctypes.c_int32) for n in (
            "tokens", "batch", "heads", "kv_heads", "dim", "width", "page_size", "max_new", "causal", "window",
            "dtype", "num_cus")] + [("scale", ctypes.c_float)]


class _Shared(ctypes.Structure):
    _fields_ = [("attend", _Extend), ("cu_groups", ctypes.c_void_p), ("prefix_lens", ctypes.c_void_p),
                ("groups", ctypes.c_int32), ("always", ctypes.c_int32)]


def _args(groups=1, always=1, **changes):
    a = _Extend(pool_rows=1024, tokens=4, batch=2, heads=8, kv_heads=2, dim=64, width=8, page_size=16, max_new=3,
                causal=1, window=0, dtype=1, num_cus=256, scale=0.125)
    for name, value in changes.items():
        setattr(a, name, value)
    return _Shared(attend=a, groups=groups, always=always)


@pytest.mark.parametrize("changes,message", [
    (dict(causal=0), "causal"), (dict(window=4), "window"), (dict(groups=-1), "groups"), (dict(dim=24), "divisible by 16"),
    (dict(tokens=-1), "positive extents"), (dict(num_cus=0), "positive extents"), (dict(), "tensors are missing")])
def test_c_entry_refusals(changes, message):
    """Refused on the host before any launch: these run where there is no GPU."""
    lib = _lib.load()
    lib.fgw_kv_last_error.restype = ctypes.c_char_p
    rc = lib.fgw_kv_shared(ctypes.byref(_args(**changes)), None)
    assert rc in (_lib.FGW_MHA_EINVAL, _lib.FGW_MHA_EUNSUPPORTED)
    assert message in lib.fgw_kv_last_error().decode()


def test_workspace_is_bounded_by_the_sizes():
    lib = _lib.load()
    floats, counters = ctypes.c_int64(), ctypes.c_int64()

    def need(**changes):
        assert lib.fgw_kv_shared_workspace(ctypes.byref(_args(**changes)), ctypes.byref(floats), ctypes.byref(counters)) == 0
        return floats.value

    assert need(tokens=0) == 0
    assert need(groups=0) == 0
    assert need(always=0) == 0    # 128 keys of two requests: nothing to save, each reads its own
    assert 0 < need() < 1 << 20
    # 512 rows of K/V head 0 .. 7 and as many splits as fill the card: below 64 MB.
    assert need(width=4096, tokens=64, batch=64, heads=64, kv_heads=8, dim=128, max_new=1) < 16 << 20
    # Many tokens: whole tiles, about the output's size in fp32.
    assert need(width=4096, tokens=8192, batch=8, heads=32, kv_heads=8, dim=128, max_new=2048) < 8192 * 32 * 130 * 1.2
