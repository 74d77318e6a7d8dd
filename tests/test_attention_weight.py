"""Attention weight of cached keys: against the 64-bit form at the sizes and masks where it can go wrong,
what has to stay as it was, not-finite values, graphs, refusals."""
import ctypes
import math

import pytest
import torch

from fgw_amd import _lib
from fgw_amd.operators.mha import eviction as E
from tests import eviction_oracle as X


def _cache(news, lens, hk, d, page, dtype, seed=0, spare=0):
    """Keys, table and offsets; every pool row that no live token holds is NaN."""
    gen = torch.Generator().manual_seed(seed)
    width = max(1, max(-(-n // page) for n in lens)) + spare
    pages = len(lens) * width + 3
    k = torch.randn(pages * page, hk, d, generator=gen).to(dtype)
    table = torch.randperm(pages, generator=gen)[:len(lens) * width].view(len(lens), width).to(torch.int32)
    live = torch.zeros(pages * page, dtype=torch.bool)
    for b, n in enumerate(lens):
        pos = torch.arange(n)
        live[table[b].long()[pos // page] * page + pos % page] = True
    k[~live] = math.nan
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    return k, table, torch.tensor(lens, dtype=torch.int32), torch.tensor(cu, dtype=torch.int32)


def _queries(t, hq, d, dtype, seed=5, std=2.0):
    return (torch.randn(t, hq, d, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def _scores(cache, hk, page, spare=0, seed=9):
    """Running sums; entries that no old key has are NaN (new keys begin anew, later ones are left)."""
    k, table, lens, cu = cache
    b, s = table.shape[0], table.shape[1] * page + spare
    x = torch.rand(b, hk, s, generator=torch.Generator().manual_seed(seed)) * 3
    for i in range(b):
        x[i, :, max(0, int(lens[i]) - int(cu[i + 1] - cu[i])):] = math.nan
    return x


def _check(got, scores, q, cache, page, last, label, **options):
    want, bound = X.weights_exact(scores, q, *cache, page, last, **options)
    got = got.cpu().double()
    both = torch.isnan(want)
    assert torch.equal(torch.isnan(got), both), label
    err = (got - want).abs()[~both]
    assert bool((err <= bound[~both]).all()), (label, float((err - bound[~both]).max()))


def _run(scores, q, cache, page, last, **options):
    dev = scores.cuda()
    E.add_weights(dev, q.cuda(), *[x.cuda() for x in cache], page, last, **options)
    return dev


# (news, lens, query heads, K/V heads, D, page, last, decay)
CASES = {
    "one": ([1], [1], 1, 1, 64, 16, 1, 1.0),
    "one_split": ([1], [5000], 8, 2, 128, 16, 1, 1.0),
    "one_head_long": ([1, 1], [9001, 3], 4, 1, 64, 64, 1, 0.5),
    "decode_ragged": ([1] * 9, [1, 2, 31, 32, 33, 500, 1024, 1025, 700], 12, 4, 128, 16, 1, 1.0),
    "empty_requests": ([0, 1, 0, 0, 3, 0], [5, 9, 0, 40, 3, 7], 6, 3, 64, 8, 4, 1.0),
    "no_keys": ([1, 2, 4], [0, 1, 2], 4, 2, 96, 16, 4, 1.0),
    "no_keys_at_all": ([2, 1], [0, 0], 4, 4, 128, 16, 2, 1.0),
    "forget": ([1, 2], [90, 400], 8, 2, 64, 32, 2, 0.0),
    "last_of_several": ([9, 3, 1], [200, 30, 77], 4, 2, 128, 16, 2, 0.9),
    "sixteen_rows": ([4, 4], [300, 1500], 8, 2, 80, 48, 4, 1.0),
    "seventeen_rows": ([17, 1], [50, 900], 3, 3, 48, 7, 17, 1.0),
    "group_of_sixteen": ([1, 1], [700, 65], 16, 1, 128, 16, 1, 1.0),
    "group_of_forty": ([3, 1], [65, 200], 40, 1, 128, 16, 3, 1.0),
    "one_token_pages": ([2, 9], [40, 9], 2, 2, 32, 1, 9, 1.0),
    "dim_16": ([5, 64], [37, 64], 4, 2, 16, 16, 64, 1.0),
    "dim_192": ([1, 2], [257, 1000], 4, 2, 192, 64, 2, 1.0),
    "dim_192_rows": ([33, 40], [257, 100], 4, 2, 192, 64, 40, 1.0),
    "dim_256": ([1, 3, 2], [513, 3000, 2], 4, 1, 256, 256, 3, 1.0),
    "dim_256_rows": ([70, 40, 2], [513, 3000, 2], 8, 1, 256, 16, 70, 0.5),
    "many_requests": ([1] * 70, [(37 * i) % 97 for i in range(70)], 4, 2, 64, 16, 1, 1.0),
    "many_mixed": ([(5 * i) % 4 for i in range(150)], [(29 * i) % 61 for i in range(150)], 2, 1, 128, 16, 3, 1.0),
    "many_mixed_rows": ([(5 * i) % 24 for i in range(150)], [(29 * i) % 161 for i in range(150)], 2, 1, 64, 16, 23, 1.0),
    "window": ([500, 31, 1], [700, 4000, 90], 16, 4, 96, 48, 32, 0.5),
    "window_long_split": ([40], [9000], 8, 2, 128, 64, 32, 1.0),
    "prompt": ([300, 129], [300, 129], 8, 2, 128, 64, 300, 1.0),
    "prompt_parts": ([700, 600, 3], [700, 900, 40], 4, 1, 64, 16, 10**9, 1.0),
    "prompt_parts_large_group": ([150, 260], [2100, 260], 24, 3, 128, 16, 260, 0.25),
    "prompt_parts_dim_256": ([530], [600], 4, 2, 256, 64, 530, 1.0),
    "parts_of_256": ([700, 260, 257], [700, 900, 300], 2, 2, 128, 16, 700, 1.0),
    "parts_of_512": ([1400] * 3, [1400, 3000 + 200, 1500], 4, 2, 64, 64, 1400, 1.0),
    "many_requests_rows": ([17 + i % 60 for i in range(130)], [17 + i % 60 + (41 * i) % 700 for i in range(130)], 8, 1, 64, 16, 70, 0.5),
    "dim_160_rows": ([90, 300], [1300, 300], 6, 2, 160, 32, 200, 1.0),
    "kept_33_rows": ([33, 40, 1, 32], [33, 3000, 50, 700], 4, 4, 128, 16, 40, 0.5),
    "kept_48_rows": ([12, 3, 12], [5000, 90, 12], 8, 2, 64, 64, 12, 1.0),
    "kept_49_rows": ([49, 7], [900, 90], 2, 2, 96, 48, 49, 1.0),
    "kept_64_rows_wide": ([16, 2, 9], [2500, 90, 9], 8, 2, 256, 64, 16, 1.0),
    "kept_65_rows_wide": ([65, 3], [300, 90], 2, 2, 160, 16, 65, 1.0),
    "longer_than_cache": ([300, 20], [100, 7], 4, 2, 128, 16, 300, 1.0),
    "parts_longer_than_cache": ([1500], [700], 2, 1, 64, 16, 1500, 1.0),
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("name", CASES)
def test_matches_the_64_bit_form(name, dtype):
    news, lens, hq, hk, d, page, last, decay = CASES[name]
    cache = _cache(news, lens, hk, d, page, dtype)
    q = _queries(sum(news), hq, d, dtype)
    scores = _scores(cache, hk, page, spare=len(news) % 3)
    print(name, dtype, flush=True)
    got = _run(scores, q, cache, page, last, decay=decay)
    _check(got, scores, q, cache, page, last, name, decay=decay)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 4, 5, 8, 9, 32, 33, 130, 257])
def test_counts_around_the_kernels_borders(new):
    for hq, hk in ((4, 4), (8, 2), (32, 2)):
        cache = _cache([new, 1, new + 1], [new + 200, 60, new + 1], hk, 128, 16, torch.bfloat16)
        q = _queries(2 * new + 2, hq, 128, torch.bfloat16)
        scores = _scores(cache, hk, 16)
        for last in (new, new + 1, new + 1000):
            print(new, hq, hk, last, flush=True)
            _check(_run(scores, q, cache, 16, last), scores, q, cache, 16, last, (new, hq, last))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 3, 40])
def test_weights_of_a_row_sum_to_one(new):
    """Each row adds 1 in all, whatever its scores: large ones, a scale of the caller's."""
    cache = _cache([new], [3000], 1, 128, 16, torch.float16)
    q = _queries(new, 4, 128, torch.float16, std=16.0)
    scores = torch.zeros(1, 1, cache[1].shape[1] * 16)
    got = _run(scores, q, cache, 16, new, softmax_scale=0.5)
    _check(got, scores, q, cache, 16, new, "sharp", scale=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [2, 40])
def test_strides_padding_and_pages_outside_the_pool(new):
    k, table, lens, cu = _cache([new, 1], [new + 250, 90], 2, 64, 16, torch.bfloat16, spare=2)
    table[0, 3], table[1, 2] = -1, 10**6
    cache = (k, table, lens, cu)
    fused = _queries(new + 4, 8, 64, torch.bfloat16)
    fused[new + 1:] = math.nan
    scores = _scores(cache, 2, 16, spare=5)
    dev = scores.cuda()
    E.add_weights(dev, fused.cuda()[:, 2:6], *[x.cuda() for x in cache], 16, new)
    _check(dev, scores, fused[:new + 1, 2:6], cache, 16, new, "padded")


@pytest.mark.gpu
@pytest.mark.parametrize("new", [2, 60])
@pytest.mark.parametrize("where", ["query", "key"])
def test_nan_reaches_the_keys_that_its_rows_see(new, where):
    k, table, lens, cu = _cache([new, new], [new + 300, new + 40], 2, 128, 16, torch.bfloat16)
    q = _queries(2 * new, 4, 128, torch.bfloat16)
    if where == "query":
        q[0, 1, 3] = math.nan                       # first new token of request 0, K/V head 0
    else:
        at = 300 + new - 1                          # the last token's own key: seen by it alone
        k[int(table[0, at // 16]) * 16 + at % 16, 0, 7] = math.nan
    cache = (k, table, lens, cu)
    scores = torch.zeros(2, 2, table.shape[1] * 16)
    got = _run(scores, q, cache, 16, new).cpu()
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[0, 0, :301 if where == "query" else 300 + new] = True
    assert torch.equal(torch.isnan(got), bad)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 50])
def test_captured_and_replayed(new):
    """One graph, with eager calls between the replays, other lengths each time; and the same bits on every run."""
    hq, hk, d, page = 8, 2, 128, 16
    caches = [_cache([new] * 3, [new + n for n in lens], hk, d, page, torch.bfloat16, seed=i, spare=s)
              for i, (lens, s) in enumerate([((500, 3, 90), 1), ((10, 512, 0), 0), ((300, 301, 302), 14)])]
    width = max(c[1].shape[1] for c in caches)
    rows = max(c[0].shape[0] for c in caches)
    caches = [(torch.cat([k, torch.zeros(rows - k.shape[0], hk, d, dtype=k.dtype)]),
               torch.cat([t, torch.full((3, width - t.shape[1]), -1, dtype=torch.int32)], 1), n, cu) for k, t, n, cu in caches]
    q = _queries(3 * new, hq, d, torch.bfloat16)
    dev, qd = [x.cuda() for x in caches[0]], q.cuda()
    scores = torch.zeros(3, hk, width * page, device="cuda")
    for _ in range(2):
        E.add_weights(scores, qd, *dev, page, new)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        E.add_weights(scores, qd, *dev, page, new)
    for turn in (0, 1, 2, 1, 0):
        for x, y in zip(dev, caches[turn]):
            x.copy_(y)
        start = _scores(caches[turn], hk, page)
        eager = start.cuda()
        E.add_weights(eager, qd, *dev, page, new)
        scores.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        _check(scores, start, q, caches[turn], page, new, turn)
        assert torch.equal(scores.view(torch.int32), eager.view(torch.int32)), turn


@pytest.mark.gpu
def test_a_table_far_wider_than_the_pool():
    """Few rows, and places for more scores than the pool has bytes."""
    k, table, lens, cu = _cache([2, 1, 2, 0], [700, 90, 2, 40], 2, 64, 64, torch.bfloat16)
    wide = torch.full((4, 17000), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    cache, q = (k, wide, lens, cu), _queries(5, 8, 64, torch.bfloat16)
    scores = _scores(cache, 2, 64)
    _check(_run(scores, q, cache, 64, 2, decay=0.5), scores, q, cache, 64, 2, "wide", decay=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [2, 60])
def test_a_pool_past_four_gib(new):
    """Rows whose offsets pass 32 bits: the same bits as in a small pool."""
    page, large = 64, 50000  # pages of 128 KB
    k, table, lens, cu = [x.cuda() for x in _cache([new, 1], [700, 90], 8, 128, page, torch.bfloat16)]
    q = _queries(new + 1, 16, 128, torch.bfloat16).cuda()
    start = torch.rand(2, 8, table.shape[1] * page, device="cuda")
    near, far = start.clone(), start.clone()
    E.add_weights(near, q, k, table, lens, cu, page, new)
    pool = torch.zeros(large * page, 8, 128, dtype=torch.bfloat16, device="cuda")
    pool[-k.shape[0]:] = k
    E.add_weights(far, q, pool, table + (large - k.shape[0] // page), lens, cu, page, new)
    assert torch.equal(near, far)


@pytest.mark.gpu
def test_two_streams_at_once():
    cache = _cache([1] * 4, [3000, 5, 900, 2], 2, 128, 16, torch.bfloat16)
    dev = [x.cuda() for x in cache]
    q = [_queries(4, 8, 128, torch.bfloat16, seed=s) for s in (1, 2)]
    qd, start = [x.cuda() for x in q], _scores(cache, 2, 16)
    streams = [torch.cuda.Stream() for _ in q]
    sums = [start.cuda() for _ in q]
    torch.cuda.synchronize()
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            E.add_weights(sums[i], qd[i], *dev, 16, 1)
    torch.cuda.synchronize()
    for i in range(2):
        _check(sums[i], start, q[i], cache, 16, 1, i)


@pytest.mark.gpu
def test_refusals():
    k, table, lens, cu = [x.cuda() for x in _cache([2, 1], [20, 9], 2, 64, 16, torch.bfloat16)]
    q = _queries(3, 4, 64, torch.bfloat16).cuda()
    scores = torch.zeros(2, 2, 32, device="cuda")
    buffer = torch.zeros(4096, device="cuda")
    for args, options, message in [
            ((scores.half(), q, k, table, lens, cu, 16, 1), {}, "FP32 scores"),
            ((scores[0], q, k, table, lens, cu, 16, 1), {}, "FP32 scores"),
            ((scores[:, :1], q, k, table, lens, cu, 16, 1), {}, "FP32 scores"),
            ((scores[:, :, :31].contiguous(), q, k, table, lens, cu, 16, 1), {}, "place for every key"),
            ((scores[:, :, ::2], q, k, table, lens, cu, 8, 1), {}, "contiguous"),
            ((scores.cpu(), q, k, table, lens, cu, 16, 1), {}, "same GPU"),
            ((scores, q.cpu(), k, table, lens, cu, 16, 1), {}, "same GPU"),
            ((scores, q.half(), k, table, lens, cu, 16, 1), {}, "FP16/BF16"),
            ((scores, q, k[:, :, :48].contiguous(), table, lens, cu, 16, 1), {}, "K/V shape"),
            ((scores, q[:, :3], k, table, lens, cu, 16, 1), {}, "multiple of the K/V heads"),
            ((scores, q, k[:-1], table, lens, cu, 16, 1), {}, "whole pool pages"),
            ((scores, q, k, table.long(), lens, cu, 16, 1), {}, "int32"),
            ((scores, q, k, table, lens, cu[1:], 16, 1), {}, "metadata"),
            ((scores, q, k, table, lens, cu, 16, 0), {}, "tokens that count"),
            ((scores, q, k, table, lens, cu, 16, 1), dict(decay=-1.0), "decay"),
            ((scores, q, k, table, lens, cu, 16, 1), dict(decay=math.inf), "decay"),
            ((scores, q, k, table, lens, cu, 16, 1), dict(softmax_scale=0.0), "scale"),
            ((buffer[:128].view(2, 2, 32), q, k, table, buffer[4:6].view(torch.int32), cu, 16, 1), {}, "share memory"),
            ((scores.clone().requires_grad_(), q, k, table, lens, cu, 16, 1), {}, "requires a gradient")]:
        with pytest.raises(ValueError, match=message):
            E.add_weights(*args, **options)


class _Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("token_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class _Weights(ctypes.Structure):
    _fields_ = [("q", _Rows), ("scores", ctypes.c_void_p), ("scores_stride", ctypes.c_int64)] + [
        (n, ctypes.c_void_p) for n in ("k_cache", "block_table", "cache_seqlens", "cu_seqlens", "workspace")] + [
        ("pool_rows", ctypes.c_int64)] + [(n, ctypes.c_int32) for n in (
            "tokens", "batch", "heads", "kv_heads", "dim", "width", "page_size", "last", "dtype", "num_cus")] + [
        ("scale", ctypes.c_float), ("decay", ctypes.c_float)]


def _args(**changes):
    a = _Weights(scores_stride=128, pool_rows=1024, tokens=4, batch=2, heads=8, kv_heads=2, dim=64, width=8,
                 page_size=16, last=3, dtype=1, num_cus=256, scale=0.125, decay=1.0)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("changes,message", [
    (dict(last=0), "tokens that count"), (dict(dtype=2), "FP16/BF16"), (dict(dim=24), "divisible by 16"),
    (dict(scores_stride=127), "place for every key"), (dict(decay=-0.5), "decay"), (dict(decay=math.nan), "decay"),
    (dict(tokens=-1), "positive extents"), (dict(kv_heads=3), "multiple of the K/V heads"),
    (dict(width=1 << 26, scores_stride=1 << 31, batch=1 << 16), "too many rows"), (dict(), "tensors are missing")])
def test_c_entry_refusals(changes, message):
    """Refused on the host before any launch: these run where there is no GPU."""
    lib = _lib.load()
    lib.fgw_kv_last_error.restype = ctypes.c_char_p
    rc = lib.fgw_kv_weights(ctypes.byref(_args(**changes)), None)
    assert rc in (_lib.FGW_MHA_EINVAL, _lib.FGW_MHA_EUNSUPPORTED)
    assert message in lib.fgw_kv_last_error().decode()


def test_workspace_follows_the_sizes():
    lib = _lib.load()
    lib.fgw_kv_weights_workspace.restype = ctypes.c_int64

    def need(**changes):
        return lib.fgw_kv_weights_workspace(ctypes.byref(_args(**changes)))

    assert need(tokens=0) == 0
    assert need(last=0) < 0
    # A decode step keeps the scores of its rows, and little beside them.
    kept = 64 * 8 * 4 * 4096
    assert kept <= need(tokens=64, batch=64, heads=32, kv_heads=8, last=1, width=256, scores_stride=4096) < kept * 1.02
    # A table with places for more scores than the pool has bytes: two passes, which keep none.
    wide = dict(tokens=64, batch=64, heads=32, kv_heads=8, last=1, width=8192, scores_stride=131072, page_size=16)
    assert need(**wide, pool_rows=1 << 22) > 64 * 8 * 4 * 131072 > (64 << 20) > need(**wide, pool_rows=1 << 16)
    # Prompts: statistics of every row, and sums of each part of 1024 of them for each key.
    assert need(tokens=8192, batch=2, heads=32, kv_heads=8, last=4096, width=256, scores_stride=4096) < 2 * 34 * 8 * 4096
