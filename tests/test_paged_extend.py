"""New tokens over the paged cache: the cache write and the attention with grouped heads, against
plain 64-bit forms at the sizes and masks where they can go wrong; graphs, streams, refusals."""
import ctypes
import math

import pytest
import torch

from fgw_amd import _lib
from fgw_amd.operators.mha import cache_pages, paged_extend as P
from fgw_amd.operators.mha.rotary import Rotary, apply_rotary
from tests import kv_oracle as K


def _cache(news, lens, hk, d, page, dtype, seed=0, spare=0, poison=True):
    """Pool, table and offsets; every pool row that no live token holds is NaN."""
    gen = torch.Generator().manual_seed(seed)
    width = max(1, max(-(-n // page) for n in lens)) + spare
    pages = len(lens) * width + 3
    k = torch.randn(pages * page, hk, d, generator=gen).to(dtype)
    v = torch.randn(pages * page, hk, d, generator=gen).to(dtype)
    table = torch.randperm(pages, generator=gen)[:len(lens) * width].view(len(lens), width).to(torch.int32)
    if poison:
        live = torch.zeros(pages * page, dtype=torch.bool)
        for b, n in enumerate(lens):
            pos = torch.arange(n)
            live[table[b].long()[pos // page] * page + pos % page] = True
        k[~live] = math.nan
        v[~live] = math.nan
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    return (k, v, table, torch.tensor(lens, dtype=torch.int32), torch.tensor(cu, dtype=torch.int32))


def _queries(t, hq, d, dtype, seed=5, std=2.0):
    return (torch.randn(t, hq, d, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def _compare(got, q, cache, page, label, **options):
    want, bound = K.extend_exact(q, *cache, page, **options)
    rows = int(cache[4][-1])
    err = (got.cpu().double()[:rows] - want[:rows]).abs()
    assert bool((err <= bound[:rows]).all()), (label, float((err - bound[:rows]).max()))


# (news, lens, query heads, K/V heads, D, page, causal, window)
CASES = {
    "one": ([1], [1], 1, 1, 64, 16, True, 0),
    "one_long_split": ([1], [5000], 8, 2, 128, 16, True, 0),
    "one_head_long": ([1, 1], [9001, 3], 4, 1, 64, 64, True, 0),
    "decode_ragged": ([1] * 9, [1, 2, 31, 32, 33, 500, 1024, 1025, 700], 12, 4, 128, 16, True, 0),
    "empty_requests": ([0, 1, 0, 0, 3, 0], [5, 9, 0, 40, 3, 7], 6, 3, 64, 8, True, 0),
    "no_keys": ([1, 2, 4], [0, 1, 2], 4, 2, 96, 16, True, 0),
    "no_keys_at_all": ([2, 1], [0, 0], 4, 4, 128, 16, True, 0),
    "not_causal": ([3, 1, 0], [70, 0, 33], 8, 2, 64, 32, False, 0),
    "window_one": ([1, 5], [90, 40], 4, 1, 64, 16, True, 1),
    "window_odd": ([1, 7, 40], [300, 129, 64], 8, 2, 128, 16, True, 37),
    "window_past_start": ([4, 70], [6, 70], 4, 4, 80, 48, True, 1000),
    "group_three": ([17, 1], [50, 17], 9, 3, 48, 7, True, 0),
    "group_of_forty": ([3, 1], [65, 200], 40, 1, 128, 16, True, 0),
    "one_token_pages": ([2, 9], [40, 9], 2, 2, 32, 1, True, 0),
    "dim_16": ([5, 64], [37, 64], 4, 2, 16, 16, True, 0),
    "dim_192": ([1, 33], [257, 100], 4, 2, 192, 64, True, 0),
    "dim_256": ([1, 40, 2], [513, 40, 2], 8, 1, 256, 256, True, 0),
    "many_requests": ([1] * 70, [(37 * i) % 97 for i in range(70)], 4, 2, 64, 16, True, 0),
    "many_mixed": ([(5 * i) % 4 for i in range(150)], [(29 * i) % 61 for i in range(150)], 2, 1, 128, 16, True, 0),
    "chunk": ([100, 1, 130], [400, 77, 130], 8, 2, 128, 16, True, 0),
    "chunk_page_64": ([257, 64], [900, 64], 4, 2, 128, 64, True, 0),
    "chunk_dim_64": ([300, 5], [1000, 2000], 4, 1, 64, 128, True, 0),
    "chunk_dim_96": ([200], [333], 4, 2, 96, 32, True, 0),
    "chunk_dim_32": ([200, 3], [333, 200], 4, 2, 32, 24, True, 0),
    "chunk_window": ([300, 1], [1500, 900], 4, 2, 128, 64, True, 129),
    "chunk_window_small_pages": ([300, 260], [301, 700], 4, 2, 64, 4, True, 65),
    "chunk_not_causal": ([140, 150], [90, 600], 4, 4, 128, 16, False, 0),
    "chunk_longer_than_cache": ([300, 20], [100, 0], 4, 2, 128, 16, True, 0),
    "chunk_few_rows_long": ([70], [6000], 2, 1, 128, 16, True, 0),
    "prompt": ([1000], [1000], 2, 1, 128, 64, True, 0),
    "prompt_dim_256": ([270], [400], 2, 1, 256, 64, True, 0),
    "chunk_uneven_splits": ([700, 60, 1], [2500, 2000, 900], 8, 2, 128, 16, True, 0),
    "chunk_uneven_short_cache": ([600, 300], [300, 290], 4, 1, 64, 64, True, 0),
    "wide_uneven_splits": ([330, 200], [2100, 1500], 2, 2, 192, 64, True, 0),
    "wide_window": ([300, 1], [700, 90], 4, 2, 256, 16, True, 129),
    "wide_odd_pages": ([140, 70], [300, 71], 4, 2, 192, 7, True, 0),
    "wide_split": ([200], [5000], 2, 1, 256, 64, True, 0),
    "wide_not_causal": ([150, 3], [1000, 33], 6, 2, 144, 48, False, 0),
    "wide_no_keys": ([200, 140], [100, 0], 4, 4, 256, 1, True, 0),
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("name", CASES)
def test_attention_matches_the_64_bit_form(name, dtype):
    news, lens, hq, hk, d, page, causal, window = CASES[name]
    cache = _cache(news, lens, hk, d, page, dtype)
    q = _queries(sum(news), hq, d, dtype)
    print(name, dtype, flush=True)
    kernel = P.build_extend_kernel(hq, hk, d, page, dtype, 0, is_causal=causal, window=window or None)
    got = kernel(q.cuda(), *[x.cuda() for x in cache], max(news))
    _compare(got, q, cache, page, name, causal=causal, window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 8, 9, 40, 130])
def test_counts_around_the_kernels_borders(new):
    """Rows of one request on both sides of every rule on their number, and the bound max_new loose."""
    for hq, hk in ((4, 4), (8, 2), (32, 2)):
        cache = _cache([new, 1, new + 1], [new + 200, 60, new + 1], hk, 128, 16, torch.bfloat16)
        q = _queries(2 * new + 2, hq, 128, torch.bfloat16)
        kernel = P.build_extend_kernel(hq, hk, 128, 16, "bfloat16", 0)
        for most in (new + 1, new + 1000):
            print(new, hq, hk, most, flush=True)
            _compare(kernel(q.cuda(), *[x.cuda() for x in cache], most), q, cache, 16, (new, hq, most))


@pytest.mark.gpu
def test_scale_sharp_scores_and_large_values():
    news, lens = [1, 40], [700, 90]
    cache = _cache(news, lens, 2, 128, 16, torch.float16)
    q = _queries(41, 8, 128, torch.float16, std=8.0)
    kernel = P.build_extend_kernel(8, 2, 128, 16, torch.float16, 0, softmax_scale=0.25)
    _compare(kernel(q.cuda(), *[x.cuda() for x in cache], 40), q, cache, 16, "sharp", scale=0.25)


@pytest.mark.gpu
@pytest.mark.parametrize("new,length", [(1, 300), (100, 260)])
def test_pages_outside_the_pool_read_as_zeros(new, length):
    k, v, table, lens, cu = _cache([new], [length], 2, 64, 16, torch.bfloat16)
    table[0, 2], table[0, 5], table[0, 7] = -1, 10**6, 2**31 - 1
    q = _queries(new, 4, 64, torch.bfloat16)
    kernel = P.build_extend_kernel(4, 2, 64, 16, "bfloat16", 0)
    got = kernel(q.cuda(), *[x.cuda() for x in (k, v, table, lens, cu)], new)
    _compare(got, q, (k, v, table, lens, cu), 16, "outside")


@pytest.mark.gpu
def test_lengths_past_the_table_are_clamped():
    k, v, table, lens, cu = _cache([2, 1], [64, 32], 2, 64, 16, torch.bfloat16)
    q = _queries(3, 4, 64, torch.bfloat16)
    kernel = P.build_extend_kernel(4, 2, 64, 16, "bfloat16", 0)
    bad = torch.tensor([1000, -5], dtype=torch.int32)
    got = kernel(q.cuda(), *[x.cuda() for x in (k, v, table, bad, cu)], 2)
    _compare(got, q, (k, v, table, torch.tensor([64, 0], dtype=torch.int32), cu), 16, "clamped")


@pytest.mark.gpu
def test_strided_queries_given_output_and_rows_behind_the_last_request():
    news, lens = [1, 50], [90, 50]
    cache = _cache(news, lens, 2, 128, 16, torch.bfloat16)
    fused = _queries(60, 12, 128, torch.bfloat16).cuda()  # 9 rows of padding
    fused[51:] = math.nan
    kernel = P.build_extend_kernel(8, 2, 128, 16, "bfloat16", 0)
    out = torch.full((60, 8, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    got = kernel(fused[:, 2:10], *[x.cuda() for x in cache], 50, out)
    assert got.data_ptr() == out.data_ptr() and bool((out[51:] == 7.0).all())
    _compare(out, fused[:, 2:10].cpu(), cache, 16, "strided")
    assert torch.equal(kernel(fused[:51, 2:10].contiguous(), *[x.cuda() for x in cache], 50), out[:51])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 40, 200])
def test_one_request_shorter_than_the_sizes(n):
    """Padding behind the only request of a call that is sized for a long one."""
    cache = _cache([n], [n + 130], 2, 64, 16, torch.bfloat16)
    q = _queries(260, 4, 64, torch.bfloat16)
    q[n:] = math.nan
    kernel = P.build_extend_kernel(4, 2, 64, 16, "bfloat16", 0)
    out = torch.full((260, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    _compare(kernel(q.cuda(), *[x.cuda() for x in cache], 260, out), q, cache, 16, n)
    assert bool((out[n:] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("window", [None, 100])
@pytest.mark.parametrize("most", [1, 5, 70, 141])
def test_tokens_past_the_bound_are_left(most, window):
    """max_new below a request's tokens: the ones within it as ever, the rest untouched."""
    news = [150, 3]
    cache = _cache(news, [900, 30], 2, 128, 16, torch.bfloat16)
    q = _queries(153, 8, 128, torch.bfloat16)
    kernel = P.build_extend_kernel(8, 2, 128, 16, "bfloat16", 0, window=window)
    full = kernel(q.cuda(), *[x.cuda() for x in cache], 150)
    out = torch.full((153, 8, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    kernel(q.cuda(), *[x.cuda() for x in cache], most, out)
    want, bound = K.extend_exact(q, *cache, 16, window=window or 0)
    for first, n in ((0, 150), (150, 3)):
        kept = slice(first, first + min(most, n))
        assert bool(((out[kept].cpu().double() - want[kept]).abs() <= bound[kept]).all())
        assert bool((out[first + min(most, n):first + n] == 7.0).all())
    _compare(full, q, cache, 16, "full", window=window or 0)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 300])
def test_one_token_of_many_behind_a_window(window):
    """The split of a tile follows the tokens within the bound, not all of the request's."""
    cache = _cache([5000], [6000], 1, 64, 16, torch.bfloat16)
    q = _queries(5000, 1, 64, torch.bfloat16)
    kernel = P.build_extend_kernel(1, 1, 64, 16, "bfloat16", 0, window=window)
    out = torch.full((5000, 1, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    kernel(q.cuda(), *[x.cuda() for x in cache], 1, out)
    want, bound = K.extend_exact(q, *cache, 16, window=window)
    assert bool(((out[0].cpu().double() - want[0]).abs() <= bound[0]).all()) and bool((out[1:] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("window", [599, 600, 2**31 - 1])
def test_windows_at_and_past_the_capacity(window):
    news, lens = [300, 4], [100, 600]
    cache = _cache(news, lens, 1, 64, 20, torch.bfloat16)
    q = _queries(304, 2, 64, torch.bfloat16)
    kernel = P.build_extend_kernel(2, 1, 64, 20, "bfloat16", 0, window=window)
    _compare(kernel(q.cuda(), *[x.cuda() for x in cache], 300), q, cache, 20, window, window=window)


@pytest.mark.gpu
def test_memory_that_rows_and_outputs_share():
    k, v, table, lens, cu = [x.cuda() for x in _cache([4], [40], 2, 64, 16, torch.bfloat16)]
    fused = torch.zeros(5, 10, 64, dtype=torch.bfloat16, device="cuda")
    fused.copy_(_queries(5, 10, 64, torch.bfloat16))
    q, other, across = fused[:4, :4], fused[:4, 4:8], fused[:4, 2:6]
    new_k, new_v = fused[:4, 8:10].clone(), fused[:4, 8:10].clone()
    rotary = Rotary(64)
    want = P.mha_paged_append(q, new_k, new_v, k, v, table, lens, cu, 16, rotary=rotary)
    args = (new_k, new_v, k, v, table, lens, cu, 16)
    assert torch.equal(P.mha_paged_append(q, *args, rotary=rotary, q_out=other), want)  # side by side
    for bad in (across, fused[1:5, :4]):
        with pytest.raises(ValueError, match="memory apart"):
            P.mha_paged_append(q, *args, rotary=rotary, q_out=bad)
    with pytest.raises(ValueError, match="apart from each other"):
        P.mha_paged_append(q, new_k, new_v, k, k, table, lens, cu, 16)
    kernel = P.build_extend_kernel(4, 2, 64, 16, "bfloat16", 0)
    flat = want.clone()
    with pytest.raises(ValueError, match="share memory"):
        kernel(flat, k, v, table, lens, cu, 4, flat)


@pytest.mark.gpu
def test_same_bits_on_every_run_and_alone_or_in_a_batch():
    """No result depends on an order of atomics; rows whose plan is the same do not see the batch."""
    cache = _cache([1, 1, 1], [900, 5000, 37], 2, 128, 16, torch.bfloat16)
    q = _queries(3, 8, 128, torch.bfloat16).cuda()
    dev = [x.cuda() for x in cache]
    kernel = P.build_extend_kernel(8, 2, 128, 16, "bfloat16", 0)
    first = kernel(q, *dev, 1)
    for _ in range(5):
        assert torch.equal(kernel(q, *dev, 1), first)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A pool of 2^32 bytes and more: the last pages of it."""
    page, hk, d = 64, 2, 128
    pages = (1 << 32) // (page * hk * d * 2) + 40
    k = torch.zeros(pages * page, hk, d, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    table = torch.arange(pages - 12, pages, dtype=torch.int32).view(2, 6)
    lens, cu = torch.tensor([300, 384], dtype=torch.int32), torch.tensor([0, 1, 301], dtype=torch.int32)
    q = _queries(301, 4, d, torch.bfloat16)
    new_k, new_v = _queries(301, hk, d, torch.bfloat16, 1, 1.0), _queries(301, hk, d, torch.bfloat16, 2, 1.0)
    base = (pages - 12) * page
    k[base:] = _queries(12 * page, hk, d, torch.bfloat16, 3, 1.0).cuda()
    v[base:] = _queries(12 * page, hk, d, torch.bfloat16, 4, 1.0).cuda()
    meta = [x.cuda() for x in (table, lens, cu)]
    P.mha_paged_append(q.cuda(), new_k.cuda(), new_v.cuda(), k, v, *meta, page)
    small = (k[base:].cpu(), v[base:].cpu(), table - (pages - 12), lens, cu)
    assert torch.equal(small[0][299], new_k[0]) and torch.equal(small[1][6 * page + 84:6 * page + 384], new_v[1:])
    kernel = P.build_extend_kernel(4, hk, d, page, "bfloat16", 0)
    _compare(kernel(q.cuda(), k, v, *meta, 300), q, small, page, "past 32 bits")


@pytest.mark.gpu
def test_replays_of_captured_calls_with_changing_lengths():
    """Two graphs of the same step, replayed in turn between eager work: each its own workspace."""
    hq, hk, d, page = 8, 2, 128, 16
    cache = _cache([1, 1, 1], [600, 2000, 40], hk, d, page, torch.bfloat16, poison=False)
    k, v, table, lens, cu = [x.cuda() for x in cache]
    q, k1, v1 = (_queries(3, n, d, torch.bfloat16).cuda() for n in (hq, hk, hk))
    kernel, rotary = P.build_extend_kernel(hq, hk, d, page, "bfloat16", 0), Rotary(128)

    def step():
        return kernel(P.mha_paged_append(q, k1, v1, k, v, table, lens, cu, page, rotary=rotary),
                      k, v, table, lens, cu, 1)

    step()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for i in range(4):
        lens.copy_(torch.tensor([600 - 7 * i, 2000 - 600 * i, 40 + i], dtype=torch.int32))
        q.copy_(_queries(3, hq, d, torch.bfloat16, seed=i))
        for g, out in zip(graphs, outs):
            g.replay()
            torch.cuda.synchronize()
            got = out.clone()
            assert torch.equal(got, step())


@pytest.mark.gpu
def test_streams_at_once():
    kernel = P.build_extend_kernel(8, 2, 128, 16, "bfloat16", 0)
    work = []
    for seed in range(4):
        cache = [x.cuda() for x in _cache([1, 1, 30], [3000, 800, 90], 2, 128, 16, torch.bfloat16, seed)]
        q = _queries(32, 8, 128, torch.bfloat16, seed).cuda()
        work.append((q, cache, kernel(q, *cache, 30)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    outs = []
    for _ in range(3):
        for s, (q, cache, _) in zip(streams, work):
            with torch.cuda.stream(s):
                outs.append(kernel(q, *cache, 30))
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert torch.equal(out, work[i % 4][2])


@pytest.mark.gpu
def test_one_call_entry_checks_its_metadata():
    cache = _cache([3, 1], [40, 9], 2, 64, 16, torch.float16)
    q = _queries(4, 4, 64, torch.float16)
    k, v, table, lens, cu = [x.cuda() for x in cache]
    _compare(P.mha_paged_extend(q.cuda(), k, v, table, lens, cu, 16), q, cache, 16, "one call")
    _compare(P.mha_paged_extend(q.cuda(), k, v, table, lens, cu, 16, False), q, cache, 16, "one call", causal=False)
    for bad_lens, bad_cu, message in (
            (lens + 1000, cu, "table capacity"), (lens - 50, cu, "table capacity"),
            (lens, cu + 1, "cu_seqlens"), (lens, torch.tensor([0, 3, 2], dtype=torch.int32).cuda(), "cu_seqlens"),
            (lens, torch.tensor([0, 3, 5], dtype=torch.int32).cuda(), "cu_seqlens"),
            (lens[:1], cu, "metadata"), (lens, cu[:2], "metadata"), (lens.long(), cu, "int32")):
        with pytest.raises(ValueError, match=message):
            P.mha_paged_extend(q.cuda(), k, v, table, bad_lens, bad_cu, 16)


@pytest.mark.gpu
def test_no_rows():
    k, v, table, lens, cu = [x.cuda() for x in _cache([0, 0], [9, 0], 2, 64, 16, torch.bfloat16)]
    q = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    kv = q[:, :2]
    assert P.build_extend_kernel(4, 2, 64, 16, "bfloat16", 0)(q, k, v, table, lens, cu, 1).shape == (0, 4, 64)
    assert P.mha_paged_append(q, kv, kv, k, v, table, lens, cu, 16).shape == (0, 4, 64)


# ---- the cache write ---------------------------------------------------------------------------

def _append_exact(q, k, v, kc, vc, table, lens, cu, page, rotate):
    """Pools after the write and rotated q, by a loop over the tokens."""
    kc, vc = kc.clone(), vc.clone()
    t = q.shape[0]
    pos = torch.zeros(t, dtype=torch.int64)
    dest = torch.full((t,), -1, dtype=torch.int64)
    for b in range(len(lens)):
        n = int(cu[b + 1]) - int(cu[b])
        for j in range(n):
            p = int(lens[b]) - n + j
            pos[int(cu[b]) + j] = p
            if 0 <= p < table.shape[1] * page and 0 <= int(table[b, p // page]) < kc.shape[0] // page:
                dest[int(cu[b]) + j] = int(table[b, p // page]) * page + p % page
    return pos, dest, kc, vc


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("news,lens,hq,hk,d,page,rot,interleaved,own_positions", [
    ([1], [1], 1, 1, 16, 1, 16, False, False),
    ([1] * 5, [1, 16, 17, 300, 64], 8, 2, 128, 16, 128, False, False),
    ([3, 0, 40, 1], [3, 5, 97, 12], 12, 3, 96, 48, 48, True, False),
    ([130, 2], [500, 2], 4, 4, 80, 7, 16, True, True),
    ([70, 700], [70, 900], 32, 8, 128, 64, 64, False, False),
    ([2] * 1500, [2 + i % 30 for i in range(1500)], 2, 1, 64, 16, 64, False, False),
    ([5, 9], [2, 9], 4, 2, 256, 16, 0, False, False),
])
def test_append_rotates_and_writes_the_pages(dtype, news, lens, hq, hk, d, page, rot, interleaved, own_positions):
    kc, vc, table, lens, cu = _cache(news, lens, hk, d, page, dtype)
    t = sum(news)
    fused = _queries(t + 3, hq + 2 * hk, d, dtype, std=1.0)  # three rows of padding
    fused[t:] = math.nan
    parts = fused[:, :hq], fused[:, hq:hq + hk], fused[:, hq + hk:]
    dev = fused.cuda()
    dq, dk, dv = dev[:, :hq], dev[:, hq:hq + hk], dev[:, hq + hk:]
    gkc, gvc = kc.cuda(), vc.cuda()
    q_out = torch.full((t + 3, hq, d), 7.0, dtype=dtype, device="cuda")
    pos, dest, kc, vc = _append_exact(*[x[:t] for x in parts], kc, vc, table, lens, cu, page, rot)
    if own_positions:
        pos = torch.randint(0, 9999, (t,))
    padded = torch.cat([pos, torch.zeros(3, dtype=torch.int64)]).cuda()
    rotary = Rotary(rot, interleaved=interleaved) if rot else None
    got = P.mha_paged_append(dq, dk, dv, gkc, gvc, table.cuda(), lens.cuda(), cu.cuda(), page, rotary=rotary,
                             positions=padded if own_positions else None, q_out=q_out)
    assert got.data_ptr() == q_out.data_ptr() and bool((q_out[t:] == 7.0).all())
    assert torch.equal(dev[:t].cpu(), fused[:t])
    live = dest >= 0
    vc[dest[live]] = parts[2][:t][live]
    assert torch.equal(gvc.cpu().view(torch.int16), vc.view(torch.int16))
    if rot:
        qx, qb = K.rotate_exact(parts[0][:t], pos, rot, interleaved=interleaved)
        kx, kb = K.rotate_exact(parts[1][:t], pos, rot, interleaved=interleaved)
        assert bool(((q_out[:t].cpu().double() - qx).abs() <= qb).all())
        written = gkc.cpu()[dest[live]].double()
        assert bool(((written - kx[live]).abs() <= kb[live]).all())
    else:
        assert torch.equal(q_out[:t].cpu(), parts[0][:t])
        assert torch.equal(gkc.cpu()[dest[live]], parts[1][:t][live])
    # Every other row of the pool as it was.
    kc[dest[live]] = gkc.cpu()[dest[live]]
    assert torch.equal(gkc.cpu().view(torch.int16), kc.view(torch.int16))


@pytest.mark.gpu
def test_append_leaves_out_tokens_without_a_place_and_works_in_place():
    kc, vc, table, lens, cu = _cache([2, 2, 4], [33, 20, 2], 2, 64, 16, torch.bfloat16, poison=False)
    table[0, 2], table[1, 1] = -1, 10**6  # position 32 of request 0; 18, 19 of request 1
    q, k, v = (_queries(8, n, 64, torch.bfloat16) for n in (4, 2, 2))
    gk, gv, gq = kc.cuda(), vc.cuda(), q.cuda()
    r = Rotary(64)
    got = P.mha_paged_append(gq, k.cuda(), v.cuda(), gk, gv, table.cuda(), lens.cuda(), cu.cuda(), 16, rotary=r,
                             q_out=gq)
    assert got.data_ptr() == gq.data_ptr()
    pos = torch.tensor([31, 32, 18, 19, -2, -1, 0, 1])
    assert torch.equal(gq, apply_rotary(q.cuda(), pos.cuda(), r))
    turned = apply_rotary(k.cuda(), pos.cuda(), r).cpu()
    for i, (b, p) in ((0, (0, 31)), (6, (2, 0)), (7, (2, 1))):
        row = int(table[b, p // 16]) * 16 + p % 16
        kc[row], vc[row] = turned[i], v[i]
    assert torch.equal(gk.cpu(), kc) and torch.equal(gv.cpu(), vc)


# ---- together ----------------------------------------------------------------------------------

@pytest.mark.gpu
def test_a_serving_loop():
    """Prompts in chunks, decode steps, a fork, a row freed, the pools compacted: the attention of
    every step against the 64-bit form over dense copies of what each row holds."""
    hq, hk, d, page, rows, width, pages = 8, 2, 64, 16, 6, 12, 40
    dtype = torch.bfloat16
    books = cache_pages.new_books(pages, rows, width)
    k_pool = torch.full((pages * page, hk, d), math.nan, dtype=dtype, device="cuda")
    v_pool = torch.full_like(k_pool, math.nan)
    rotary = Rotary(64, interleaved=True, scaling=dict(kind="linear", factor=2.0))
    kernel = P.build_extend_kernel(hq, hk, d, page, dtype, 0)
    dense = [(torch.empty(0, hk, d, dtype=dtype), torch.empty(0, hk, d, dtype=dtype)) for _ in range(rows)]
    gen = torch.Generator().manual_seed(11)

    def step(counts):
        counts_dev = torch.tensor(counts, dtype=torch.int32, device="cuda")
        assert cache_pages.reserve_rows(*books, counts_dev, page).tolist() == [0, 0]
        cu = torch.tensor([sum(counts[:i]) for i in range(rows + 1)], dtype=torch.int32)
        t = sum(counts)
        q, k, v = ((torch.randn(t, n, d, generator=gen)).to(dtype) for n in (hq, hk, hk))
        meta = (books.table, books.lens, cu.cuda())
        qr = P.mha_paged_append(q.cuda(), k.cuda(), v.cuda(), k_pool, v_pool, *meta, page, rotary=rotary)
        out = kernel(qr, k_pool, v_pool, *meta, max(counts))
        pos = torch.cat([torch.arange(len(dense[r][0]), len(dense[r][0]) + n) for r, n in enumerate(counts)])
        kr = apply_rotary(k.cuda(), pos.cuda(), rotary).cpu()
        for r, n in enumerate(counts):
            a = int(cu[r])
            dense[r] = (torch.cat([dense[r][0], kr[a:a + n]]), torch.cat([dense[r][1], v[a:a + n]]))
        assert books.lens.tolist() == [len(x[0]) for x in dense]
        longest = max(len(x[0]) for x in dense)
        kd, vd = torch.zeros(rows * longest, hk, d, dtype=dtype), torch.zeros(rows * longest, hk, d, dtype=dtype)
        for r, (x, y) in enumerate(dense):
            kd[r * longest:r * longest + len(x)], vd[r * longest:r * longest + len(y)] = x, y
        table = torch.arange(rows, dtype=torch.int32)[:, None]
        _compare(out, qr.cpu(), (kd, vd, table, books.lens.cpu(), cu), longest, counts)

    def ids(*x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    step([33, 70, 0, 0, 0, 0])
    step([20, 1, 48, 0, 0, 0])
    assert cache_pages.fork_rows([k_pool, v_pool], *books, ids(1, 2, 1), ids(3, 4, 5), page).tolist() == [0, 0]
    dense[3], dense[4], dense[5] = dense[1], dense[2], dense[1]
    step([1, 1, 1, 1, 1, 1])
    step([5, 0, 2, 17, 1, 30])
    cache_pages.free_rows(*books, ids(0, 5, 0), page)
    dense[0] = dense[5] = (dense[0][0][:0], dense[0][1][:0])
    step([0, 3, 1, 1, 1, 9])
    moved = int(cache_pages.compact_pages([k_pool, v_pool], *books, page))
    live = int((books.refs > 0).sum())
    assert moved > 0 and bool((books.refs[:live] > 0).all())
    step([40, 1, 1, 1, 1, 1])


# ---- refusals ----------------------------------------------------------------------------------

@pytest.mark.parametrize("args,options,message", [
    ((8, 3, 64, 16, "bfloat16", 0), {}, "multiple of the K/V heads"),
    ((0, 1, 64, 16, "bfloat16", 0), {}, "multiple of the K/V heads"),
    ((8, 2, 72, 16, "bfloat16", 0), {}, "divisible by 16"), ((8, 2, 272, 16, "bfloat16", 0), {}, "divisible by 16"),
    ((8, 2, 64, 0, "bfloat16", 0), {}, "page size"), ((8, 2, 64, 16, "float32", 0), {}, "FP16/BF16"),
    ((8, 2, 64, 16, "bfloat16", 0), dict(window=0), "window"),
    ((8, 2, 64, 16, "bfloat16", 0), dict(window=8, is_causal=False), "window"),
    ((8, 2, 64, 16, "bfloat16", 0), dict(softmax_scale=0.0), "scale"),
    ((8, 2, 64, 16, "bfloat16", 0), dict(softmax_scale=math.inf), "scale"),
])
def test_build_refusals(args, options, message):
    with pytest.raises(ValueError, match=message):
        P.build_extend_kernel(*args, **options)


class _Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("token_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class _Extend(ctypes.Structure):
    _fields_ = [("q", _Rows)] + [(n, ctypes.c_void_p) for n in (
        "out", "k_cache", "v_cache", "block_table", "cache_seqlens", "cu_seqlens", "workspace", "counters")] + [
        ("pool_rows", ctypes.c_int64)] + [(n, ctypes.c_int32) for n in (
            "tokens", "batch", "heads", "kv_heads", "dim", "width", "page_size", "max_new", "causal", "window",
            "dtype", "num_cus")] + [("scale", ctypes.c_float)]


def _extend_args(**changes):
    a = _Extend(pool_rows=1024, tokens=4, batch=2, heads=8, kv_heads=2, dim=64, width=8, page_size=16, max_new=3,
                causal=1, window=0, dtype=1, num_cus=256, scale=0.125)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("changes,message", [
    (dict(dtype=2), "FP16/BF16"), (dict(dim=24), "divisible by 16"), (dict(dim=512), "divisible by 16"),
    (dict(page_size=0), "page size"), (dict(pool_rows=1000), "whole pool pages"), (dict(width=0), "table width"),
    (dict(width=1 << 28), "31 bits"), (dict(tokens=-1), "positive extents"), (dict(batch=0), "positive extents"),
    (dict(max_new=0), "positive extents"), (dict(num_cus=0), "positive extents"),
    (dict(kv_heads=3), "multiple of the K/V heads"), (dict(window=-1), "window"),
    (dict(window=4, causal=0), "window"), (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"),
    (dict(tokens=1 << 30), "too many rows"), (dict(), "tensors are missing"),
])
def test_c_entry_refusals(changes, message):
    """Refused on the host before any launch: these run where there is no GPU."""
    lib = _lib.load()
    lib.fgw_kv_last_error.restype = ctypes.c_char_p
    rc = lib.fgw_kv_extend(ctypes.byref(_extend_args(**changes)), None)
    assert rc in (_lib.FGW_MHA_EINVAL, _lib.FGW_MHA_EUNSUPPORTED)
    assert message in lib.fgw_kv_last_error().decode()


def test_workspace_is_bounded_by_the_sizes():
    lib = _lib.load()
    floats, counters = ctypes.c_int64(), ctypes.c_int64()

    def need(**changes):
        assert lib.fgw_kv_extend_workspace(ctypes.byref(_extend_args(**changes)), ctypes.byref(floats),
                                           ctypes.byref(counters)) == 0
        return floats.value

    assert need(width=8) == 0            # 128 keys: nothing to split
    assert need(tokens=0) == 0
    assert need(width=4096, tokens=2, max_new=1) > 0
    assert need(width=4096, tokens=2, max_new=1, window=100) == 0
    assert need(width=4096, batch=64, tokens=64, max_new=1) < 64 << 20


@pytest.mark.gpu
def test_tensor_refusals():
    cache = [x.cuda() for x in _cache([2, 1], [20, 9], 2, 64, 16, torch.bfloat16)]
    k, v, table, lens, cu = cache
    q = _queries(3, 4, 64, torch.bfloat16).cuda()
    kernel = P.build_extend_kernel(4, 2, 64, 16, "bfloat16", 0)
    wide = torch.zeros(3, 4, 72, dtype=torch.bfloat16, device="cuda")
    cases = [
        ((q.half(), k, v, table, lens, cu, 2), "FP16/BF16"), ((q, k.half(), v.half(), table, lens, cu, 2), "FP16/BF16"),
        ((q[:, :2], k, v, table, lens, cu, 2), "built kernel"), ((q, k[:, :1].contiguous(), v[:, :1].contiguous(), table, lens, cu, 2), "built kernel"),
        ((q, k, v[:-16], table, lens, cu, 2), "K/V shape"), ((q, k[:-1], v[:-1], table, lens, cu, 2), "whole pool pages"),
        ((q, k, v, table.long(), lens, cu, 2), "int32"), ((q, k, v, table, lens[:1], cu, 2), "metadata"),
        ((q, k, v, table, lens, cu[:2], 2), "metadata"), ((q, k, v, table[0], lens, cu, 2), "rank-2"),
        ((q, k, v, table.t().contiguous().t(), lens, cu, 2), "contiguous"), ((q.cpu(), k, v, table, lens, cu, 2), "same GPU"),
        ((q, k, v, table, lens.cpu(), cu, 2), "same GPU"), ((q, k, v, table, lens, cu, 0), "max_new"),
        ((wide[:, :, 4:68], k, v, table, lens, cu, 2), "16-byte"), ((q, k, v, table, lens, cu, 2, q), "out must not"),
        ((q, k, v, table, lens, cu, 2, q[:2]), "out does not match"),
    ]
    for args, message in cases:
        with pytest.raises(ValueError, match=message):
            kernel(*args)
    k1, v1 = (_queries(3, 2, 64, torch.bfloat16).cuda() for _ in range(2))
    r = Rotary(64)
    for args, options, message in [
            ((q, k1[:2], v1[:2], k, v, table, lens, cu, 16), {}, "K/V shape"),
            ((q, k1, v1.half(), k, v, table, lens, cu, 16), {}, "FP16/BF16"),
            ((q, k1, v1, k, v, table, lens, cu, 0), {}, "page size"),
            ((q, k1, v1, k, v, table, lens, cu, 16), dict(positions=lens), "need a rotary"),
            ((q, k1, v1, k, v, table, lens, cu, 16), dict(positions=lens, rotary=r), "positions must be"),
            ((q, k1, v1, k, v, table, lens, cu, 16), dict(rotary=Rotary(128)), "at most the head dim"),
            ((q, k1, v1, k, v, table, lens, cu[1:], 16), {}, "metadata")]:
        with pytest.raises(ValueError, match=message):
            P.mha_paged_append(*args, **options)
