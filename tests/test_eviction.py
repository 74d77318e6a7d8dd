"""Rows shortened to the keys with the most attention weight: books, pools and sums bit by bit against the
host's, at the sizes where choosing and moving can go wrong; a decoding loop on a bounded cache; refusals."""
import ctypes
import math

import pytest
import torch

from fgw_amd import _lib
from fgw_amd.operators.mha import cache_pages, eviction as E, paged_extend as P, shared_prefix as S
from fgw_amd.operators.mha.rotary import Rotary, apply_rotary
from tests import eviction_oracle as X, kv_oracle as K


def _state(lens, page, width, pages, heads, dims, dtype, layers=1, seed=0, shared=0, kind="ties"):
    """(k_pools, v_pools, scores, refs, table, lens) on the CPU; odd rows share the first `shared` pages of
    the row before."""
    gen = torch.Generator().manual_seed(seed)
    ids = torch.randperm(pages, generator=gen).tolist()
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    for r, n in enumerate(lens):
        for j in range(-(-n // page)):
            table[r, j] = table[r - 1, j] if r % 2 and j < shared else ids.pop()
            refs[int(table[r, j])] += 1
    k_dim, v_dim = dims

    def pools(d):
        return [torch.randn(pages * page, heads, d, generator=gen).to(dtype) for _ in range(layers)]

    k, v = pools(k_dim), pools(v_dim)
    scores = [torch.rand(len(lens), heads, width * page + 3, generator=gen) for _ in range(layers)]
    for x in scores:
        if kind == "ties":
            x.copy_(torch.round(x * 6) / 6)
        elif kind == "equal":
            x.fill_(0.25)
        elif kind == "mixed":  # signs, zeros of both signs, infinities, NaN, tiny and huge ones
            x.copy_((x - 0.5) * 10.0 ** torch.randint(-45, 38, x.shape, generator=gen).float())
            pick = torch.randint(0, 9, x.shape, generator=gen)
            for i, value in enumerate((0.0, -0.0, math.inf, -math.inf, math.nan)):
                x[pick == i] = value
    return k, v, scores, refs, table, torch.tensor(lens, dtype=torch.int32)


def _bits(x):
    return x.view({1: torch.int8, 2: torch.int16, 4: torch.int32}[x.element_size()])


def _evict(state, keep, page, **options):
    """One call against the host's: everything bit by bit, what no row holds any more too."""
    k, v, scores, refs, table, lens = state
    keep = torch.tensor(keep, dtype=torch.int32)
    dev = [[x.cuda() for x in part] for part in (k, v, scores)] + [x.cuda() for x in (refs, table, lens)]
    status = E.evict_rows(*dev, keep.cuda(), page, **options)
    want = X.evict_exact(k, v, scores, refs, table, lens, keep, page, **options)
    assert status.tolist() == want
    for name, x, y in (("refs", dev[3], refs), ("table", dev[4], table), ("lens", dev[5], lens)):
        assert torch.equal(x.cpu(), y), name
    for name, got, host in (("scores", dev[2], scores), ("k", dev[0], k), ("v", dev[1], v)):
        for i, (x, y) in enumerate(zip(got, host)):
            assert torch.equal(_bits(x.cpu()), _bits(y)), (name, i)
    return want


# name: (lens, keep, page, width, heads, (K dim, V dim), layers, first, recent, shared pages, scores)
CASES = {
    "one_of_two": ([2], [1], 16, 1, 1, (64, 64), 1, 0, 0, 0, "ties"),
    "one_dropped": ([100], [99], 16, 8, 2, (64, 64), 1, 4, 8, 0, "ties"),
    "to_nothing": ([33, 40], [0, 20], 16, 4, 2, (64, 64), 2, 0, 0, 0, "ties"),
    "nothing_to_choose": ([60, 61], [20, 20], 16, 4, 2, (64, 64), 1, 12, 8, 0, "ties"),
    "all_chosen": ([60, 17], [30, 9], 8, 8, 3, (64, 64), 2, 0, 0, 0, "ties"),
    "first_past_a_page": ([90, 90], [60, 47], 16, 6, 2, (64, 64), 1, 40, 5, 0, "ties"),
    "first_to_a_page": ([90, 90], [32, 33], 16, 6, 2, (64, 64), 1, 32, 0, 0, "ties"),
    "rows_that_stay": ([50, 50, 0, 50, 50], [-1, 50, 0, 51, 20], 16, 4, 2, (64, 64), 1, 2, 3, 0, "ties"),
    "shared_pages": ([100, 120, 64, 70], [70, 60, 20, 69], 16, 8, 2, (64, 64), 2, 0, 4, 3, "ties"),
    "shared_and_kept_whole": ([100, 120], [70, 60], 16, 8, 2, (64, 64), 1, 48, 4, 3, "ties"),
    "equal_scores": ([500], [123], 16, 32, 2, (32, 32), 1, 5, 7, 0, "equal"),
    "mixed_scores": ([800, 300], [300, 299], 16, 50, 3, (32, 32), 1, 1, 1, 0, "mixed"),
    "one_token_pages": ([40, 9], [11, 8], 1, 40, 2, (16, 32), 1, 3, 2, 0, "ties"),
    "odd_pages_and_dims": ([200, 77], [90, 33], 7, 30, 5, (80, 16), 3, 9, 2, 0, "ties"),
    "wide_heads": ([150], [70], 64, 3, 8, (256, 128), 1, 4, 16, 0, "ties"),
    "many_rows": ([(37 * i) % 60 for i in range(130)], [(11 * i) % 40 - 1 for i in range(130)], 8, 8, 1, (32, 32), 1, 2, 3, 0, "ties"),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", CASES)
def test_matches_the_host(name):
    lens, keep, page, width, heads, dims, layers, first, recent, shared, kind = CASES[name]
    pages = 2 * sum(-(-n // page) for n in lens) + 5
    print(name, flush=True)
    _evict(_state(lens, page, width, pages, heads, dims, torch.bfloat16, layers, shared=shared, kind=kind), keep, page,
           first=first, recent=recent)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32, torch.int8])
def test_types_of_the_pools(dtype):
    _evict(_state([300], 16, 20, 60, 2, (32, 48), dtype), [130], 16, first=3, recent=9)


@pytest.mark.gpu
@pytest.mark.parametrize("length,keep", [(1023, 500), (1025, 1024), (16384, 8000), (16386, 16385), (16400, 3), (40000, 20001)])
def test_lengths_around_what_a_program_holds(length, keep):
    """The sums of up to 16384 candidates stay in registers, more are read again."""
    state = _state([length], 64, -(-length // 64), 2 * -(-length // 64) + 1, 1, (16, 16), torch.float16, kind="ties")
    _evict(state, [keep], 64)


@pytest.mark.gpu
def test_more_layers_than_one_launch_takes():
    _evict(_state([90, 50, 20], 16, 6, 30, 2, (16, 16), torch.float16, layers=35, shared=1), [40, 20, 19], 16, first=2, recent=4)


@pytest.mark.gpu
@pytest.mark.parametrize("free", [0, 1, 4, 5, 6, 20])
def test_want_of_pages(free):
    """Rows in order; one that finds too few pages stays whole, and so do those behind it that need any."""
    lens, keep = [100, 90, 64, 80], [60, 16, 0, 33]   # need 4, 1, 0 and 3 pages
    live = sum(-(-n // 16) for n in lens)
    state = _state(lens, 16, 8, live + free, 2, (16, 16), torch.float16)
    short, _ = _evict(state, keep, 16)
    assert short == {0: 3, 1: 3, 4: 2, 5: 1, 6: 1, 20: 0}[free]


@pytest.mark.gpu
def test_counts_below_what_has_to_stay():
    state = _state([50, 50, 10, 50], 16, 4, 40, 2, (16, 16), torch.float16)
    assert _evict(state, [11, 12, 5, 2**31 - 1], 16, first=4, recent=8) == [0, 2]
    state = _state([50], 16, 4, 40, 2, (16, 16), torch.float16)
    assert _evict(state, [30], 16, first=2**31 - 1, recent=2**31 - 1) == [0, 1]


@pytest.mark.gpu
def test_pages_outside_the_pool_move_as_zeros():
    page, zeros = 16, 39
    bad = _state([90, 70], page, 8, 40, 2, (64, 32), torch.bfloat16, kind="")
    bad[3][zeros] = 3  # held, and all zeros
    for x in bad[0] + bad[1]:
        x[zeros * page:] = 0.0
    assert not (bad[4] == zeros).any()
    good = [[x.clone() for x in part] for part in bad[:3]] + [x.clone() for x in bad[3:]]
    for r, j, value in ((0, 1, -1), (0, 4, 40), (1, 0, 2**31 - 1)):
        bad[3][int(bad[4][r, j])] -= 1
        good[3][int(good[4][r, j])] -= 1
        bad[4][r, j], good[4][r, j] = value, zeros
    keep = torch.tensor([50, 33], dtype=torch.int32)
    dev = [[x.cuda() for x in part] for part in bad[:3]] + [x.cuda() for x in bad[3:]]
    assert E.evict_rows(*dev, keep.cuda(), page, first=2, recent=7).tolist() == [0, 0]
    assert X.evict_exact(*good, keep, page, first=2, recent=7) == [0, 0]
    good[3][zeros] = 3
    for x, y in zip(dev[0] + dev[1] + dev[2] + dev[3:], good[0] + good[1] + good[2] + good[3:]):
        assert torch.equal(_bits(x.cpu()), _bits(y))


@pytest.mark.gpu
def test_pools_past_four_gib():
    """Rows whose offsets pass 32 bits: the same bits as in a small pool."""
    page, small, large = 64, 30, 50000  # pages of 128 KB
    state = _state([700, 512], page, 12, small, 8, (128, 128), torch.bfloat16)
    keep = torch.tensor([300, 512 - 65], dtype=torch.int32).cuda()
    near = [[x.cuda() for x in part] for part in state[:3]] + [x.cuda() for x in state[3:]]
    want = E.evict_rows(*near, keep, page, first=70, recent=9)
    far = [[torch.zeros(large * page, 8, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]]
    for x, y in zip(far[0], (state[0][0], state[1][0])):
        x[(large - small) * page:] = y.cuda()
    scores = [state[2][0].cuda()]
    refs = torch.ones(large, dtype=torch.int32, device="cuda")
    refs[large - small:] = state[3].cuda()
    table, lens = torch.where(state[4] < 0, -1, state[4] + large - small).to(torch.int32).cuda(), state[5].cuda()
    got = E.evict_rows(far[0][:1], far[0][1:], scores, refs, table, lens, keep, page, first=70, recent=9)
    assert got.tolist() == want.tolist() == [0, 0]
    assert torch.equal(refs[large - small:], near[3]) and torch.equal(lens, near[5])
    assert torch.equal(table, torch.where(near[4] < 0, -1, near[4] + large - small))
    assert torch.equal(scores[0], near[2][0])
    for x, y in zip(far[0], (near[0][0], near[1][0])):
        assert torch.equal(x[(large - small) * page:], y)


@pytest.mark.gpu
def test_captured_and_replayed():
    """One graph, with eager calls between its replays, from other books each time."""
    page, width, heads = 16, 8, 2
    lens = [[100, 120, 30], [128, 5, 64], [17, 90, 90]]
    keeps = [[50, -1, 29], [60, 3, 0], [16, 20, 89]]
    states = [_state(x, page, width, 60, heads, (64, 64), torch.bfloat16, 2, seed=i) for i, x in enumerate(lens)]

    def flat(state):
        return state[0] + state[1] + state[2] + list(state[3:])

    dev = [[x.cuda() for x in part] for part in states[0][:3]] + [x.cuda() for x in states[0][3:]]
    keep = torch.tensor(keeps[0], dtype=torch.int32, device="cuda")
    for _ in range(2):
        E.evict_rows(*dev, keep, page, first=2, recent=3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        status = E.evict_rows(*dev, keep, page, first=2, recent=3)
    for turn in (0, 1, 2, 1):
        for x, y in zip(dev[0] + dev[1] + dev[2] + dev[3:], flat(states[turn])):
            x.copy_(y)
        keep.copy_(torch.tensor(keeps[turn], dtype=torch.int32))
        host = [[x.clone() for x in part] for part in states[turn][:3]] + [x.clone() for x in states[turn][3:]]
        _evict([[x.clone() for x in part] for part in host[:3]] + [x.clone() for x in host[3:]], keeps[turn], page, first=2, recent=3)
        graph.replay()
        torch.cuda.synchronize()
        want = X.evict_exact(*host, torch.tensor(keeps[turn]), page, first=2, recent=3)
        assert status.tolist() == want
        for x, y in zip(dev[0] + dev[1] + dev[2] + dev[3:], host[0] + host[1] + host[2] + host[3:]):
            assert torch.equal(_bits(x.cpu()), _bits(y)), turn


@pytest.mark.gpu
def test_versions_move():
    state = _state([50], 16, 4, 20, 2, (64, 64), torch.bfloat16)
    dev = [[x.cuda() for x in part] for part in state[:3]] + [x.cuda() for x in state[3:]]
    flat = dev[0] + dev[1] + dev[2] + dev[3:]
    before = [x._version for x in flat]
    E.evict_rows(*dev, torch.tensor([20], dtype=torch.int32, device="cuda"), 16)
    assert all(x._version > n for x, n in zip(flat, before))


# ---- together ----------------------------------------------------------------------------------

@pytest.mark.gpu
def test_samples_of_one_prompt_on_a_bounded_cache():
    """A prompt, forked; its samples decode over the shared prefix while the weight of every key is added up;
    rows past their budget are cut. Attention and sums of every step against the 64-bit forms over dense
    copies of what each row and head holds."""
    hq, hk, d, page, rows, width, pages = 8, 2, 64, 16, 5, 16, 90
    dtype = torch.bfloat16
    books = cache_pages.new_books(pages, rows, width)
    k_pool, v_pool = (torch.zeros(pages * page, hk, d, dtype=dtype, device="cuda") for _ in range(2))
    scores = torch.zeros(rows, hk, width * page, device="cuda")
    rotary = Rotary(64)
    kernel = S.build_shared_kernel(hq, hk, d, page, dtype, 0)
    gen = torch.Generator().manual_seed(3)
    dense = [[torch.zeros(0, hk, d, dtype=dtype), torch.zeros(0, hk, d, dtype=dtype)] for _ in range(rows)]
    position = [0] * rows   # of the next token: no longer the length, once keys were dropped

    def ints(*x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    def step(counts, first, prefixes, budget=None):
        assert cache_pages.reserve_rows(*books, ints(*counts), page).tolist() == [0, 0]
        cu = torch.tensor([sum(counts[:i]) for i in range(rows + 1)], dtype=torch.int32)
        t = sum(counts)
        q, k, v = (torch.randn(t, n, d, generator=gen).to(dtype) for n in (hq, hk, hk))
        pos = torch.cat([torch.arange(position[r], position[r] + n) for r, n in enumerate(counts)])
        meta = (books.table, books.lens, cu.cuda())
        qr = P.mha_paged_append(q.cuda(), k.cuda(), v.cuda(), k_pool, v_pool, *meta, page, rotary=rotary,
                                positions=pos.cuda())
        out = kernel(qr, k_pool, v_pool, *meta, ints(*first), ints(*prefixes), max(counts))
        before = scores.cpu()
        E.add_weights(scores, qr, k_pool, *meta, page, max(counts))
        kr = apply_rotary(k.cuda(), pos.cuda(), rotary).cpu()
        for r, n in enumerate(counts):
            a = int(cu[r])
            dense[r] = [torch.cat([dense[r][0], kr[a:a + n]]), torch.cat([dense[r][1], v[a:a + n]])]
            position[r] += n
        longest = max(len(x[0]) for x in dense)
        kd, vd = (torch.zeros(rows * longest, hk, d, dtype=dtype) for _ in range(2))
        for r, (x, y) in enumerate(dense):
            kd[r * longest:r * longest + len(x)], vd[r * longest:r * longest + len(y)] = x, y
        table, lens = torch.arange(rows, dtype=torch.int32)[:, None], books.lens.cpu()
        assert lens.tolist() == [len(x[0]) for x in dense]
        want, bound = K.extend_exact(qr.cpu(), kd, vd, table, lens, cu, longest)
        assert bool(((out.cpu().double() - want).abs() <= bound).all())
        want, bound = X.weights_exact(before, qr.cpu(), kd, table, lens, cu, longest, max(counts))
        assert bool(((scores.cpu().double() - want).abs() <= bound).all())
        if budget is None:
            return
        sums = scores.cpu()
        keep = torch.where(books.lens > budget + 8, budget, -1).to(torch.int32)
        assert E.evict_rows([k_pool], [v_pool], [scores], *books, keep, page, first=4, recent=10).tolist() == [0, 0]
        for r, n in enumerate(lens.tolist()):
            if n <= budget + 8:
                continue
            new = [torch.empty(budget, hk, d, dtype=dtype) for _ in range(2)]
            for h in range(hk):
                order = torch.sort(sums[r, h, 4:n - 10], descending=True, stable=True)[1][:budget - 14].sort()[0]
                at = torch.cat([torch.arange(4), 4 + order, torch.arange(n - 10, n)])
                for i in range(2):
                    new[i][:, h] = dense[r][i][at, h]
            dense[r] = new

    step([70, 0, 33, 0, 0], [0, 0, 0], [0, 0])
    assert cache_pages.fork_rows([k_pool, v_pool], *books, ints(0, 2, 0), ints(1, 3, 4), page).tolist() == [0, 0]
    scores[1], scores[3], scores[4] = scores[0].clone(), scores[2].clone(), scores[0].clone()
    dense[1], dense[3], dense[4] = list(dense[0]), list(dense[2]), list(dense[0])
    position[1], position[3], position[4] = position[0], position[2], position[0]
    for i in range(4):
        step([1, 1, 1, 2, 1], [0, 2, 4], [70, 33])
    for i in range(6):  # from here on rows are cut, and share nothing but what was not
        step([5, 3, 1, 2, 9], [0, 2, 4], [0, 0], budget=48)
    assert books.lens.max() <= 56
    held = torch.zeros(pages, dtype=torch.int32)
    for r in range(rows):
        for j in range(-(-int(books.lens[r]) // page)):
            held[int(books.table[r, j])] += 1
    assert torch.equal(held, books.refs.cpu())


# ---- refusals ----------------------------------------------------------------------------------

@pytest.mark.gpu
def test_refusals():
    k, v, scores, refs, table, lens = _state([50, 20], 16, 4, 30, 2, (64, 64), torch.bfloat16, 2)
    k, v, scores = ([x.cuda() for x in part] for part in (k, v, scores))
    refs, table, lens = refs.cuda(), table.cuda(), lens.cuda()
    keep = torch.tensor([10, 5], dtype=torch.int32, device="cuda")
    odd = [torch.zeros(30 * 16, 2, 12, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    grad = [k[0], k[1].clone().requires_grad_()]
    for args, options, message in [
            ((k, v, scores[:1], refs, table, lens, keep, 16), {}, "as many K pools"),
            ((k[:1], v, scores, refs, table, lens, keep, 16), {}, "as many K pools"),
            (([], [], [], refs, table, lens, keep, 16), {}, "as many K pools"),
            ((k, v, [x.half() for x in scores], refs, table, lens, keep, 16), {}, "FP32 scores"),
            ((k, v, [x[:1] for x in scores], refs, table, lens, keep, 16), {}, "FP32 scores"),
            ((k, v, [scores[0], scores[1][:, :, 1:].contiguous()], refs, table, lens, keep, 16), {}, "same shape"),
            ((k, v, [x[:, :, :63].contiguous() for x in scores], refs, table, lens, keep, 16), {}, "place for every key"),
            ((k, v, [x[:, :1].contiguous() for x in scores], refs, table, lens, keep, 16), {}, "heads of the scores"),
            ((odd, v, scores, refs, table, lens, keep, 16), {}, "16 bytes"),
            (([k[0], k[0]], v, scores, refs, table, lens, keep, 16), {}, "share memory"),
            ((k, k, scores, refs, table, lens, keep, 16), {}, "share memory"),
            ((k, v, [scores[0], scores[0]], refs, table, lens, keep, 16), {}, "share memory"),
            ((k, v, scores, refs, table, lens, lens, 16), {}, "share memory"),
            ((k, [x[:-16] for x in v], scores, refs, table, lens, keep, 16), {}, "pages \\* page_size rows"),
            ((k, v, scores, refs, table, lens, keep.long(), 16), {}, "int32"),
            ((k, v, scores, refs, table, lens, keep[:1], 16), {}, "metadata"),
            ((k, v, scores, refs, table, lens, keep.cpu(), 16), {}, "same GPU"),
            ((k, v, scores, refs, table, lens, keep, 0), {}, "page"),
            ((k, v, scores, refs, table, lens, keep, 16), dict(first=-1), "must not be negative"),
            ((k, v, scores, refs, table, lens, keep, 16), dict(recent=-1), "must not be negative"),
            ((grad, v, scores, refs, table, lens, keep, 16), {}, "requires a gradient")]:
        with pytest.raises(ValueError, match=message):
            E.evict_rows(*args, **options)
    with pytest.raises(TypeError, match="list or a tuple"):
        E.evict_rows(k, v, scores[0], refs, table, lens, keep, 16)


class _Books(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("refs", "table", "lens")] + [
        (n, ctypes.c_int32) for n in ("pages", "rows", "width", "page_size")]


class _Evict(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("keep", "k_pools", "v_pools", "k_head_bytes", "v_head_bytes", "scores")] + [
        ("scores_stride", ctypes.c_int64)] + [(n, ctypes.c_int32) for n in ("layers", "heads", "first", "recent")]


@pytest.mark.parametrize("books,changes,message", [
    (dict(refs=0), {}, "books are missing"), (dict(pages=0), {}, "positive pages"), (dict(pages=1 << 21), {}, "at most"),
    ({}, dict(layers=0), "positive layers"), ({}, dict(heads=0), "positive layers"), ({}, dict(first=-1), "negative"),
    ({}, dict(scores_stride=127), "place for every key"), (dict(rows=1 << 24, width=1), dict(heads=64), "too many rows"),
    (dict(width=(1 << 24) - 1, page_size=128, rows=1), dict(scores_stride=1 << 31), "31 bits"),
    ({}, {}, "tensors are missing")])
def test_c_entry_refusals(books, changes, message):
    """Refused on the host before any launch: these run where there is no GPU."""
    lib = _lib.load()
    lib.fgw_kv_last_error.restype = ctypes.c_char_p
    b = dict(refs=16, table=16, lens=16, pages=64, rows=4, width=8, page_size=16)
    b.update(books)
    a = dict(scores_stride=128, layers=2, heads=2)
    a.update(changes)
    rc = lib.fgw_pages_evict(ctypes.byref(_Books(**b)), ctypes.byref(_Evict(**a)), None, None, None)
    assert rc in (_lib.FGW_MHA_EINVAL, _lib.FGW_MHA_EUNSUPPORTED)
    assert message in lib.fgw_kv_last_error().decode()


def test_workspace_is_bounded():
    """Kept positions of as many layers as fit 256 MB, and the plan."""
    lib = _lib.load()
    lib.fgw_pages_evict_workspace.restype = ctypes.c_int64
    b = _Books(refs=16, table=16, lens=16, pages=1 << 16, rows=64, width=1024, page_size=16)
    need = lib.fgw_pages_evict_workspace(ctypes.byref(b), ctypes.byref(_Evict(scores_stride=16384, layers=80, heads=8)))
    assert 64 * 8 * 16384 <= need <= (1 << 26) + (1 << 16) + 64 * 1040
