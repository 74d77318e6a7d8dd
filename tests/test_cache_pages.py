"""Books and pages of the cache against books kept with Python integers; copies, graphs, refusals."""
import random

import pytest
import torch

from fgw_amd.operators.mha import cache_pages as C
from tests.kv_oracle import Books


def _pools(pages, page, shapes=((2, 64), (2, 64)), dtype=torch.bfloat16):
    gen = torch.Generator(device="cuda").manual_seed(3)
    return [torch.randn(pages * page, *s, generator=gen, device="cuda").to(dtype) for s in shapes]


def _ids(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _same(books, want):
    assert books.refs.tolist() == want.refs
    assert books.lens.tolist() == want.lens
    for r, row in enumerate(books.table.tolist()):
        assert row == want.table[r], r


def _moved(pools, moves, page):
    out = []
    for p in pools:
        p = p.clone()
        pages = p.view(p.shape[0] // page, -1)
        old = pages.clone()
        for a, b in moves:
            pages[b] = old[a]
        out.append(p)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("pages,rows,width,page", [(1, 1, 1, 16), (24, 5, 7, 4), (200, 30, 16, 1), (700, 64, 40, 16),
                                                   (40000, 1500, 33, 8)])
def test_random_books(pages, rows, width, page):
    """A run of all operations with the pool near its end, requests refused among them."""
    rng = random.Random(pages)
    small = [(8,), (2, 16)] if pages > 1000 else [(2, 64), (8,)]
    pools = _pools(pages, page, small)
    books = C.new_books(pages, rows, width)
    want = Books(*[x.cpu() for x in books], page)
    for turn in range(12):
        counts = [rng.choice((0, 0, 1, rng.randint(0, width * page // 2), -1, width * page + 1)) for _ in range(rows)]
        assert C.reserve_rows(*books, _ids(counts), page).tolist() == want.reserve(counts)
        _same(books, want)
        n = rng.randint(0, min(rows, 40))
        parents = [rng.randint(-1, rows) for _ in range(n)]
        children = [rng.randint(-1, rows) for _ in range(n)]
        empty = [r for r in range(rows) if want.lens[r] == 0]
        rng.shuffle(empty)
        for i, r in enumerate(empty[:n // 2]):
            children[i] = r
        status, moves = want.fork(parents, children)
        expected = _moved(pools, moves, page)
        assert C.fork_rows(pools, *books, _ids(parents), _ids(children), page).tolist() == status
        _same(books, want)
        assert all(torch.equal(a, b) for a, b in zip(pools, expected))
        gone = [rng.randint(-1, rows) for _ in range(rng.randint(0, rows // 2 + 1))]
        C.free_rows(*books, _ids(gone), page)
        want.free(gone)
        _same(books, want)
        if turn % 3 == 2:
            moves = want.compact()
            expected = _moved(pools, moves, page)
            assert C.compact_pages(pools, *books, page).tolist() == [len(moves)]
            _same(books, want)
            assert all(torch.equal(a, b) for a, b in zip(pools, expected))


@pytest.mark.gpu
def test_more_pairs_and_rows_than_threads():
    pages, rows, width, page = 5000, 3000, 3, 4
    books = C.new_books(pages, rows, width)
    want = Books(*[x.cpu() for x in books], page)
    counts = [5] * 100 + [0] * (rows - 100)
    assert C.reserve_rows(*books, _ids(counts), page).tolist() == want.reserve(counts) == [0, 0]
    parents, children = [i % 100 for i in range(2900)], list(range(100, rows))
    children[2000] = children[5]  # an earlier pair's child, in another step of the scan
    parents[2500] = rows - 1      # ... and a parent that is a child
    pools = _pools(pages, page, [(8,)])
    status, moves = want.fork(parents, children)
    expected = _moved(pools, moves, page)
    assert C.fork_rows(pools, *books, _ids(parents), _ids(children), page).tolist() == status
    _same(books, want)
    assert torch.equal(pools[0], expected[0])


@pytest.mark.gpu
def test_refused_for_want_of_pages():
    books = C.new_books(4, 4, 4)
    # 1 and 3 pages are there; the other two rows find none, and one that needs none still grows.
    assert C.reserve_rows(*books, _ids([2, 20, 3, 1]), 8).tolist() == [2, 0]
    assert books.lens.tolist() == [2, 20, 0, 0] and books.table[2].tolist() == [-1] * 4
    assert C.reserve_rows(*books, _ids([7, 0, 1, 0]), 8).tolist() == [2, 0]
    assert C.reserve_rows(*books, _ids([6, 4, 1, 0]), 8).tolist() == [1, 0]
    assert books.lens.tolist() == [8, 24, 0, 0]
    assert C.fork_rows([], *books, _ids([1]), _ids([2]), 8).tolist() == [0, 0]  # whole pages: shared
    assert books.refs.tolist() == [1, 2, 2, 2]
    C.free_rows(*books, _ids([0]), 8)
    assert C.reserve_rows(*books, _ids([3, 0, 0, 0]), 8).tolist() == [0, 0]
    assert C.fork_rows([], *books, _ids([0]), _ids([3]), 8).tolist() == [1, 0]  # no page for the copy
    assert books.lens.tolist() == [3, 24, 24, 0] and books.refs.tolist() == [1, 2, 2, 2]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,shape", [(torch.bfloat16, (8, 128)), (torch.float32, (3, 4)), (torch.uint8, (16,)),
                                         (torch.float16, (1, 1000 * 8))], ids=str)
def test_copies_of_any_type_and_many_pools(dtype, shape):
    page, pages = 4, 60
    pools = [torch.randint(0, 100, (pages * page, *shape), device="cuda").to(dtype) for _ in range(67)]
    src, dst = [3, 3, -1, 59, 5, 70, 6], [0, 1, 2, 40, 60, 7, 58]
    want = _moved(pools, [(a, b) for a, b in zip(src, dst) if 0 <= a < pages and 0 <= b < pages], page)
    C.copy_pages(pools, _ids(src), _ids(dst), page)
    assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(pools, want))


@pytest.mark.gpu
def test_copies_past_32_bits():
    page, pages = 64, (1 << 32) // (64 * 2048) + 4
    pool = torch.zeros(pages * page, 1024, dtype=torch.bfloat16, device="cuda")
    pool[:page] = 1.0
    C.copy_pages([pool], _ids([0]), _ids([pages - 1]), page)
    assert bool((pool[-page:] == 1.0).all()) and bool((pool[-2 * page:-page] == 0.0).all())


@pytest.mark.gpu
def test_replays_of_captured_books():
    """reserve, fork, free and compact in one graph: each replay like the calls made eagerly."""
    pages, rows, width, page = 64, 8, 8, 4
    pools = _pools(pages, page)
    start = C.new_books(pages, rows, width)
    C.reserve_rows(*start, _ids([9, 13, 3, 0, 0, 0, 20, 0]), page)
    keep = [x.clone() for x in start]
    kept = [x.clone() for x in pools]
    counts, parents, children, gone = _ids([1, 1, 1, 0, 0, 0, 1, 0]), _ids([1, 0]), _ids([3, 5]), _ids([0, 2])

    def step():
        return (C.reserve_rows(*start, counts, page), C.fork_rows(pools, *start, parents, children, page),
                C.free_rows(*start, gone, page), C.compact_pages(pools, *start, page))

    def reset():
        for a, b in zip((*start, *pools), (*keep, *kept)):
            a.copy_(b)

    eager = [x.tolist() for x in step() if x is not None]
    after = [x.clone() for x in (*start, *pools)]
    reset()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = step()
    for _ in range(3):
        reset()
        graph.replay()
        torch.cuda.synchronize()
        assert [x.tolist() for x in result if x is not None] == eager
        assert all(torch.equal(a, b) for a, b in zip((*start, *pools), after))


@pytest.mark.gpu
def test_books_in_one_buffer_at_any_offset():
    """Views that start at odd elements: the reads of refs need no alignment."""
    pages, rows, width, page = 50, 4, 6, 4
    buf = torch.zeros(1 + pages + rows * width + rows, dtype=torch.int32, device="cuda")
    refs, table = buf[1:1 + pages], buf[1 + pages:1 + pages + rows * width].view(rows, width)
    lens = buf[1 + pages + rows * width:]
    table.fill_(-1)
    want = Books(refs.cpu(), table.cpu(), lens.cpu(), page)
    assert C.reserve_rows(refs, table, lens, _ids([24, 9, 0, 1]), page).tolist() == want.reserve([24, 9, 0, 1])
    _same(C.PageBooks(refs, table, lens), want)


@pytest.mark.gpu
def test_refusals():
    books = C.new_books(8, 2, 4)
    pools = _pools(8, 4)
    with pytest.raises(ValueError, match="page size"):
        C.reserve_rows(*books, _ids([1, 1]), 0)
    with pytest.raises(ValueError, match="metadata"):
        C.reserve_rows(*books, _ids([1]), 4)
    with pytest.raises(ValueError, match="int32"):
        C.reserve_rows(*books, _ids([1, 1]).long(), 4)
    with pytest.raises(ValueError, match="pages \\* page_size"):
        C.compact_pages([pools[0][:-1]], *books, 4)
    with pytest.raises(ValueError, match="multiples of 16"):
        C.compact_pages([torch.zeros(32, 3, dtype=torch.uint8, device="cuda")], *books, 4)
    with pytest.raises(ValueError, match="same GPU"):
        C.compact_pages([pools[0].cpu()], *books, 4)
    with pytest.raises(ValueError, match="contiguous"):
        C.compact_pages([pools[0].transpose(1, 2)], *books, 4)
    with pytest.raises(ValueError, match="metadata"):
        C.fork_rows(pools, *books, _ids([0, 1]), _ids([1]), 4)
    with pytest.raises(TypeError, match="list or a tuple"):
        C.fork_rows(pools[0], *books, _ids([0]), _ids([1]), 4)
    with pytest.raises(ValueError, match="whole pool pages"):
        C.copy_pages([pools[0][:-1]], _ids([0]), _ids([1]), 4)
    with pytest.raises(ValueError, match="at most"):
        C.free_rows(torch.zeros((1 << 20) + 1, dtype=torch.int32, device="cuda"), books.table, books.lens, _ids([0]), 4)


def test_refusals_without_a_gpu():
    books = C.new_books(8, 2, 4, device="cpu")
    with pytest.raises(ValueError, match="same GPU"):
        C.reserve_rows(*books, torch.zeros(2, dtype=torch.int32), 4)
    with pytest.raises(ValueError, match="positive pages"):
        C.new_books(0, 2, 4, device="cpu")
    with pytest.raises(ValueError, match="at least one pool"):
        C.copy_pages([], books.lens, books.lens, 4)


def test_the_python_books_themselves():
    b = Books(torch.zeros(6, dtype=torch.int32), torch.full((4, 3), -1), torch.zeros(4, dtype=torch.int32), 4)
    assert b.reserve([5, 0, 9, 0]) == [0, 0] and b.table[:3] == [[0, 1, -1], [-1] * 3, [2, 3, 4]]
    assert b.fork([0, 2], [1, 3]) == ([1, 0], [(1, 5)])
    assert b.table[1] == [0, 5, -1] and b.refs == [2, 1, 1, 1, 1, 1] and b.lens == [5, 5, 9, 0]
    b.free([2, 2])
    assert b.refs == [2, 1, 0, 0, 0, 1] and b.compact() == [(5, 2)] and b.table[1] == [0, 2, -1]
