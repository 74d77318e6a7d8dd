"""What the cache operators write in place moves its version: a gradient that saved the old contents is
refused, where it would be computed from the new ones."""
import pytest
import torch

from fgw_amd.operators.mha import cache_pages as C, paged_extend as P
from fgw_amd.operators.mha.rotary import Rotary, apply_rotary

pytestmark = pytest.mark.gpu


def _ids(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _versions(*tensors):
    return [x._version for x in tensors]


def test_a_gradient_with_rows_that_were_rotated_in_place_is_refused():
    x, w = torch.randn(6, 2, 16, device="cuda"), torch.randn(16, 4, device="cuda", requires_grad=True)
    pos, r = torch.arange(6, dtype=torch.int32, device="cuda"), Rotary(16)
    y = x @ w  # saves x
    apply_rotary(x, pos, r, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = x @ w
    rotated = apply_rotary(x, pos, r)  # a new tensor: nothing is lost
    y.sum().backward()
    assert rotated._version == 0


def test_a_gradient_at_positions_that_the_books_changed_is_refused():
    books = C.new_books(8, 4, 2)
    C.reserve_rows(*books, _ids(3, 1, 0, 2), 16)
    x = torch.randn(4, 2, 16, device="cuda", requires_grad=True)
    y = apply_rotary(x, books.lens, Rotary(16))
    C.reserve_rows(*books, _ids(1, 1, 1, 1), 16)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_append_and_attention_move_what_they_write():
    q, k, v = (torch.randn(3, n, 64, device="cuda").half() for n in (4, 2, 2))
    kc, vc = (torch.zeros(64, 2, 64, device="cuda").half() for _ in range(2))
    meta = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2), _ids(9, 20), _ids(0, 2, 3)
    w = torch.randn(64, 2, 64, device="cuda", requires_grad=True)
    saved = (kc.float() * w).sum() + (kc * w.half()).sum()  # the second product saves the pool itself
    out = torch.empty_like(q)
    before = _versions(q, k, v, kc, vc, out, *meta)
    P.mha_paged_append(q, k, v, kc, vc, *meta, 16)
    assert _versions(q, k, v, kc, vc, out, *meta) == [n + (i in (3, 4)) for i, n in enumerate(before)]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()
    P.mha_paged_append(q, k, v, kc, vc, *meta, 16, q_out=q)
    kernel = P.build_extend_kernel(4, 2, 64, 16, "float16", 0)
    kernel(q, kc, vc, *meta, 2, out)
    assert _versions(q, k, v, kc, vc, out, *meta) == [n + (1, 0, 0, 2, 2, 1, 0, 0, 0)[i] for i, n in enumerate(before)]
    kernel(q, kc, vc, *meta, 2)
    assert out._version == before[5] + 1


def test_books_and_pools_move():
    books, pool = C.new_books(8, 4, 2), torch.zeros(8 * 16, 8, device="cuda")
    watch = (*books, pool)
    for call, moved in (
            (lambda: C.reserve_rows(*books, _ids(20, 0, 0, 0), 16), 0), (lambda: C.fork_rows([pool], *books, _ids(0), _ids(1), 16), 1),
            (lambda: C.free_rows(*books, _ids(0), 16), 0), (lambda: C.compact_pages((pool,), *books, 16), 1)):
        before = _versions(*watch)
        call()
        assert _versions(*watch) == [before[0] + 1, before[1] + 1, before[2] + 1, before[3] + moved]
    before = _versions(*watch)
    C.copy_pages([pool], _ids(0), _ids(7), 16)
    assert _versions(*watch) == [*before[:3], before[3] + 1]


def test_inference_tensors_are_written():
    with torch.inference_mode():
        x, pos, r = torch.randn(6, 2, 16, device="cuda"), torch.arange(6, dtype=torch.int32, device="cuda"), Rotary(16)
        want = apply_rotary(x, pos, r)
        assert torch.equal(apply_rotary(x, pos, r, out=x), want)
        books = C.new_books(8, 4, 2)
        assert C.reserve_rows(*books, _ids(3, 1, 0, 2), 16).tolist() == [0, 0] and books.lens.tolist() == [3, 1, 0, 2]
