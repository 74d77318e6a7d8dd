"""Outputs and pools that record a gradient are not overwritten while gradients are recorded."""
import pytest
import torch

from fgw_amd.operators.mha import cache_pages as C, paged_extend as P
from fgw_amd.operators.mha.rotary import Rotary, apply_rotary

pytestmark = pytest.mark.gpu


def _calls():
    q, k, v = (torch.randn(3, n, 64, device="cuda").half() for n in (4, 2, 2))
    kc, vc = (torch.randn(64, 2, 64, device="cuda").half() for _ in range(2))
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2)
    lens, cu = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([9, 20], [0, 2, 3]))
    r, kernel = Rotary(64), P.build_extend_kernel(4, 2, 64, 16, "float16", 0)
    leaf = torch.zeros_like(q)
    books = C.new_books(4, 2, 2)
    ids = torch.tensor([1], dtype=torch.int32, device="cuda")
    return {
        "rotary": (leaf, lambda: apply_rotary(q, torch.zeros(3, dtype=torch.int32, device="cuda"), r, out=leaf)),
        "append": (leaf, lambda: P.mha_paged_append(q, k, v, kc, vc, table, lens, cu, 16, rotary=r, q_out=leaf)),
        "k_pool": (kc, lambda: P.mha_paged_append(q, k, v, kc, vc, table, lens, cu, 16)),
        "v_pool": (vc, lambda: P.mha_paged_append(q, k, v, kc, vc, table, lens, cu, 16)),
        "attention": (leaf, lambda: kernel(q, kc, vc, table, lens, cu, 2, leaf)),
        "fork": (kc, lambda: C.fork_rows([vc, kc], *books, ids, ids - 1, 16)),
        "compact": (kc, lambda: C.compact_pages([kc], *books, 16)),
        "copy": (kc, lambda: C.copy_pages([vc, kc], ids, ids + 1, 16)),
    }


@pytest.mark.parametrize("name", ["rotary", "append", "k_pool", "v_pool", "attention", "fork", "compact", "copy"])
def test_refused_unless_no_gradient_is_recorded(name):
    written, call = _calls()[name]
    written.requires_grad_()
    kept = written.detach().clone()
    with pytest.raises(ValueError, match="requires a gradient"):
        call()
    assert torch.equal(written, kept)
    with torch.no_grad():
        call()
    written.requires_grad_(False)
    call()


@pytest.mark.parametrize("name", ["rotary", "attention"])
def test_a_view_of_what_requires_a_gradient_is_refused(name):
    base = torch.zeros(2, 3, 4, 64, device="cuda", dtype=torch.float16, requires_grad=True)
    q = torch.randn(3, 4, 64, device="cuda").half()
    if name == "rotary":
        with pytest.raises(ValueError, match="requires a gradient"):
            apply_rotary(q, torch.zeros(3, dtype=torch.int32, device="cuda"), Rotary(64), out=base[1])
    else:
        kc = torch.randn(64, 2, 64, device="cuda").half()
        table = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2)
        lens, cu = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([9, 20], [0, 2, 3]))
        with pytest.raises(ValueError, match="requires a gradient"):
            P.build_extend_kernel(4, 2, 64, 16, "float16", 0)(q, kc, kc, table, lens, cu, 2, base[0])
