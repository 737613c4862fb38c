"""Paged decode: where the codes of K and V lie relative to each other."""

import pytest
import torch

from tritonkv_b200.kernels import paged_decode_attention

from paged_util import DEV, check, make_pools

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("order", ["K below V", "V below K", "close together", "K is V"])
@pytest.mark.parametrize("page", [16, 32, 48])
@pytest.mark.parametrize("nbits,D", [(4, 128), (2, 128), (4, 64), (2, 64)])
def test_places_of_the_pools(nbits, D, page, order):
    """One copy brings a run of K and of V where their codes lie apart far enough, either one first; two copies
    where they do not: here where K and V are the same pool, and where they overlap."""
    lens = [700, 0, 33, 2 * page + 5]
    k, v, table, NP = make_pools(lens, 2, D, nbits, 32, page, seed=page + D + nbits)
    n = k.packed.numel()
    slab = torch.empty(2 * n, dtype=torch.uint8, device=DEV)
    if order == "K is V":
        v = k
    elif order == "close together":  # V's pages begin one page behind K's, in the same memory
        one = k.packed[0].numel()
        slab[: n + one].copy_(torch.cat([k.packed.flatten(), v.packed.flatten()])[: n + one])
        k.packed, v.packed = slab[:n].view_as(k.packed), slab[one:one + n].view_as(v.packed)
    else:
        for i, t in enumerate((k, v) if order == "K below V" else (v, k)):
            part = slab[i * n:(i + 1) * n].view_as(t.packed)
            part.copy_(t.packed)
            t.packed = part
    for HQ in (2, 12):  # (8 and 4 units: the 4-warp family; one sequence of 2 heads below: the 8-warp one)
        q = torch.randn(len(lens), HQ, D, generator=torch.Generator().manual_seed(HQ)).to(DEV).half()
        sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
        check(paged_decode_attention(q, k, v, table, sl), q, k, v, table, lens, order)
        check(paged_decode_attention(q[:1], k, v, table[:1], sl[:1]), q[:1], k, v, table[:1], lens[:1], order + ", one")
