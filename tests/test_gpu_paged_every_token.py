"""Paged decode: every token is counted once, whatever the cut of the work, and a call repeats itself."""

import pytest
import torch

from tritonkv_b200.kernels import paged_decode_attention, paged_fp16_decode_attention
from tritonkv_b200.quantize import QuantizedTensor, pack_codes

from paged_util import DEV, make_pools, reference

pytestmark = pytest.mark.gpu


def marker_pools(lens, HKV, D, nbits, gs, page, seed):
    """K of any kind and V of zeros and ones (scale 1, zero point 0), in pages of random order; and the
    ones, (tokens, HKV, D) per sequence."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    k, _, table, NP = make_pools(lens, HKV, D, nbits, gs, page, seed=seed, width=max(-(-n // page) for n in lens) + 2)
    ones = torch.randint(0, 2, (NP, HKV, page, D), generator=g, device=DEV, dtype=torch.uint8)
    if nbits == 16:
        v = ones.half()
    else:
        unit = torch.ones_like(k.scale)
        v = QuantizedTensor(pack_codes(ones, nbits), unit, torch.zeros_like(unit), nbits, gs, D)
    return k, v, table, NP, ones


@pytest.mark.parametrize("nbits,D,gs", [(4, 128, 32), (2, 128, 32), (4, 64, 16), (2, 64, 64), (4, 128, 128), (16, 128, 0), (16, 64, 0)])
@pytest.mark.parametrize("page", [16, 48, 64])
@pytest.mark.parametrize("lens,HKV,G", [
    ([65536], 1, 2), ([20011], 2, 6), ([9000, 8223, 7446], 8, 1), ([4096 - 61 * i for i in range(16)], 8, 4),
    ([(i * 977) % 3000 for i in range(40)], 8, 2), ([30000, 5, 0, 64, 1, 250], 4, 7), ([(i * 37) % 200 for i in range(300)], 2, 9)])
def test_every_token_once(lens, HKV, G, page, nbits, D, gs):
    """q = 0: every token has weight 1/n, and n times the output is the number of ones in the column.  All
    weights are one power of two, the sums whole numbers below 2^24, so what is off is a few roundings of
    float32 at the end (2^-21 of at most 65536, less than 0.04); a tile of 32 that is missing or counted twice moves
    each of the columns by half the root of 8, about."""
    k, v, table, NP, ones = marker_pools(lens, HKV, D, nbits, gs, page, seed=sum(lens) % 1000 + page)
    holes = {(0, 1), (len(lens) - 1, 0)} if page == 48 else set()
    for b, i in holes:
        table[b, i] = (-1, NP)[b % 2]
    q = torch.zeros(len(lens), HKV * G, D, dtype=torch.float16, device=DEV)
    fn = paged_fp16_decode_attention if nbits == 16 else paged_decode_attention
    got = fn(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=DEV)).double()
    for b, n in enumerate(lens):
        if n == 0:
            assert bool((got[b] == 0).all())
            continue
        keep = torch.ones(n, dtype=torch.bool, device=DEV)
        for hb, i in holes:
            if hb == b:
                keep[i * page:(i + 1) * page] = False
        ids = table[b, : -(-n // page)].long().clamp(0, NP - 1)
        seen = ones[ids].transpose(0, 1).flatten(1, 2)[:, :n][:, keep].double()
        col = seen.sum(1)  # (HKV, D)
        count = int(keep.sum())
        if count == 0:
            assert bool((got[b] == 0).all())
            continue
        off = (got[b].view(HKV, G, D) * count - col[:, None]).abs().max()
        assert float(off) < 0.25, f"sequence {b} of {n}: off by {float(off):.3g} tokens"
        if count > 64:  # (and a tile that is left out would be seen, in every head)
            less = seen[:, 32:].sum(1) * count / (count - 32)
            assert bool(((less - col).abs().amax(-1) > 1).all())


@pytest.mark.parametrize("nbits,page", [(4, 16), (4, 128), (2, 64), (2, 48)])
@pytest.mark.parametrize("B,HKV,ctx", [(1, 2, 20011), (1, 1, 65536), (3, 8, 9000)])
def test_long_histories_in_the_2_norm(nbits, page, B, HKV, ctx):
    """The element-wise bound adds up worst cases over the tokens; in the 2-norm the roundings are 4.9e-4, and
    8 tiles of 20011 tokens would be 1e-1."""
    lens = [ctx - 777 * b for b in range(B)]
    k, v, table, _ = make_pools(lens, HKV, 128, nbits, 32, page, seed=ctx)
    q = torch.randn(B, HKV * 6, 128, generator=torch.Generator().manual_seed(3)).to(DEV).half()
    got = paged_decode_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=DEV))
    ref, _ = reference(q, k, v, table, lens)
    assert float((got.double() - ref).norm() / ref.norm()) <= 1e-3


@pytest.mark.parametrize("nbits", [2, 4, 16])
def test_repeats_bit_for_bit(nbits):
    """The same call gives the same bits, whichever CTA merges and whatever ran between."""
    ws = {}
    for lens, HKV in (([500], 2), ([65536], 2), ([4096 - 61 * i for i in range(16)], 8), ([(i * 977) % 4000 for i in range(64)], 8)):
        k, v, table, _ = make_pools(lens, HKV, 128, nbits, 32, 32, seed=len(lens))
        q = torch.randn(len(lens), HKV * 4, 128, generator=torch.Generator().manual_seed(1)).to(DEV).half()
        sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
        fn = paged_fp16_decode_attention if nbits == 16 else paged_decode_attention
        first = fn(q, k, v, table, sl)
        for _ in range(20):
            fn(q.flip(0), k, v, table.flip(0).contiguous(), sl.flip(0).contiguous(), _workspace=ws)
            assert torch.equal(fn(q, k, v, table, sl, _workspace=ws), first)
