"""The quantiser's codes where its quotient needs care: ties of the rounding to a code, scales that
underflow or overflow float16, minima outside float16.  Against the definition, operation by operation
in torch (float32 on the CPU: IEEE division and rounding to even)."""

import pytest
import torch

from tritonkv_b200.quantize import quantize_groupwise, unpack_codes

pytestmark = pytest.mark.gpu
DEV = "cuda"


def definition(x, nbits, gs):
    g = x.cpu().float().unflatten(-1, (x.shape[-1] // gs, gs))
    lo, hi = g.amin(-1), g.amax(-1)
    qmax = torch.tensor(2.0 ** nbits - 1)
    s = (hi - lo) / qmax
    s = torch.where(s > 0, s, torch.ones_like(s)).half()
    z = lo.half()
    q = ((g - z.float()[..., None]) / s.float()[..., None]).round()
    q = torch.where(q.isnan(), torch.zeros_like(q), q).clamp(0, 2 ** nbits - 1)
    return q.flatten(-2).to(torch.uint8), s, z


def compare(x, nbits, gs):
    qt = quantize_groupwise(x, nbits, gs)
    code, s, z = definition(x, nbits, gs)
    assert torch.equal(qt.scale.cpu().nan_to_num(nan=-1.0), s.nan_to_num(nan=-1.0))
    assert torch.equal(qt.zero.cpu().nan_to_num(nan=-1.0), z.nan_to_num(nan=-1.0))
    assert torch.equal(unpack_codes(qt.packed, nbits, x.shape[-1]).cpu(), code)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nbits", [2, 4])
def test_coarse_inputs_are_full_of_ties(nbits, dtype):
    g = torch.Generator().manual_seed(nbits)
    for step in (1.0, 0.5, 0.25, 2.0 ** -7, 3.0, 0.1):
        x = torch.randint(-60, 61, (400, 128), generator=g).float() * step
        for gs in (16, 32, 128):
            compare(x.to(dtype).to(DEV), nbits, gs)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nbits", [2, 4])
def test_sizes_from_the_smallest_to_the_largest(nbits, dtype):
    """Ranges and offsets of every size the type has, far offsets with small ranges among them."""
    g = torch.Generator().manual_seed(7 + nbits)
    lo, hi = {torch.float16: (-24, 16), torch.bfloat16: (-133, 127), torch.float32: (-149, 127)}[dtype]
    e = torch.randint(lo, hi, (4000, 1), generator=g).double()
    off = torch.randint(lo, hi, (4000, 1), generator=g).double()
    x = torch.randn(4000, 64, generator=g).double() * 2.0 ** e + torch.randn(4000, 1, generator=g).double() * 2.0 ** off
    big = torch.finfo(dtype).max
    compare(x.clamp(-big, big).to(dtype).to(DEV), nbits, 16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nbits", [2, 4])
def test_infinities_nan_and_constants(nbits, dtype):
    x = torch.randn(24, 64, generator=torch.Generator().manual_seed(3))
    inf, nan = float("inf"), float("nan")
    for i, v in enumerate((inf, -inf, nan, 0.0, 3e38, -3e38, 65504.0, -65504.0, 65519.0, 65520.0, -65520.0, 1e-45, 2.0 ** -24, 2.0 ** -26)):
        x[i, 5] = v
    x[14] = 0.0
    x[15] = -1.25
    x[16], x[17] = inf, -inf
    x[18] = -70000.0
    x[18, ::3] += 512.0
    x[19] = 70000.0
    x[19, ::3] += 512.0
    x[20] = torch.arange(64) * 2.0 ** -28
    x[21] = torch.arange(64) * -(2.0 ** -140)
    x[22, :32], x[22, 32:] = inf, -inf
    x[23] = nan
    compare(x.to(dtype).to(DEV), nbits, 16)
