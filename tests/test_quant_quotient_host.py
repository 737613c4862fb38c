"""The quotient of the group-wise quantiser (``tritonkv_b200/csrc/tkv_quant_part.cuh``), restated in numpy.

``code = clamp(rint((x - zero) / scale))`` is formed without a division: with y the rounded reciprocal of the
scale s, ``q = a*y`` and ``q = fma(fma(-q, s, a), y, q)``, both scaled by powers of two so that a saturation to
[0, 1] is the clamp.  It must give the codes of the IEEE division, in particular around the borders from one code to
the next and where a quotient is a tie.  (The per-channel quantiser keeps the reciprocal with a redo, see
``test_quant_arith_host.py``.)"""

import numpy as np
import pytest

f32, f64 = np.float32, np.float64


def fma32(a, b, c):
    """a*b + c of float32 arrays with one rounding to float32."""
    p = a.astype(f64) * b.astype(f64)  # (exact: 48 bits)
    c = c.astype(f64)
    s = p + c
    t = s - p
    e = (p - (s - t)) + (c - t)  # s + e is the exact sum
    return np.where(e == 0, s, np.nextafter(s, np.where(e > 0, np.inf, -np.inf))).astype(f32)


def codes(a, s, nbits):
    n = f32(1 << nbits)
    top = f32(((1 << nbits) - 1) / (1 << nbits))
    y, ss = ((f32(1) / s).astype(f32) / n).astype(f32), (s * n).astype(f32)
    q = (a * y).astype(f32)
    u = fma32(fma32(-q, ss, a), y, q)
    u = np.minimum(np.clip(np.where(np.isnan(u), f32(0), u), f32(0), f32(1)), top)
    return np.rint(u.astype(f64) * float(n))  # (the product is exact: one rounding, half to even)


def ieee(a, s, nbits):
    return np.clip(np.rint((a / s).astype(f32)), 0, (1 << nbits) - 1)


def test_the_fused_operation():
    """fma32 against exact integer arithmetic."""
    from fractions import Fraction

    g = np.random.default_rng(0)
    a, b, c = (g.standard_normal(4000).astype(f32) for _ in range(3))
    c[:2000] = -(a[:2000].astype(f64) * b[:2000].astype(f64)).astype(f32)  # (cancellation)
    for x, y, z, got in zip(a, b, c, fma32(a, b, c)):
        exact = Fraction(float(x)) * Fraction(float(y)) + Fraction(float(z))
        near = [np.nextafter(got, f32(-np.inf)), got, np.nextafter(got, f32(np.inf))]
        off = [abs(Fraction(float(v)) - exact) for v in near]
        assert off[1] == min(off)


@pytest.mark.parametrize("nbits", [2, 4])
def test_around_every_border_of_the_codes(nbits):
    """Scales of every mantissa (a few exponents, all subnormals); floats around every (code + 1/2) * scale."""
    bits = np.concatenate([np.arange(1, 1024)] + [np.arange(1024 * e, 1024 * (e + 1)) for e in (1, 9, 15, 16, 30)])
    s = bits.astype(np.uint16).view(np.float16).astype(f32)[:, None, None]
    border = ((np.arange(-1, 1 << nbits) + 0.5)[None, :, None] * s.astype(f64)).astype(f32)
    step = np.arange(-6, 7, dtype=np.int32)[None, None]
    a = (border.view(np.int32) + step).view(f32)
    s = np.broadcast_to(s, a.shape)
    assert np.array_equal(codes(a, s, nbits), ieee(a, s, nbits))


@pytest.mark.parametrize("nbits", [2, 4])
def test_over_the_range(nbits):
    g = np.random.default_rng(nbits)
    s = g.integers(1, 0x7c00, 1_000_000).astype(np.uint16).view(np.float16).astype(f32)
    a = (g.uniform(-2, (1 << nbits) + 2, s.shape) * s).astype(f32)
    a[::3] = (np.rint(a[::3] / s[::3] * 2) / 2 * s[::3].astype(f64)).astype(f32)  # (ties and whole codes)
    assert np.array_equal(codes(a, s, nbits), ieee(a, s, nbits))
