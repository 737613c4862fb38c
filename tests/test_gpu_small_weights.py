"""Tokens of small weight beside one of large weight, and values of every size, against float64.

A few tokens take most of the softmax and have values near zero, so the output is made of the many
others.  Their weights and the products with the value scales are float16 operands.

The bound is on the 2-norm of the whole output.  A rounding to float16 is off by 2^-11 / sqrt(6) =
2.0e-4 of the value, root mean square (half a step of 2^-11 at most, uniform in it, over a binade).
A float16 cache has one, of the weight: 2.0e-4 of the output.  A packed one has a second, of weight
times scale, in front of the codes: over groups of 32 normal values code * scale is about 2 standard
deviations off zero, sqrt(1 + 4) of the values' size, so 2.0e-4 * sqrt(1 + 5) = 4.9e-4 in all.  Twice that is
allowed; a hundredth of the weight lost would be 1e-2."""

import math

import pytest
import torch

from tritonkv_b200 import quantize as Q
from tritonkv_b200.kernels import (fp16_decode_attention, fused_decode_attention, kivi_decode_attention,
                                   paged_decode_attention, paged_fp16_decode_attention, quantize_kv_kivi)
from tritonkv_b200.quantize import QuantizedTensor, quantize_groupwise

from paged_util import DEV, values64

pytestmark = pytest.mark.gpu
SIZES = [1.0, 2.0 ** -4, 2.0 ** -6, 2.0 ** -8, 8.0, 256.0, "late"]


def inputs(B, HKV, G, S, D, size, weight, seed):
    """q, K and V: `weight` of the softmax goes to S / 1000 tokens with values of a thousandth."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *shape: torch.randn(*shape, generator=g, device=DEV)
    u = rnd(B, HKV, D)
    q = (u[:, :, None] + 0.05 * rnd(B, HKV, G, D)).flatten(1, 2).half()
    k, v = 0.3 * rnd(B, HKV, S, D), rnd(B, HKV, S, D)
    if size == "late":  # small values first, large ones in one group of some tokens behind
        v *= 2.0 ** -6
        v[:, :, S // 3::97, :32] *= 2.0 ** 14
    else:
        v *= size
    if weight:
        n = max(1, S // 1000)
        at = torch.randperm(S // 2, generator=g, device=DEV)[:n]
        score = math.log(weight / (1 - weight) * (S - n) / n)
        k[:, :, at] = (u * (score * math.sqrt(D) / (u * u).sum(-1, keepdim=True)))[:, :, None]
        v[:, :, at] *= 1e-3
    return q, k.half(), v.half()


def exact(q, k, v):
    """softmax(q k / sqrt(D)) v in float64, sequence by sequence."""
    B, HQ, D = q.shape
    out = []
    for b in range(B):
        s = q[b].double().view(k.shape[1], -1, D) @ k[b].double().transpose(-1, -2) / math.sqrt(D)
        out.append((torch.softmax(s, -1) @ v[b].double()).flatten(0, 1))
    return torch.stack(out)


def values(x):
    return values64(x)[0]


def bound(nbits, gs, size):
    if size == "late":
        return 2 * 2.0 ** -11 / math.sqrt(3) * math.sqrt(1 + (0 if nbits == 16 else 1 + 4 * max(gs, 32) / 32))
    return 4e-4 if nbits == 16 else 1e-3


def close(got, ref, allowed, what):
    e = float((got.double() - ref).norm() / ref.norm())
    assert e <= allowed, f"{what}: {e:.2e} of the 2-norm, {allowed:.2e} allowed"


def pages(t, page):
    B, H, S, X = t.shape
    return t.view(B, H, S // page, page, X).transpose(1, 2).reshape(B * S // page, H, page, X).contiguous()


def paged(x, page):
    if isinstance(x, torch.Tensor):
        return pages(x, page)
    return QuantizedTensor(pages(x.packed, page), pages(x.scale, page), pages(x.zero, page), x.nbits, x.group_size, x.head_dim)


CASES = [(1, 2, 6, 4096, *f) for f in ((4, 128, 32), (2, 128, 32), (4, 64, 64), (2, 64, 16), (4, 128, 128), (2, 128, 16),
                                       (16, 128, 0))]
CASES += [(40, 8, 4, 2048, *f) for f in ((4, 128, 32), (2, 128, 32), (4, 64, 64), (16, 128, 0))]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("weight", [0.0, 0.3, 0.74, 0.95])
@pytest.mark.parametrize("B,HKV,G,S,nbits,D,gs", CASES)
def test_decode(B, HKV, G, S, nbits, D, gs, weight, size):
    """Contiguous and paged caches, one sequence and a batch."""
    q, k, v = inputs(B, HKV, G, S, D, size, weight, seed=B + nbits + gs)
    if nbits < 16:
        k, v = (quantize_groupwise(x, nbits, gs) for x in (k, v))
    ref = exact(q, values(k), values(v))
    one = fp16_decode_attention if nbits == 16 else fused_decode_attention
    allowed = bound(nbits, gs, size)
    close(one(q, k, v), ref, allowed, "contiguous")
    many = paged_fp16_decode_attention if nbits == 16 else paged_decode_attention
    for page in (16, 64):
        table = torch.arange(B * S // page, dtype=torch.int32, device=DEV).view(B, -1)
        lens = torch.full((B,), S, dtype=torch.int32, device=DEV)
        close(many(q, paged(k, page), paged(v, page), table, lens), ref, allowed, f"pages of {page}")


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("weight", [0.3, 0.95])
@pytest.mark.parametrize("nbits", [2, 4])
def test_per_channel_keys(nbits, weight, size):
    q, k, v = inputs(3, 2, 4, 4096, 128, size, weight, seed=nbits)
    cache = quantize_kv_kivi(k, v, nbits)
    ref = exact(q, Q.dequantize_keys_per_channel(cache.k), values(cache.v))
    close(kivi_decode_attention(q, cache), ref, bound(nbits, 32, size), "per channel")


@pytest.mark.parametrize("nbits", [2, 4])
def test_scales_at_the_end_of_float16(nbits):
    """Scales of 2^13 and more (the products of weight and scale have to stay finite), then small ones in the
    same sequence, and a scale that is infinite beside rows that are not attended with it."""
    S, D = 2048, 128
    q, k, v = inputs(2, 2, 4, S, D, 1.0, 0.3, seed=9)
    kq, vq = quantize_groupwise(k, nbits, 32), quantize_groupwise(v, nbits, 32)
    vq.scale[0, :, ::5] = 60000.0
    vq.scale[1, :, S // 2::31] = 9000.0
    ref = exact(q, values(kq), values(vq))
    close(fused_decode_attention(q, kq, vq), ref, bound(nbits, 32, 1.0), "contiguous")
    lens = torch.full((2,), S, dtype=torch.int32, device=DEV)
    table = torch.arange(2 * S // 32, dtype=torch.int32, device=DEV).view(2, -1)
    kp, vp = paged(kq, 32), paged(vq, 32)
    close(paged_decode_attention(q, kp, vp, table, lens), ref, bound(nbits, 32, 1.0), "paged")
    vp.scale[5] = float("inf")  # its page is a hole of the table below
    table[0, 5] = -1
    keep = torch.ones(S, dtype=torch.bool, device=DEV)
    keep[5 * 32:6 * 32] = False
    ref[0] = exact(q[:1], values(kq)[:1, :, keep], values(vq)[:1, :, keep])[0]
    close(paged_decode_attention(q, kp, vp, table, lens), ref, bound(nbits, 32, 1.0), "a hole")
