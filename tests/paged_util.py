"""Inputs and 64-bit references of the paged-cache tests."""

import math

import torch

from tritonkv_b200.quantize import QuantizedTensor, quantize_groupwise

DEV = "cuda"
H16 = 2.0 ** -11  # half a step of float16, relative


def values64(pool):
    """float64 values of a pool (..., D); for packed ones also the code*scale part, both exact."""
    if isinstance(pool, torch.Tensor):
        x = pool.double()
        return x, x.abs(), torch.zeros_like(x), torch.zeros_like(x)
    P, DP = 8 // pool.nbits, pool.packed.shape[-1]
    code = torch.cat([(pool.packed.long() >> (pool.nbits * p)) & (2 ** pool.nbits - 1) for p in range(P)], -1).double()
    s, z = (t.double().repeat_interleave(pool.group_size, -1) for t in (pool.scale, pool.zero))
    return code * s + z, code * s + z.abs(), code, s


def rows_of(pool, ids, n, at=None):
    """The first n token rows (HKV, n, ...) of the pages `ids` of a pool tensor."""
    t = pool[ids.long()]  # (pages, HKV, page, X)
    return t.transpose(0, 1).flatten(1, 2)[:, :n]


def gather(pool, ids, n):
    if isinstance(pool, torch.Tensor):
        return rows_of(pool, ids, n)
    return QuantizedTensor(rows_of(pool.packed, ids, n), rows_of(pool.scale, ids, n), rows_of(pool.zero, ids, n),
                           pool.nbits, pool.group_size, pool.head_dim)


def reference(q, kp, vp, table, lens, sm_scale=None, out_dtype=torch.float32):
    """(output, tolerance) in float64.

    The tolerance adds up what the kernels round, worst case, element by element.  A weight
    w_n = p_n / sum p is formed from p in float16: off by half a step, H16 relative, or -- below the
    normal range -- by 2^-25 where the largest p of its part of the history is 2^-4 or more: 2^-21 of the
    largest weight.  On packed pages the scale is multiplied in and rounded to float16 again, in
    front of the code.  The sum of the p is made of the rounded ones.  Scores are exact products
    summed in float32: their error is at most (D + 16) * 2^-24 of the sum of the terms'
    magnitudes (in the zero point, q sums enter as two float16 parts: 2^-22), and changes the
    weight by ln 2 times that, relative, in numerator and denominator.  The sums over n tokens run in float32
    over steps of 16."""
    B, HQ, D = q.shape
    page, NP, HKV = (kp if isinstance(kp, torch.Tensor) else kp.packed).shape[2], *(
        (kp if isinstance(kp, torch.Tensor) else kp.packed).shape[:2])
    scale = (1.0 / math.sqrt(D) if sm_scale is None else sm_scale) * math.log2(math.e)
    packed = not isinstance(kp, torch.Tensor)
    out = torch.zeros(B, HQ, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    G = HQ // HKV
    for b in range(B):
        n = min(max(int(lens[b]), 0), table.shape[1] * page)
        pages = -(-n // page)
        ids = table[b, :pages].long()
        ok = (ids >= 0) & (ids < NP)
        keep = ok.repeat_interleave(page)[:n]
        if n == 0 or not bool(keep.any()):
            continue
        ids = torch.where(ok, ids, 0)
        k, ka, _, _ = values64(gather(kp, ids, n))
        v, va, vc, vs = values64(gather(vp, ids, n))
        k, ka, v, va, vc, vs = (x[:, keep] for x in (k, ka, v, va, vc, vs))
        m = k.shape[1]
        qb = q[b].half().double().view(HKV, G, D)
        s = (qb @ k.transpose(1, 2)) * scale
        mag = (qb.abs() @ ka.transpose(1, 2)).amax(-1, keepdim=True) * abs(scale)
        w = torch.softmax(s * math.log(2.0), -1)
        o = w @ v
        wm = w.amax(-1, keepdim=True)
        lost = torch.maximum(H16 * w, 2.0 ** -21 * wm)
        e = lost @ va + o.abs() * lost.sum(-1, keepdim=True)
        if packed:
            e = e + H16 * (w @ (vc * vs)) + (2.0 ** -21 * wm) * vc.sum(1, keepdim=True)
        e = e + (w @ va) * (2 * math.log(2.0) * mag * ((D + 16) * 2.0 ** -24 + 2.0 ** -22 * 2)
                            + (m / 16 + 64) * 2.0 ** -23)
        out[b], tol[b] = o.reshape(HQ, D), e.reshape(HQ, D)
    half = {torch.float32: 2.0 ** -24, torch.float16: H16, torch.bfloat16: 2.0 ** -8}[out_dtype]
    small = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}[out_dtype]
    return out, tol * (1 + half) + out.abs() * half + small + 1e-30


def check(got, q, kp, vp, table, lens, what="", sm_scale=None):
    ref, tol = reference(q, kp, vp, table, lens, sm_scale, got.dtype)
    diff = (got.double() - ref).abs()
    worst = (diff / tol).nan_to_num(nan=float("inf"))
    i = int(worst.argmax())
    assert bool((diff <= tol).all()), (
        f"{what}: off by {diff.flatten()[i]:.3g} where {tol.flatten()[i]:.3g} is the bound "
        f"(value {ref.flatten()[i]:.4g}, at {i}); {int((~(diff <= tol)).sum())} of {diff.numel()} values")
    return float(worst.max())


def make_pools(lens, HKV, D, nbits, gs, page, seed, poison=True, spare=3, width=None):
    """(k pool, v pool, table, pages): pages in random order; rows behind a sequence's last token, spare
    pages and their metadata hold NaN and infinities when `poison`."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    need = [-(-max(n, 0) // page) for n in lens]
    NP = sum(need) + spare
    perm = torch.randperm(NP, generator=g).tolist()
    W = width or max(need + [1]) + 1
    table = torch.randint(-3, NP + 3, (len(lens), W), generator=g, dtype=torch.int64)  # what lies behind a row may be anything
    live = torch.zeros(NP, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for i in range(need[b]):
            p = perm.pop()
            table[b, i] = p
            live[p, : min(page, n - i * page)] = True
    x = [torch.randn(NP, HKV, page, D, generator=g) * torch.where(torch.rand(NP, HKV, page, D, generator=g) < 0.01, 5.0, 1.0)
         for _ in range(2)]
    x = [t.to(DEV).half() for t in x]
    dead = ~live.to(DEV)[:, None, :, None]
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")], device=DEV).half()
    pools = []
    for t in x:
        if nbits == 16:
            if poison:
                t = torch.where(dead, bad[torch.arange(D, device=DEV) % 3], t)
            pools.append(t.contiguous())
        else:
            qt = quantize_groupwise(t, nbits, gs)
            if poison:
                ng = qt.scale.shape[-1]
                junk = bad[torch.arange(ng, device=DEV) % 3]
                qt.scale.copy_(torch.where(dead, junk, qt.scale))
                qt.zero.copy_(torch.where(dead, junk, qt.zero))
            pools.append(qt)
    return pools[0], pools[1], table.to(torch.int32).to(DEV), NP
