"""Decode attention over paged caches against its definition in float64."""

import math

import pytest
import torch

from tritonkv_b200.kernels import (fused_decode_attention, paged_decode_attention,
                                   paged_fp16_decode_attention)
from tritonkv_b200.quantize import QuantizedTensor

from paged_util import DEV, check, make_pools

pytestmark = pytest.mark.gpu


def attend(q, k, v, table, lens, **kw):
    fn = paged_decode_attention if isinstance(k, QuantizedTensor) else paged_fp16_decode_attention
    return fn(q, k, v, table, lens, **kw)


def make_q(B, HQ, D, seed, dtype=torch.float16):
    return torch.randn(B, HQ, D, generator=torch.Generator().manual_seed(seed)).to(DEV).to(dtype)


def lens_t(lens):
    return torch.tensor(lens, dtype=torch.int32, device=DEV)


FORMATS = [(4, 128, 32), (4, 128, 16), (4, 128, 64), (4, 128, 128), (2, 128, 32), (2, 128, 16), (2, 128, 64),
           (2, 128, 128), (4, 64, 16), (4, 64, 32), (4, 64, 64), (2, 64, 16), (2, 64, 32), (2, 64, 64),
           (16, 128, 0), (16, 64, 0)]


@pytest.mark.parametrize("page", [16, 32, 48, 64, 128, 272])
@pytest.mark.parametrize("nbits,D,gs", FORMATS)
def test_formats_and_pages(nbits, D, gs, page):
    """Every format and page size, lengths around tiles and pages, empty rows, NaN behind the ends."""
    lens = [0, 1, 15, 16, 17, 31, 32, 33, page - 1, page, page + 1, 2 * page + 5, 700]
    k, v, table, _ = make_pools(lens, 2, D, nbits, gs, page, seed=page + D)
    q = make_q(len(lens), 6, D, seed=gs)
    out = attend(q, k, v, table, lens_t(lens))
    assert out.dtype == torch.float32
    check(out, q, k, v, table, lens, f"{nbits} bits D={D} gs={gs} page={page}")
    assert bool((out[0] == 0).all()), "an empty sequence gives zero"


@pytest.mark.parametrize("HQ,HKV", [(1, 1), (4, 4), (7, 1), (8, 1), (9, 1), (12, 1), (28, 4), (40, 2), (32, 8)])
@pytest.mark.parametrize("nbits,D,gs", [(4, 128, 32), (2, 64, 64), (16, 128, 0)])
def test_heads(HQ, HKV, nbits, D, gs):
    lens = [300, 0, 45]
    k, v, table, _ = make_pools(lens, HKV, D, nbits, gs, 16, seed=HQ)
    q = make_q(3, HQ, D, seed=HKV)
    check(attend(q, k, v, table, lens_t(lens)), q, k, v, table, lens, f"{HQ}/{HKV}")


@pytest.mark.parametrize("qdt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("odt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nbits", [4, 16])
def test_types(qdt, odt, nbits):
    lens = [513, 64]
    k, v, table, _ = make_pools(lens, 2, 128, nbits, 32, 32, seed=5)
    q = make_q(2, 8, 128, 6, qdt)
    out = torch.full((2, 8, 128), float("nan"), dtype=odt, device=DEV)
    assert attend(q, k, v, table, lens_t(lens), out=out) is out
    check(out, q, k, v, table, lens, f"{qdt} {odt}")


@pytest.mark.parametrize("nbits", [2, 4, 16])
@pytest.mark.parametrize("page", [16, 32, 64])
def test_entries_that_name_no_page(nbits, page):
    """Holes at the start, in the middle, at the end, and a row of nothing but holes: their tokens
    are not attended and nothing is read through them."""
    lens = [page * 6, page * 6 - 3, page * 5 + 1, page * 3, 400]
    k, v, table, NP = make_pools(lens, 2, 64, nbits, 32, page, seed=9)
    bad = [-1, NP, 2 ** 31 - 1, -2 ** 31, NP + 17]
    for i in range(3):
        table[0, i] = bad[i]
    table[1, 1], table[1, 3], table[1, 5] = bad[3], bad[4], bad[0]
    table[2, 5] = -1
    table[3, :] = -7
    q = make_q(len(lens), 4, 64, 1)
    out = attend(q, k, v, table, lens_t(lens))
    check(out, q, k, v, table, lens, f"holes, page {page}")
    assert bool((out[3] == 0).all())


@pytest.mark.parametrize("nbits", [4, 16])
def test_lengths_outside_the_table(nbits):
    """Negative lengths are empty rows, too long ones are cut to the table."""
    k, v, table, _ = make_pools([96, 96, 96], 1, 64, nbits, 32, 32, seed=2, width=3)
    q = make_q(3, 2, 64, 2)
    for lens in ([-5, 97, 2 ** 31 - 1], [-2 ** 31, 96, 95]):
        check(attend(q, k, v, table, lens_t(lens)), q, k, v, table, lens, str(lens))


@pytest.mark.parametrize("nbits,page", [(4, 16), (4, 128), (2, 64), (16, 16)])
@pytest.mark.parametrize("B,HKV,ctx", [(1, 2, 20011), (1, 1, 65536), (3, 8, 9000)])
def test_long(nbits, page, B, HKV, ctx):
    lens = [ctx - 777 * b for b in range(B)]
    k, v, table, _ = make_pools(lens, HKV, 128, nbits, 32, page, seed=ctx)
    q = make_q(B, HKV * 6, 128, 3)
    check(attend(q, k, v, table, lens_t(lens)), q, k, v, table, lens, "long")


@pytest.mark.parametrize("nbits", [4, 16])
@pytest.mark.parametrize("B", [300, 2100])
def test_many_sequences(nbits, B):
    lens = [(i * 37) % 90 for i in range(B)]
    k, v, table, _ = make_pools(lens, 1, 64, nbits, 32, 16, seed=B)
    q = make_q(B, 2, 64, 4)
    check(attend(q, k, v, table, lens_t(lens)), q, k, v, table, lens, "many")


@pytest.mark.parametrize("nbits", [2, 4, 16])
def test_one_sequence_among_short_ones(nbits):
    """One long history beside many short ones: the work is cut by tiles, not by sequences."""
    lens = [5, 30000, 0, 17, 64, 1, 0, 250]
    k, v, table, _ = make_pools(lens, 4, 128, nbits, 32, 32, seed=1)
    q = make_q(len(lens), 28, 128, 8)
    check(attend(q, k, v, table, lens_t(lens)), q, k, v, table, lens, "uneven")


def test_table_of_a_wider_one_and_shared_pages():
    """Rows that are slices of a wider table, and one page row used by every sequence (stride 0)."""
    lens = [200, 131]
    k, v, table, _ = make_pools(lens, 2, 128, 4, 32, 16, seed=3)
    wide = torch.full((2, table.shape[1] + 7), -1, dtype=torch.int32, device=DEV)
    wide[:, 5:5 + table.shape[1]] = table
    part = wide[:, 5:5 + table.shape[1]]
    q = make_q(2, 4, 128, 2)
    check(attend(q, k, v, part, lens_t(lens)), q, k, v, table, lens, "slice")
    same = table[:1].expand(2, -1)
    check(attend(q, k, v, same, lens_t([200, 77])), q, k, v, same, [200, 77], "stride 0")


def test_strided_q_scale_and_heavy_scores():
    k, v, table, _ = make_pools([333], 2, 64, 4, 16, 16, seed=4)
    q = make_q(1, 8, 128, 7)[:, :, ::2] * 4
    check(attend(q, k, v, table, lens_t([333]), sm_scale=0.5), q, k, v, table, [333], "scale", sm_scale=0.5)
    check(attend(q, k, v, table, lens_t([333]), sm_scale=-0.2), q, k, v, table, [333], "negative", sm_scale=-0.2)


def test_rising_scores():
    """Scores that rise along the history: the running maximum is raised at every tile."""
    for nbits in (4, 16):
        lens = [2048]
        k, v, table, _ = make_pools(lens, 1, 64, nbits, 32, 32, seed=8)
        ids = table[0, :64].long()
        ramp = (torch.arange(2048, device=DEV).view(64, 1, 32, 1) / 256).half()
        if nbits == 16:
            k[ids] = k[ids] * 0.1 + ramp
        else:
            k.zero[ids] = k.zero[ids] + ramp
        q = torch.ones(1, 3, 64, device=DEV).half()
        check(attend(q, k, v, table, lens_t(lens)), q, k, v, table, lens, f"rising {nbits}")


@pytest.mark.parametrize("power", [-8, -4, 8, 12])
@pytest.mark.parametrize("nbits", [2, 4, 16])
def test_small_and_large_values(nbits, power):
    """Values far from 1: weights times scales at both ends of float16."""
    lens = [700, 31]
    k, v, table, _ = make_pools(lens, 2, 64, nbits, 32, 32, seed=power + 20)
    for t in ([v] if nbits == 16 else [v.scale, v.zero]):
        t.mul_(2.0 ** power)
    q = make_q(2, 8, 64, 3)
    check(attend(q, k, v, table, lens_t(lens)), q, k, v, table, lens, f"2^{power}")


def test_agrees_with_the_contiguous_kernel():
    """Pages in order are the contiguous cache: the two kernels round alike."""
    from oracle.workloads import make_random_kv
    from tritonkv_b200.quantize import quantize_kv

    B, HQ, HKV, S, D = 3, 12, 2, 512, 128
    q, kc, vc = make_random_kv(B, HQ, HKV, S, D, device=DEV, seed=3)
    kq, vq = quantize_kv(kc, vc, 4, 32)
    lens = torch.tensor([512, 77, 300], dtype=torch.int32, device=DEV)
    want = fused_decode_attention(q, kq, vq, seq_lens=lens)

    def pages(t):
        return t.view(B, HKV, S // 64, 64, -1).transpose(1, 2).reshape(B * S // 64, HKV, 64, -1).contiguous()

    kp, vp = (QuantizedTensor(pages(x.packed), pages(x.scale), pages(x.zero), 4, 32, D) for x in (kq, vq))
    table = torch.arange(B * S // 64, dtype=torch.int32, device=DEV).view(B, -1)
    got = paged_decode_attention(q, kp, vp, table, lens)
    assert float((got - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max())


@pytest.mark.parametrize("nbits", [4, 16])
def test_streams_graphs_and_workspaces(nbits):
    """Captured once, replayed on grown lengths and another table; two graphs with a workspace each,
    replayed on two streams at once; the same numbers every time."""
    lens = [700, 129, 0, 1500]
    k, v, table, _ = make_pools(lens, 2, 128, nbits, 32, 32, seed=12)
    q = make_q(4, 8, 128, 13)
    sl, tb = lens_t(lens), table.clone()
    runs = []
    for i in range(2):
        out, ws, s = torch.empty(4, 8, 128, device=DEV), {}, torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            attend(q, k, v, tb, sl, out=out, _workspace=ws)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            attend(q, k, v, tb, sl, out=out, _workspace=ws)
        runs.append((g, out, s, ws))  # a captured call's workspace lives as long as its graph
    for now in (lens, [1500, 0, 3, 64], [0, 0, 0, 0]):
        sl.copy_(lens_t(now))
        if now is not lens:
            tb.copy_(table[[3, 1, 0, 0]])
        torch.cuda.synchronize()
        for _ in range(3):
            for g, _, s, _ in runs:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for _, out, _, _ in runs:
            check(out, q, k, v, tb, now, f"replayed {now}")
        assert torch.equal(runs[0][1], runs[1][1])
        assert torch.equal(attend(q, k, v, tb, sl), runs[0][1])


def test_graphed_step_over_pages():
    """The captured host-in, host-out step on a paged cache: equal to the direct call, as the lengths grow and
    the table moves."""
    from tritonkv_b200 import GraphedDecodeStep

    lens = [300, 77, 0]
    k, v, table, _ = make_pools([300, 90, 40], 2, 128, 4, 32, 16, seed=21)
    sl, tb = lens_t(lens), table.clone()
    step = GraphedDecodeStep(k, v, 6, seq_lens=sl, block_table=tb)
    for i in range(4):
        q = make_q(3, 6, 128, i)
        step.run(q.cpu())
        got = step.result().clone().to(DEV)
        assert torch.equal(got, attend(q, k, v, tb, sl))
        check(got, q, k, v, tb, sl.tolist(), f"step {i}")
        if i < 2:  # (what make_pools filled: up to 300, 90 and 40 tokens)
            sl.add_(lens_t([0, 4, 10]))
        if i == 1:
            tb.copy_(tb[[2, 1, 0]])
            sl.copy_(sl[[2, 1, 0]])


def test_no_allocation_with_workspace():
    k, v, table, _ = make_pools([900, 40], 2, 128, 4, 32, 16, seed=1)
    q, sl, out, ws = make_q(2, 8, 128, 1), lens_t([900, 40]), torch.empty(2, 8, 128, device=DEV), {}
    attend(q, k, v, table, sl, out=out, _workspace=ws)
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    attend(q, k, v, table, sl, out=out, _workspace=ws)
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before


@pytest.mark.parametrize("seed", range(40))
def test_random_batches(seed, ws={}):
    """Batches of every kind in turn, all with one workspace: few and many units, one merge and the other, ranges
    that cross units, skewed lengths, holes."""
    import random

    rng = random.Random(seed)
    D = rng.choice((64, 128))
    nbits, gs = rng.choice(((4, 32), (2, 16), (4, 64), (2, 64), (16, 0), (16, 0)))
    HKV, G, page = rng.choice((1, 2, 4, 8)), rng.choice((1, 3, 4, 8, 12)), rng.choice((16, 32, 48, 64, 128))
    B = rng.choice((1, 2, 3, 7, 16, 28, 40, 64, 100, 230))
    top = max(2, min(3000, 60000 // (B * HKV)))
    lens = [rng.choice((0, 1, rng.randrange(top), top, rng.randrange(1, 40))) for _ in range(B)]
    if seed % 4 == 0:
        lens[rng.randrange(B)] = 6 * top
    k, v, table, NP = make_pools(lens, HKV, D, nbits, gs, page, seed=seed)
    if seed % 3 == 0:
        for _ in range(B):
            table[rng.randrange(B), rng.randrange(table.shape[1])] = rng.choice((-1, NP, -2 ** 31))
    q = make_q(B, HKV * G, D, seed)
    out = torch.full((B, HKV * G, D), float("nan"), device=DEV)
    attend(q, k, v, table, lens_t(lens), out=out, _workspace=ws)
    check(out, q, k, v, table, lens, f"B={B} HKV={HKV} G={G} D={D} {nbits} bits page={page}")
    again = attend(q, k, v, table, lens_t(lens), _workspace=ws)
    assert torch.equal(out, again) and torch.equal(out, attend(q, k, v, table, lens_t(lens)))


def test_too_small_a_workspace_is_refused():
    from tritonkv_b200 import _cabi

    k, v, table, NP = make_pools([64], 1, 64, 4, 32, 16, seed=1)
    q, sl, out = make_q(1, 2, 64, 0), lens_t([64]), torch.empty(1, 2, 64, device=DEV)
    pools = [t.data_ptr() for p in (k, v) for t in (p.packed, p.scale, p.zero)]
    rc = _cabi.load().tkv_paged_decode(_cabi.PAGED_DECODE_ARGS.pack(
        q.data_ptr(), *pools, table.data_ptr(), sl.data_ptr(), out.data_ptr(), out.data_ptr(), 0, table.stride(0), 64, 0, 2, 1,
        2, 1, NP, 16, table.shape[1], 64, 4, 32, 0.125), _cabi.stream_ptr(q.device))
    assert rc == _cabi.TKV_ERR_INVALID and "tkv_paged_workspace" in _cabi.last_error()


def test_pool_past_two_to_the_31_bytes():
    """Pages whose bytes lie past 2^31 and 2^32 of the pool."""
    D, page, HKV = 128, 64, 8
    NP = (9 << 29) // (HKV * page * D * 2)  # 4.5 GiB of float16 pages
    k = torch.zeros(NP, HKV, page, D, dtype=torch.float16, device=DEV)
    ids = [NP - 1, 0, NP // 2, NP - 2]
    small, sv, _, _ = make_pools([page * 4], HKV, D, 16, 0, page, seed=3, poison=False, spare=0)
    k[ids] = small
    table = torch.tensor([ids], dtype=torch.int32, device=DEV)
    v = torch.zeros_like(k)
    v[ids] = sv
    q = make_q(1, 16, D, 3)
    got = attend(q, k, v, table, lens_t([page * 4 - 5]))
    own = torch.arange(4, dtype=torch.int32, device=DEV)[None]
    check(got, q, small, sv, own, [page * 4 - 5], "far pages")


def test_empty_batch_and_empty_table():
    k, v, _, _ = make_pools([32], 1, 64, 4, 32, 16, seed=1)
    none = torch.zeros(0, 3, dtype=torch.int32, device=DEV)
    assert attend(make_q(0, 2, 64, 0), k, v, none, lens_t([])).shape == (0, 2, 64)
    out = attend(make_q(2, 2, 64, 0), k, v, torch.zeros(2, 0, dtype=torch.int32, device=DEV), lens_t([4, 0]))
    assert bool((out == 0).all())
    assert math.isfinite(float(out.sum()))
