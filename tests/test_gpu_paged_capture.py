"""Paged-cache calls captured with a workspace that no call has used before, and that workspace afterwards."""

import pytest
import torch

from tritonkv_b200.kernels import paged_decode_attention, paged_fp16_decode_attention
from tritonkv_b200.paged import compact_pages, fork_pages

from paged_util import DEV, check, make_pools

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def warm():
    """The library's own one-time set-up, outside any capture."""
    k, v, table, _ = make_pools([40], 1, 64, 4, 32, 16, seed=1)
    for pool, fn in ((k, paged_decode_attention), (k.scale.repeat_interleave(32, -1).contiguous(), paged_fp16_decode_attention)):
        fn(torch.zeros(1, 2, 64, device=DEV).half(), pool, pool, table, ints([40]))
    compact_pages([k, v], table)
    torch.cuda.synchronize()


@pytest.mark.parametrize("nbits", [4, 16])
def test_attention_captured_first(nbits):
    warm()
    lens = [700, 129, 0, 1500]
    k, v, table, _ = make_pools(lens, 2, 64, nbits, 32, 32, seed=12)
    q, sl, ws = torch.randn(4, 8, 64, device=DEV).half(), ints(lens), {}
    fn = paged_fp16_decode_attention if nbits == 16 else paged_decode_attention
    fn(q, k, v, table, sl)
    torch.cuda.synchronize()
    graph, out = torch.cuda.CUDAGraph(), torch.empty(4, 8, 64, device=DEV)
    with torch.cuda.graph(graph):
        fn(q, k, v, table, sl, out=out, _workspace=ws)
    for _ in range(3):
        mine = torch.full_like(out, float("nan"))
        fn(q, k, v, table, sl, out=mine, _workspace=ws)
        check(mine, q, k, v, table, lens, "called directly")
        out.fill_(float("nan"))
        graph.replay()
        assert torch.equal(out, mine)


def test_pages_captured_first():
    warm()
    k, v, _, NP = make_pools([160], 1, 64, 4, 32, 16, seed=3)
    table, lens, par, ws = ints([[3, 4, -1], [5, -1, -1]]), ints([20, 3]), ints([1, 0, 0]), {}
    out = tuple(torch.zeros(s, dtype=torch.int32, device=DEV) for s in ((3, 3), (3,), (1,)))
    moved = tuple(torch.zeros(s, dtype=torch.int32, device=DEV) for s in ((3, 3), (1,)))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fork_pages([k, v], table, lens, par, reserve=1, out=out, _workspace=ws)
        compact_pages([k, v], out[0], out=moved, _workspace=ws)
    for _ in range(3):
        for direct in (True, False):
            for t in out + moved:
                t.fill_(-9)
            if direct:
                fork_pages([k, v], table, lens, par, reserve=1, out=out, _workspace=ws)
                compact_pages([k, v], out[0], out=moved, _workspace=ws)
            else:
                graph.replay()
            assert out[0].tolist() == [[5, -1, -1], [3, 4, -1], [3, 0, -1]] and out[2].tolist() == [0]
            assert moved[0].tolist() == [[2, -1, -1], [3, 1, -1], [3, 0, -1]] and moved[1].tolist() == [4]
            assert out[1].tolist() == [3, 20, 20]


def test_calls_in_turn_allocate_nothing():
    """Two pools and two shapes of the attention on one workspace: nothing new after the first round."""
    ws = {}
    work = []
    for lens, page, HKV in (([900, 40], 16, 2), ([30] * 40, 32, 4)):
        k, v, table, _ = make_pools(lens, HKV, 64, 4, 32, page, seed=page)
        q, sl = torch.randn(len(lens), 2 * HKV, 64, device=DEV).half(), ints(lens)
        o, par = torch.empty(len(lens), 2 * HKV, 64, device=DEV), ints(list(range(len(lens))))
        new = (torch.empty_like(table), torch.empty_like(sl), ints([0]))
        work.append((k, v, table, q, sl, o, par, new))

    def turn():
        for k, v, table, q, sl, o, par, new in work:
            paged_decode_attention(q, k, v, table, sl, out=o, _workspace=ws)
            fork_pages([k, v], table, sl, par, out=new, _workspace=ws)

    turn()
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    for _ in range(5):
        turn()
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before
