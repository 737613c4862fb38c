"""Write side and page management of a paged cache, against walks over the rows in Python."""

import pytest
import torch

from tritonkv_b200.kernels import paged_decode_attention, paged_fp16_decode_attention
from tritonkv_b200.paged import append_kv_paged, compact_pages, fork_pages
from tritonkv_b200.quantize import QuantizedTensor, dequantize_groupwise, empty_cache, quantize_groupwise

from paged_util import DEV, check, make_pools

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def tensors(pool):
    return [pool] if isinstance(pool, torch.Tensor) else [pool.packed, pool.scale, pool.zero]


def same(a, b):
    """Bit for bit, NaN included."""
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def random_pool(NP, HKV, page, D, nbits, gs, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(NP, HKV, page, D, generator=g, device=DEV).half()
    return x if nbits == 16 else quantize_groupwise(x, nbits, gs)


def copy_of(pool):
    if isinstance(pool, torch.Tensor):
        return pool.clone()
    return QuantizedTensor(pool.packed.clone(), pool.scale.clone(), pool.zero.clone(), pool.nbits, pool.group_size,
                           pool.head_dim)


# ------------------------------------------------------------------------------ append
def expect_append(pool, new, table, pos, lens):
    """The pool after the call, token by token."""
    want = copy_of(pool)
    rows = [new.half()] if isinstance(pool, torch.Tensor) else tensors(quantize_groupwise(new.clone(), pool.nbits, pool.group_size))
    NP, _, page, _ = tensors(pool)[0].shape
    written = torch.zeros(new.shape[0], new.shape[2], dtype=torch.bool)
    tab = table.tolist()
    for b in range(new.shape[0]):
        for t in range(min(lens[b], new.shape[2])):
            p = pos[b] + t
            if 0 <= p < len(tab[b]) * page and 0 <= tab[b][p // page] < NP:
                written[b, t] = True
                for w, r in zip(tensors(want), rows):
                    w[tab[b][p // page], :, p % page] = r[b, :, t]
    return want, written.to(DEV)


def make_new(B, HKV, T, D, dtype, seed, strided):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, T, HKV, D, generator=g) * torch.where(torch.rand(B, T, HKV, D, generator=g) < 0.02, 6.0, 1.0)
    x = x.to(DEV).to(dtype).transpose(1, 2)
    return x if strided else x.contiguous()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nbits,D,gs", [(4, 128, 32), (4, 128, 128), (2, 128, 16), (2, 64, 64), (4, 64, 16), (4, 64, 8),
                                        (4, 16, 8), (2, 32, 8), (4, 256, 64), (2, 256, 256), (16, 128, 0), (16, 64, 0),
                                        (16, 256, 0), (16, 16, 0)])
@pytest.mark.parametrize("T,strided", [(1, True), (1, False), (37, True), (40, False)])
def test_append(dtype, nbits, D, gs, T, strided):
    B, HKV, page = 5, 3, 16
    lens, pos = [T, 0, 1, T - 1, T + 9], [0, 5, 31, 14, 3]
    NP, W = 30, 5
    k, v = (random_pool(NP, HKV, page, D, nbits, gs, s) for s in (1, 2))
    table = torch.randperm(NP, generator=torch.Generator().manual_seed(T))[:B * W].view(B, W).to(torch.int32).to(DEV)
    kn, vn = (make_new(B, HKV, T, D, dtype, s, strided) for s in (3, 4))
    kn[0, 0, 0, : D // 2] = 1.5                              # a constant group
    vn[0, 1, 0, 0], vn[2, 2, 0, 1] = float("nan"), float("inf")
    want = [expect_append(p, n, table, pos, lens) for p, n in ((k, kn), (v, vn))]
    kval, vval = (torch.full_like(kn, 7.0) for _ in range(2))
    got = append_kv_paged(k, v, kn, vn, table, ints(pos), lengths=ints(lens), k_values=kval, v_values=vval)
    assert got[0] is k and got[1] is v
    for pool, new, val, (w, written) in zip((k, v), (kn, vn), (kval, vval), want):
        for a, b in zip(tensors(pool), tensors(w)):
            assert same(a, b)
        exact = (new.half().to(dtype) if nbits == 16 else
                 dequantize_groupwise(quantize_groupwise(new, nbits, gs), dtype=dtype))
        expect = torch.where(written[:, None, :, None], exact, 7.0)
        assert torch.equal(val.nan_to_num(nan=9.0, posinf=8.0), expect.nan_to_num(nan=9.0, posinf=8.0))


@pytest.mark.parametrize("nbits", [4, 16])
def test_append_drops_what_has_no_place(nbits):
    """Positions before and behind the table, entries that name no page: nothing else changes."""
    B, HKV, D, page, NP = 6, 2, 64, 16, 9
    k, v = (random_pool(NP, HKV, page, D, nbits, 32, s) for s in (1, 2))
    table = ints([[0, 1], [-1, 2], [NP, 3], [2 ** 31 - 1, 4], [5, -2 ** 31], [6, 7]])
    pos, lens = [-3, 10, 12, 0, 14, 2 ** 31 - 4], [20, 20, 20, 20, 20, 20]
    kn, vn = (make_new(B, HKV, 20, D, torch.float16, s, False) for s in (3, 4))
    want = [expect_append(p, n, table, pos, lens)[0] for p, n in ((k, kn), (v, vn))]
    append_kv_paged(k, v, kn, vn, table, ints(pos))
    for pool, w in zip((k, v), want):
        for a, b in zip(tensors(pool), tensors(w)):
            assert same(a, b)


def test_append_int_position_offsets_and_wide_table():
    """positions as an int, new tokens that start off a 16-byte boundary, a table cut from a wider one, and a
    long prompt over odd pages."""
    B, HKV, D, page = 2, 2, 128, 24
    T = 1000
    k = empty_cache(100, HKV, page, D, 4, 32, DEV)
    v = empty_cache(100, HKV, page, D, 4, 32, DEV)
    W = 44
    wide = torch.randperm(100, generator=torch.Generator().manual_seed(0))[:88].to(torch.int32).to(DEV)
    big = torch.full((2, 60), -1, dtype=torch.int32, device=DEV)
    big[:, 3:47] = wide.view(2, W)
    table = big[:, 3:47]
    buf = torch.randn(B * HKV * T * D + 1, device=DEV).half()
    kn = buf[1:].view(B, HKV, T, D)
    vn = make_new(B, HKV, T, D, torch.float16, 1, True)
    want = [expect_append(p, n, table, [11] * B, [T] * B)[0] for p, n in ((k, kn), (v, vn))]
    append_kv_paged(k, v, kn, vn, table, 11)
    for pool, w in zip((k, v), want):
        for a, b in zip(tensors(pool), tensors(w)):
            assert same(a, b)


def test_append_values_of_one_side_and_nothing_to_do():
    k, v = (random_pool(4, 1, 16, 64, 4, 32, s) for s in (1, 2))
    kn = make_new(1, 1, 3, 64, torch.float16, 1, False)
    val = torch.zeros(1, 1, 3, 64, dtype=torch.float16, device=DEV)
    append_kv_paged(k, v, kn, kn, ints([[2]]), 0, v_values=val)
    assert torch.equal(val, dequantize_groupwise(quantize_groupwise(kn, 4, 32), dtype=torch.float16))
    before = [t.clone() for t in tensors(k)]
    append_kv_paged(k, v, kn[:, :, :0], kn[:, :, :0], ints([[2]]), 0)
    append_kv_paged(k, v, kn[:0], kn[:0], torch.zeros(0, 2, dtype=torch.int32, device=DEV), 0)
    assert all(same(a, b) for a, b in zip(before, tensors(k)))


# ------------------------------------------------------------------------------ fork
def walk_fork(table, lens, parents, reserve, NP, page):
    """(table, lens, missing, copies) row by row."""
    W = len(table[0]) if table else 0
    ok = lambda p: 0 <= p < NP
    used, seen, rows = set(), set(), []
    for b, p in enumerate(parents):
        row, n, copy = [-1] * W, 0, None
        if 0 <= p < len(table):
            n = min(max(lens[p], 0), W * page)
            full, held = n // page, -(-n // page)
            keep = held if p not in seen else full
            row[:keep] = [x if ok(x) else -1 for x in table[p][:keep]]
            if held > full and p in seen and ok(table[p][full]):
                copy = table[p][full]
            seen.add(p)
            used.update(x for x in row if x >= 0)
        rows.append((row, n, copy))
    free = [p for p in range(NP) if p not in used]
    out, copies, missing = [], [], 0
    for b, (row, n, copy) in enumerate(rows):
        places = []
        if 0 <= parents[b] < len(table):
            held = -(-n // page)
            places = ([n // page] if copy is not None else []) + list(range(held, min(W, -(-(n + max(0, reserve[b])) // page))))
        for i in places:
            if free:
                row[i] = free.pop(0)
                if copy is not None and i == n // page:
                    copies.append((copy, row[i]))
            else:
                missing += 1
        out.append(row)
    return out, [n for _, n, _ in rows], missing, copies


def check_fork(pools, table, lens, parents, reserve, per_row=False):
    NP, _, page, _ = tensors(pools[0])[0].shape
    before = [[t.clone() for t in tensors(p)] for p in pools]
    B = len(parents)
    got = fork_pages(pools, ints(table).view(len(table), -1), ints(lens), ints(parents),
                     reserve=ints(reserve) if per_row else reserve)
    want = walk_fork(table, lens, parents, reserve if per_row else [reserve] * B, NP, page)
    assert got[0].tolist() == want[0]
    assert got[1].tolist() == want[1]
    assert got[2].tolist() == [want[2]]
    for old, p in zip(before, pools):
        for o, t in zip(old, tensors(p)):
            for s, d in want[3]:
                o[d] = o[s]
            assert same(o, t)
    return got, want


def random_table(B, W, NP, page, seed, full=False):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randperm(NP, generator=g).tolist()
    lens, table = [], []
    for b in range(B):
        n = int(torch.randint(0, W * page + 1, (1,), generator=g))
        need = -(-n // page)
        if len(ids) < need:
            n = need = 0
        table.append([ids.pop() for _ in range(need)] + [-1] * (W - need))
        lens.append(n)
    return table, lens


@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("seed", range(4))
def test_fork(page, seed):
    B, W, NP = 9, 6, 70
    table, lens = random_table(B, W, NP, page, seed)
    g = torch.Generator().manual_seed(seed)
    pools = [random_pool(NP, 2, page, 64, 4, 32, 1), random_pool(NP, 1, page, 128, 16, 0, 2)]
    for parents in (list(range(B)), torch.randint(-1, B, (B,), generator=g).tolist(),
                    torch.randint(0, 3, (17,), generator=g).tolist(), [B, -7, 2 ** 31 - 1, -2 ** 31, 0, 0, 0]):
        check_fork(pools, table, lens, parents, 0)
        check_fork(pools, table, lens, parents, page * 2 + 1)
        per = torch.randint(-2, 3 * page + 1, (len(parents),), generator=g).tolist()
        check_fork(pools, table, lens, parents, per, per_row=True)


def test_fork_holes_and_lengths_outside():
    """Entries that name no page stay holes and are not copied; lengths are cut to the table."""
    NP, page = 12, 8
    pools = [random_pool(NP, 1, page, 64, 2, 16, 1)]
    table = [[3, NP, 5], [-4, 2 ** 31 - 1, 6], [7, 8, 9], [1, 2, -1]]
    for lens in ([20, 13, 24, 17], [-5, 2 ** 31 - 1, 1, 0], [9, 9, 9, 9]):
        check_fork(pools, table, lens, [0, 0, 1, 1, 2, 2, 3, 3], 3)


def test_fork_out_of_pages():
    NP, page = 10, 4
    pools = [random_pool(NP, 2, page, 64, 4, 32, 1), random_pool(NP, 2, page, 64, 4, 32, 2)]
    table = [[0, 1, 2, -1, -1], [3, 4, 5, -1, -1]]
    got, want = check_fork(pools, table, [10, 11], [0, 0, 1, 1, 1, -1], 9)
    assert want[2] > 0


def test_fork_keeps_nothing_then_starts_again():
    """Everything freed, then rows started from nothing: the lowest pages in order."""
    pools = [random_pool(40, 1, 16, 64, 16, 0, 1)]
    t, n, _ = fork_pages(pools, ints([[9, 8, 7, 6], [5, 4, -1, -1]]), ints([64, 20]), ints([-1, -1]))
    assert t.tolist() == [[-1] * 4] * 2 and n.tolist() == [0, 0]
    t, n, miss = fork_pages(pools, t, n, ints([0, 1]), reserve=ints([33, 16]))
    assert t.tolist() == [[0, 1, 2, -1], [3, -1, -1, -1]] and n.tolist() == [0, 0] and miss.tolist() == [0]


@pytest.mark.parametrize("NP", [31, 33, 70000])
def test_fork_large(NP):
    """Many rows, many pages: the scans go over several rounds."""
    B, page, W = (2500, 16, 20) if NP > 1000 else (4, 16, 5)
    table, lens = random_table(B, W, NP, page, 3)
    pools = [random_pool(NP, 1, page, 16, 16, 0, 1)]
    parents = [(i * 7) % B if i % 5 else (i // 2) % B for i in range(B)]
    check_fork(pools, table, lens, parents, 40)


def test_fork_many_layers():
    """K and V of many layers under one table: more tensors than one launch takes."""
    NP, page = 20, 16
    pools = [random_pool(NP, 1, page, 64, 4, 32, i) for i in range(22)] + [random_pool(NP, 1, page, 64, 16, 0, 99)]
    check_fork(pools, [[4, 5, 6], [7, -1, -1]], [40, 9], [0, 0, 0, 1, 1], 1)


def test_fork_into_given_tensors_and_refusals():
    pools = [random_pool(12, 1, 16, 64, 4, 32, 1)]
    table, lens, par = ints([[3, 4], [5, -1]]), ints([20, 3]), ints([1, 0, 0])
    out = (torch.zeros(3, 2, dtype=torch.int32, device=DEV), ints([9, 9, 9]), ints([9]))
    ws = {}
    got = fork_pages(pools, table, lens, par, reserve=1, out=out, _workspace=ws)
    assert all(a is b for a, b in zip(got, out))
    assert got[0].tolist() == [[5, -1], [3, 4], [3, 0]] and got[1].tolist() == [3, 20, 20]
    big = torch.zeros(6, 2, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="share memory"):
        fork_pages(pools, big[:2], lens, par, out=(big[1:4], out[1], out[2]))
    with pytest.raises(ValueError, match=r"out\[0\]"):
        fork_pages(pools, table, lens, par, out=(out[0][:2], out[1], out[2]))
    with pytest.raises(ValueError, match="share memory"):
        compact_pages(pools, big[:2], out=(big[:2], out[2]))


# ------------------------------------------------------------------------------ compact
def walk_compact(table, NP):
    used = sorted({p for r in table for p in r if 0 <= p < NP})
    n, among = len(used), set(used)
    holes = [p for p in range(n) if p not in among]
    to = dict(zip([p for p in used if p >= n], holes))
    return [[to.get(p, p) if 0 <= p < NP else -1 for p in r] for r in table], n, list(to.items())


def check_compact(pools, table):
    NP = tensors(pools[0])[0].shape[0]
    before = [[t.clone() for t in tensors(p)] for p in pools]
    old = ints(table).view(len(table), -1)
    got, live = compact_pages(pools, old)
    want, n, moves = walk_compact(table, NP)
    assert got.tolist() == want and live.tolist() == [n]
    assert old.tolist() == table
    for o, p in zip(before, pools):
        for x, t in zip(o, tensors(p)):
            if moves:
                x[[d for _, d in moves]] = x[[s for s, _ in moves]]
            assert same(x, t)


@pytest.mark.parametrize("NP", [1, 31, 32, 33, 64, 500])
@pytest.mark.parametrize("nbits,page", [(4, 16), (16, 32), (2, 3)])
def test_compact(NP, nbits, page):
    pools = [random_pool(NP, 2, page, 64, nbits, 16, s) for s in (1, 2)]
    g = torch.Generator().manual_seed(NP)
    for share in (0.0, 0.1, 0.5, 0.9, 1.0):
        ids = torch.randperm(NP, generator=g).tolist()[: int(NP * share)]
        W = 7
        ids += [-1] * (-len(ids) % W) or [-1] * (0 if ids else W)
        table = [ids[i:i + W] for i in range(0, len(ids), W)]
        table.append([table[0][0], NP, -9, 2 ** 31 - 1, -2 ** 31, table[-1][0], -1])  # shared pages, holes
        check_compact(pools, table)


def test_compact_large_pool():
    """More pages than one round of the scans takes, and moves by the ten thousand."""
    NP = 150000
    pools = [torch.arange(NP * 8, device=DEV, dtype=torch.int32).view(torch.float16).view(NP, 1, 1, 16)]
    ids = torch.randperm(NP, generator=torch.Generator().manual_seed(1))[:70000].tolist()
    check_compact(pools, [ids[i:i + 1000] for i in range(0, 70000, 1000)])


def test_compact_into_given_tensors_and_empty():
    pools = [random_pool(8, 1, 16, 64, 4, 32, 1)]
    out = (torch.zeros(1, 2, dtype=torch.int32, device=DEV), ints([7]))
    got = compact_pages(pools, ints([[6, 2]]), out=out, _workspace={})
    assert got[0] is out[0] and out[0].tolist() == [[1, 0]] and got[1] is out[1] and out[1].tolist() == [2]
    t, n = compact_pages(pools, torch.zeros(0, 4, dtype=torch.int32, device=DEV))
    assert t.shape == (0, 4) and n.tolist() == [0]
    t, n = compact_pages(pools, torch.zeros(3, 0, dtype=torch.int32, device=DEV))
    assert t.shape == (3, 0) and n.tolist() == [0]


def test_one_workspace_for_many_calls():
    """Forks and compactions of different sizes and pools in turn with one workspace."""
    ws = {}
    for i in range(12):
        NP, B, W, page = [(70, 9, 6, 16), (500, 40, 9, 32), (33, 3, 4, 16)][i % 3]
        pools = [random_pool(NP, 1, page, 64, 4, 32, i)]
        table, lens = random_table(B, W, NP, page, i)
        parents = [(j * 5 + i) % (B + 1) - 1 for j in range(B)]
        want = walk_fork(table, lens, parents, [3] * B, NP, page)
        t, n, miss = fork_pages(pools, ints(table), ints(lens), ints(parents), reserve=3, _workspace=ws)
        assert (t.tolist(), n.tolist(), miss.tolist()) == (want[0], want[1], [want[2]])
        c, live = compact_pages(pools, t, _workspace=ws)
        assert (c.tolist(), live.tolist()) == (walk_compact(t.tolist(), NP)[0], [walk_compact(t.tolist(), NP)[1]])


# ------------------------------------------------------------------------------ together
@pytest.mark.parametrize("nbits", [2, 4, 16])
@pytest.mark.parametrize("captured", [False, True])
def test_a_served_batch(nbits, captured):
    """Prompts arrive, tokens are generated, beams fork, sequences end, the pool is compacted: after
    every round the attention equals the definition on the tokens that each row has seen."""
    HKV, HQ, D, page, NP, W, B = 2, 6, 64, 16, 60, 8, 5
    gs = 32
    pools = [random_pool(NP, HKV, page, D, nbits, gs, s) for s in (1, 2)]
    fn = paged_fp16_decode_attention if nbits == 16 else paged_decode_attention
    table = torch.full((B, W), -1, dtype=torch.int32, device=DEV)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(4)
    seen = [[] for _ in range(B)]  # (k, v) rows of every sequence, float16 (HKV, D)

    def rand(*shape):
        return torch.randn(*shape, generator=g).half().to(DEV)

    def compare(what):
        L = [len(s) for s in seen]
        assert lens.tolist() == L, what
        q = rand(B, HQ, D)
        got = fn(q, *pools, table, lens)
        ids, kp, vp = [], [], []
        flat = [[torch.stack([x[i] for x in s]) if s else torch.zeros(0, HKV, D, device=DEV).half() for s in seen] for i in range(2)]
        T = max(L)
        own = [torch.zeros(B, HKV, T, D, device=DEV).half() for _ in range(2)]
        for i in range(2):
            for b in range(B):
                own[i][b, :, : L[b]] = flat[i][b].transpose(0, 1)
        ref = own if nbits == 16 else [quantize_groupwise(x, nbits, gs) for x in own]
        pages = torch.arange(B, dtype=torch.int32, device=DEV)[:, None]
        check(got, q, ref[0], ref[1], pages, L, what)

    # the captured step: reserve, append, grow, on tensors that stay where they are
    step_k, step_v = rand(B, HKV, 1, D), rand(B, HKV, 1, D)
    alive = torch.ones(B, dtype=torch.int32, device=DEV)
    same_rows = torch.arange(B, dtype=torch.int32, device=DEV)
    out, ws = (torch.empty_like(table), torch.empty_like(lens), ints([0])), {}

    def step():
        fork_pages(pools, table, lens, same_rows, reserve=alive, out=out, _workspace=ws)
        table.copy_(out[0])
        append_kv_paged(*pools, step_k, step_v, table, lens, lengths=alive)
        lens.add_(alive)

    graph = None
    for rnd in range(6):
        if rnd in (0, 3):  # prompts into the rows that are free
            T = 37
            want = [T - 9 * b if not seen[b] else 0 for b in range(B)]
            t, n, miss = fork_pages(pools, table, lens, ints([b for b in range(B)]), reserve=ints(want))
            assert miss.tolist() == [0]
            table.copy_(t)
            k, v = rand(B, T, HKV, D).transpose(1, 2), rand(B, T, HKV, D).transpose(1, 2)
            append_kv_paged(*pools, k, v, table, lens, lengths=ints(want))
            lens.add_(ints(want))
            for b in range(B):
                seen[b] += [(k[b, :, t], v[b, :, t]) for t in range(want[b])]
            compare(f"prompts {rnd}")
        for _ in range(7):
            on = [1 if seen[b] and len(seen[b]) < W * page else 0 for b in range(B)]
            alive.copy_(ints(on))
            step_k.copy_(rand(B, HKV, 1, D))
            step_v.copy_(rand(B, HKV, 1, D))
            if captured and graph is None:
                s = torch.cuda.Stream()
                s.wait_stream(torch.cuda.current_stream())
                keep = [x.clone() for x in (table, lens)]
                with torch.cuda.stream(s):
                    step()
                s.synchronize()
                table.copy_(keep[0]), lens.copy_(keep[1])
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=s):
                    step()
            graph.replay() if captured else step()
            assert out[2].tolist() == [0]
            for b in range(B):
                if on[b]:
                    seen[b] = seen[b] + [(step_k[b, :, 0].clone(), step_v[b, :, 0].clone())]
        compare(f"steps {rnd}")
        parents = [[0, 0, 2, 2, 2], [4, 3, 2, 1, 0], [1, 1, -1, 3, 3], [0, 1, 2, 3, 4], [3, 3, 3, 3, 3], [0, -1, 1, -1, 2]][rnd]
        t, n, miss = fork_pages(pools, table, lens, ints(parents))
        assert miss.tolist() == [0]
        table.copy_(t), lens.copy_(n)
        seen = [list(seen[p]) if p >= 0 else [] for p in parents]
        compare(f"fork {rnd}")
        if rnd % 2:
            t, live = compact_pages(pools, table)
            table.copy_(t)
            assert int(live) == len({p for r in t.tolist() for p in r if p >= 0}) and int(table.max()) == int(live) - 1
            compare(f"compact {rnd}")
