"""Workloads of the paged-cache operators, with their plain forms.

A paged cache keeps the tokens of many sequences in one pool of equal pages.  Page ``i`` of
sequence ``b`` is pool page ``block_table[b, i]``; a pool holds, for every page and KV head,
``page`` token rows in this package's cache formats:

* packed: codes uint8 ``(pages, HKV, page, D*nbits/8)``, split-P, and float16 scale and zero
  ``(pages, HKV, page, D/group)``; the value is ``code * scale + zero``;
* float16: ``(pages, HKV, page, D)``.

Operators (``case["op"]``):

``decode``    attention of one new token over packed pages
``decode16``  the same over float16 pages
``append``    quantise new tokens of every sequence into its pages; also gives the values the
              cache now stands for, as a prompt's own attention wants them
``fork``      next round of sequences from the present ones: each new row continues a parent
              row, shares its full pages, gets a copy of a partly filled page that a brother
              continues too, and room for the tokens to come
``compact``   move the pages that are in use to the front of the pool

``own`` chooses between the framework's calls and the plain forms below.  Lengths follow from
the case alone (their order from the seed), so ``work`` knows them.
"""

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one user, a short chat on a 1.5B-class model with small pages: latency is all there is
        dict(name="decode one short", op="decode", B=1, HQ=12, HKV=2, D=128, nbits=4, group=32, page=16, ctx=500, low=500,
             empty=0, dtype="f16"),
        # a small serving batch of an 8B-class model, ragged lengths
        dict(name="decode batch 16", op="decode", B=16, HQ=32, HKV=8, D=128, nbits=4, group=32, page=64, ctx=4096, low=1024,
             empty=0, dtype="bf16"),
        # a full batch at 2 bits, the smallest pages, some slots of the batch idle
        dict(name="decode batch 64 2-bit", op="decode", B=64, HQ=32, HKV=8, D=128, nbits=2, group=32, page=16, ctx=4096,
             low=2048, empty=3, dtype="f16"),
        # one long document: few heads, the work is split along the history
        dict(name="decode one long", op="decode", B=1, HQ=12, HKV=2, D=128, nbits=4, group=32, page=128, ctx=65536, low=65536,
             empty=0, dtype="f16"),
        # float16 pages: a few ragged sequences with seven query heads to a KV head
        dict(name="decode16 batch 4", op="decode16", B=4, HQ=28, HKV=4, D=128, page=16, ctx=1000, low=37, empty=0,
             dtype="bf16"),
        # float16 pages: a serving batch
        dict(name="decode16 batch 32", op="decode16", B=32, HQ=32, HKV=8, D=128, page=32, ctx=4096, low=1024, empty=1,
             dtype="f16"),
        # write side of a decode step: one token for every sequence
        dict(name="append step", op="append", B=64, HKV=8, D=128, nbits=4, group=32, page=16, T=1, low=1, at=2047,
             dtype="f16"),
        # prompts of ragged length arriving together in a padded batch
        dict(name="append prompts", op="append", B=8, HKV=8, D=128, nbits=2, group=64, page=64, T=4000, low=700, at=0,
             dtype="bf16"),
        # one step of a beam search on a packed cache
        dict(name="fork beams", op="fork", groups=4, beams=4, HKV=2, D=128, nbits=4, group=32, page=16, ctx=700, reserve=1,
             ended=0),
        # many samples of many prompts on float16 pages, two prompts done, room for a draft of 8 tokens
        dict(name="fork samples", op="fork", groups=48, beams=8, HKV=8, D=128, nbits=16, group=0, page=64, ctx=2050, reserve=8,
             ended=2),
        # a small pool after a day of short chats
        dict(name="compact small", op="compact", pages=600, live=250, B=24, HKV=2, D=64, nbits=2, group=32, page=16),
        # a large pool of float16 pages, half of it in use
        dict(name="compact large", op="compact", pages=8000, live=4000, B=64, HKV=8, D=128, nbits=16, group=0, page=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("decode", "decode", "decode16", "append", "fork", "compact"))
    D = rng.choice((64, 128))
    HKV = rng.choice((1, 2, 4, 8))
    nbits = rng.choice((2, 4))
    group = rng.choice([g for g in (16, 32, 64, 128) if g <= D])
    page = rng.choice((16, 32, 48, 64, 128))
    if op in ("decode", "decode16"):
        ctx = _log(rng, 1, 65536)
        B = _log(rng, 1, max(1, min(200, (1 << 17) // ctx)))
        c = dict(op=op, B=B, HQ=HKV * rng.choice((1, 2, 4, 6, 7, 8, 12)), HKV=HKV, D=D, page=page, ctx=ctx,
                 low=_log(rng, 1, ctx), empty=rng.choice((0, 0, 1)) if B > 1 else 0, dtype=rng.choice(("f16", "bf16")))
        return c if op == "decode16" else dict(c, nbits=nbits, group=group)
    if op == "append":
        T = _log(rng, 1, 4000)
        return dict(op=op, B=_log(rng, 1, max(1, min(200, 32000 // T))), HKV=HKV, D=D, nbits=nbits, group=group, page=page, T=T,
                    low=_log(rng, 1, T), at=rng.randrange(3000), dtype=rng.choice(("f16", "bf16")))
    nbits = rng.choice((2, 4, 16))
    group = group if nbits < 16 else 0
    if op == "fork":
        groups = _log(rng, 1, 48)
        return dict(op=op, groups=groups, ended=groups // 8, beams=rng.randint(2, 8), HKV=HKV, D=D, nbits=nbits, group=group, page=page,
                    ctx=_log(rng, 20, 2050), reserve=rng.choice((0, 1, 8, 40)))
    pages = _log(rng, 40, 4000)
    return dict(op=op, pages=pages, live=rng.randint(pages // 4, pages * 9 // 10), B=rng.randint(2, 64), HKV=HKV, D=D,
                nbits=nbits, group=group, page=page)


# ------------------------------------------------------------------------------ inputs
def _lengths(c):
    """Lengths of a ragged batch: evenly spread over [low, ctx], `empty` of them zero."""
    n, hi = c["B"], c.get("ctx", c.get("T"))
    got = [c["low"] + (hi - c["low"]) * (i + 1) // n for i in range(n)]
    for i in range(min(c.get("empty", 0), n - 1)):
        got[i] = 0
    return got


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(g, shape, dtype, outliers=0.0):
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)
    if outliers:
        x *= torch.where(torch.rand(shape, generator=g, device=DEV) < outliers, 6.0, 1.0)
    return x.to(dtype)


def _quantise(x, nbits, group):
    """(codes in split-P bytes, scale, zero, value of every element) of float32 x (..., D)."""
    D, P = x.shape[-1], 8 // nbits
    g = x.unflatten(-1, (D // group, group))
    lo, hi = g.amin(-1), g.amax(-1)
    scale = (hi - lo) / hi.new_full((), 2.0 ** nbits - 1)
    scale = torch.where(scale > 0, scale, 1.0).half()
    zero = lo.half()
    s, z = scale.float()[..., None], zero.float()[..., None]
    code = ((g - z) / s).round().clamp(0, 2 ** nbits - 1)
    value = (code * s + z).flatten(-2)
    sl = code.flatten(-2).to(torch.uint8).unflatten(-1, (P, D // P))
    shift = nbits * torch.arange(P, device=x.device, dtype=torch.uint8)[:, None]
    return (sl << shift).sum(-2, dtype=torch.uint8), scale, zero, value


def _values(packed, scale, zero, nbits):
    """float32 values of packed rows."""
    P = 8 // nbits
    shift = nbits * torch.arange(P, device=packed.device, dtype=torch.uint8)[:, None]
    code = ((packed[..., None, :] >> shift) & (2 ** nbits - 1)).flatten(-2).float()
    code = code.unflatten(-1, (scale.shape[-1], -1))
    return (code * scale.float()[..., None] + zero.float()[..., None]).flatten(-2)


def _pool(c, g, pages, outliers=0.0):
    """One pool: a float16 tensor, or the three tensors of a packed one."""
    shape = (pages, c["HKV"], c["page"], c["D"])
    if c.get("nbits", 16) == 16:
        return {"x": _normal(g, shape, torch.float16, outliers)}
    packed, scale, zero, _ = _quantise(_normal(g, shape, torch.float32, outliers), c["nbits"], c["group"])
    return {"packed": packed, "scale": scale, "zero": zero}


def _table(rows, pages, width, rng):
    """Pool pages, in random order, for rows of (shared pages of an earlier row, own pages)."""
    ids = list(range(pages))
    rng.shuffle(ids)
    out = []
    for share, count, mine in rows:
        out.append((out[share][:count] if count else []) + [ids.pop() for _ in range(mine)])
    return torch.tensor([r + [-1] * (width - len(r)) for r in out], dtype=torch.int32, device=DEV), out


def _up(n, page):
    return -(-n // page)


def prepare(case, seed):
    c, g, rng = case, _gen(seed), random.Random(seed)
    st = {"case": c, "ws": {}}
    if c["op"] in ("decode", "decode16"):
        lens = _lengths(c)
        rng.shuffle(lens)
        need = [_up(n, c["page"]) for n in lens]
        pages = sum(need) + max(1, sum(need) // 8)
        st["table"], _ = _table([(0, 0, n) for n in need], pages, max(need) + 1, rng)
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        st["k"], st["v"] = _pool(c, g, pages, 0.01), _pool(c, g, pages)
        st["q"] = _normal(g, (c["B"], c["HQ"], c["D"]), DTYPES[c["dtype"]])
        st["out"] = torch.empty_like(st["q"])
    elif c["op"] == "append":
        lens = _lengths(c)
        rng.shuffle(lens)
        at = [max(0, c["at"] - 37 * i) for i in range(c["B"])]
        need = [_up(p + n, c["page"]) for p, n in zip(at, lens)]
        st["table"], _ = _table([(0, 0, n) for n in need], sum(need) + 3, max(need), rng)
        st["at"] = torch.tensor(at, dtype=torch.int32, device=DEV)
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        st["k"], st["v"] = _pool(c, g, sum(need) + 3), _pool(c, g, sum(need) + 3)
        # a projection gives (B, T, HKV, D): the operator takes the view with the heads in front
        for x in ("k", "v"):
            st[x + "_new"] = _normal(g, (c["B"], c["T"], c["HKV"], c["D"]), DTYPES[c["dtype"]], 0.01).transpose(1, 2)
            st[x + "_values"] = torch.zeros(c["B"], c["HKV"], c["T"], c["D"], dtype=DTYPES[c["dtype"]], device=DEV)
    elif c["op"] == "fork":
        lens, rows = _fork_rows(c)
        fresh = sum(mine for _, _, mine in rows)
        width = max(_up(n + c["reserve"], c["page"]) for n in lens) + 1
        pages = fresh + len(rows) * (1 + _up(c["reserve"], c["page"])) + 5
        st["table"], _ = _table(rows, pages, width, rng)
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        parents, W = [], c["beams"]
        for i in range(c["groups"]):
            alive = rng.sample(range(W), (W + 1) // 2)
            kids = [alive[j % len(alive)] for j in range(W)]
            rng.shuffle(kids)
            parents += [i * W + j if i >= c["ended"] else -1 for j in kids]
        st["parents"] = torch.tensor(parents, dtype=torch.int32, device=DEV)
        st["k"], st["v"] = _pool(c, g, pages), _pool(c, g, pages)
    else:
        rows, width = _compact_rows(c)
        st["table"], _ = _table(rows, c["pages"], width, rng)
        st["k"], st["v"] = _pool(c, g, c["pages"]), _pool(c, g, c["pages"])
    return st


def _fork_rows(c):
    """Lengths, and (earlier row, pages shared with it, own pages) of every beam of every group."""
    lens, rows = [], []
    for i in range(c["groups"]):
        n = max(1, c["ctx"] - 29 * (i % 16))
        common = (n * 3 // 4) // c["page"]
        for j in range(c["beams"]):
            shared = common if j else 0
            rows.append((i * c["beams"], shared, _up(n, c["page"]) - shared))
            lens.append(n)
    return lens, rows


def _compact_rows(c):
    """B rows with `live` pages of their own; every second row also shares three pages of the row before."""
    per = [c["live"] * (i + 1) // c["B"] - c["live"] * i // c["B"] for i in range(c["B"])]
    rows = [(i - 1, min(3, per[i - 1]), n) if i % 2 else (0, 0, n) for i, n in enumerate(per)]
    return rows, max(count + n for _, count, n in rows) + 2


# ------------------------------------------------------------------------------ one pass
def run(st):
    return _RUN[st["case"]["op"]](st)


def _tensors(st):
    return {a + "_" + n: t for a in ("k", "v") for n, t in st[a].items()}


def _framework(c, pool):
    """The framework's container of a packed pool (or the float16 tensor itself)."""
    if "x" in pool:
        return pool["x"]
    from tritonkv_b200 import QuantizedTensor

    return QuantizedTensor(pool["packed"], pool["scale"], pool["zero"], c["nbits"], c["group"], c["D"])


def _run_decode(st):
    c = st["case"]
    if own:
        from tritonkv_b200.kernels import paged_decode_attention

        return paged_decode_attention(st["q"], _framework(c, st["k"]), _framework(c, st["v"]), st["table"], st["lens"],
                                      out=st["out"], _workspace=st["ws"])
    k, v = (_values(**st[x], nbits=c["nbits"]) for x in ("k", "v"))
    return _plain_attention(st, k, v)


def _run_decode16(st):
    if own:
        from tritonkv_b200.kernels import paged_fp16_decode_attention

        return paged_fp16_decode_attention(st["q"], st["k"]["x"], st["v"]["x"], st["table"], st["lens"], out=st["out"],
                                           _workspace=st["ws"])
    return _plain_attention(st, st["k"]["x"].float(), st["v"]["x"].float())


def _plain_attention(st, k, v):
    """softmax(q k / sqrt(D)) v over the tokens that the table gives each sequence; zero for an empty one."""
    c, lens = st["case"], st["lens"]
    B, HQ, HKV, D = c["B"], c["HQ"], c["HKV"], c["D"]
    at = st["table"].clamp(min=0).long()
    k, v = (x[at].transpose(1, 2).flatten(2, 3) for x in (k, v))  # (B, HKV, tokens, D)
    q = st["q"].float().view(B, HKV, HQ // HKV, D) / math.sqrt(D)
    s = q @ k.transpose(-1, -2)
    there = torch.arange(k.shape[2], device=DEV) < lens[:, None]
    s = torch.where(there[:, None, None], s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total > 0, total, 1.0)
    return o.reshape(B, HQ, D).to(st["q"].dtype)


def _run_append(st):
    c = st["case"]
    outs = dict(_tensors(st), k_values=st["k_values"], v_values=st["v_values"])
    if own:
        from tritonkv_b200.paged import append_kv_paged

        append_kv_paged(_framework(c, st["k"]), _framework(c, st["v"]), st["k_new"], st["v_new"], st["table"], st["at"],
                        lengths=st["lens"], k_values=st["k_values"], v_values=st["v_values"])
        return outs
    t = torch.arange(c["T"], device=DEV)
    pos = st["at"][:, None] + t
    keep = t < st["lens"][:, None]
    page = st["table"].gather(1, (pos // c["page"]).clamp(max=st["table"].shape[1] - 1).long())[keep].long()
    row = (pos % c["page"])[keep].long()
    _plain_write(st, "k", keep, page, row)
    _plain_write(st, "v", keep, page, row)
    return outs


def _plain_write(st, a, keep, page, row):
    c, pool, x = st["case"], st[a], st[a + "_new"]
    packed, scale, zero, value = _quantise(x.float(), c["nbits"], c["group"])
    st[a + "_values"].copy_(torch.where(keep[:, None, :, None], value.to(x.dtype), st[a + "_values"]))
    pool["packed"][page, :, row] = packed.transpose(1, 2)[keep]
    pool["scale"][page, :, row] = scale.transpose(1, 2)[keep]
    pool["zero"][page, :, row] = zero.transpose(1, 2)[keep]


def _run_fork(st):
    c = st["case"]
    if own:
        from tritonkv_b200.paged import fork_pages

        table, lens, missing = fork_pages([_framework(c, st["k"]), _framework(c, st["v"])], st["table"], st["lens"],
                                          st["parents"], reserve=c["reserve"], _workspace=st["ws"])
        return dict(_tensors(st), table=table, lens=lens, missing=missing)
    P, pages = c["page"], next(iter(st["k"].values())).shape[0]
    goes_on, par = st["parents"] >= 0, st["parents"].clamp(min=0).long()
    B, W = par.shape[0], st["table"].shape[1]
    n = torch.where(goes_on, st["lens"][par], 0)
    old = st["table"][par].long()
    full, held = n // P, (n + P - 1) // P
    col = torch.arange(W, device=DEV)
    first = torch.where((par[:, None] == par) & goes_on, torch.arange(B, device=DEV), B).amin(1) == torch.arange(B, device=DEV)
    last = old.gather(1, full[:, None].clamp(max=W - 1).long())[:, 0]
    copy = (held > full) & ~first & (last >= 0)
    kept = torch.where((col < full[:, None]) | ((col < held[:, None]) & first[:, None]), old, -1)
    used = torch.zeros(pages + 1, dtype=torch.bool, device=DEV)
    used[torch.where(kept >= 0, kept, pages)] = True
    free = (~used[:pages]).nonzero()[:, 0]  # lowest first
    want = torch.where(goes_on, (n + c["reserve"] + P - 1) // P, 0).clamp(max=W)
    count = copy.long() + (want - held).clamp(min=0)
    start = count.cumsum(0) - count
    rank = torch.where((col == full[:, None]) & copy[:, None], start[:, None],
                       torch.where((col >= held[:, None]) & (col < want[:, None]),
                                   (start + copy)[:, None] + col - held[:, None], -1))
    room = (rank >= 0) & (rank < free.shape[0])
    table = torch.where(room, free[rank.clamp(0, free.shape[0] - 1)], kept)
    src = last[copy]
    dst = table.gather(1, full[:, None].clamp(max=W - 1).long())[:, 0][copy]
    src, dst = src[dst >= 0], dst[dst >= 0]
    st["k"].update({k: t.index_copy_(0, dst, t[src]) for k, t in st["k"].items()})
    st["v"].update({k: t.index_copy_(0, dst, t[src]) for k, t in st["v"].items()})
    missing = (count.sum() - free.shape[0]).clamp(min=0).to(torch.int32).view(1)
    return dict(_tensors(st), table=table.to(torch.int32), lens=n, missing=missing)


def _run_compact(st):
    c = st["case"]
    if own:
        from tritonkv_b200.paged import compact_pages

        table, live = compact_pages([_framework(c, st["k"]), _framework(c, st["v"])], st["table"], _workspace=st["ws"])
        return dict(_tensors(st), table=table, live=live)
    pages, table = c["pages"], st["table"].long()
    used = torch.zeros(pages + 1, dtype=torch.bool, device=DEV)
    used[torch.where(table >= 0, table, pages)] = True
    used = used[:pages]
    live = used.sum()
    ids = torch.arange(pages, device=DEV)
    src, dst = (used & (ids >= live)).nonzero()[:, 0], (~used & (ids < live)).nonzero()[:, 0]
    moved = ids.index_copy(0, src, dst)
    st["k"].update({k: t.index_copy_(0, dst, t[src]) for k, t in st["k"].items()})
    st["v"].update({k: t.index_copy_(0, dst, t[src]) for k, t in st["v"].items()})
    table = torch.where(table >= 0, moved[table.clamp(min=0)], -1)
    return dict(_tensors(st), table=table.to(torch.int32), live=live.to(torch.int32).view(1))


_RUN = {"decode": _run_decode, "decode16": _run_decode16, "append": _run_append, "fork": _run_fork, "compact": _run_compact}


# ------------------------------------------------------------------------------ what a pass needs
def _row_bytes(c):
    """Bytes of one token of one KV head in one pool."""
    return 2 * c["D"] if c.get("nbits", 16) == 16 else c["D"] * c["nbits"] // 8 + 4 * (c["D"] // c["group"])


def work(case):
    c = case
    if c["op"] in ("decode", "decode16"):
        lens = _lengths(c)
        cache = 2 * sum(lens) * c["HKV"] * _row_bytes(c)
        table = 4 * sum(_up(n, c["page"]) for n in lens) + 4 * c["B"]
        return {"bytes": cache + table + 2 * 2 * c["B"] * c["HQ"] * c["D"], "flops": 4 * sum(lens) * c["HQ"] * c["D"]}
    if c["op"] == "append":
        n = sum(_lengths(c)) * c["HKV"]
        return {"bytes": 2 * n * (2 * 2 * c["D"] + _row_bytes(c)), "flops": 2 * n * c["D"] * 6}
    page = 2 * c["HKV"] * c["page"] * _row_bytes(c)
    if c["op"] == "fork":
        lens, rows = _fork_rows(c)
        W = max(_up(n + c["reserve"], c["page"]) for n in lens) + 1
        copies = sum(n % c["page"] > 0 for n in lens[c["ended"] * c["beams"]::c["beams"]]) * (c["beams"] - (c["beams"] + 1) // 2)
        return {"bytes": 2 * copies * page + 8 * len(rows) * W, "flops": 0}
    _, width = _compact_rows(c)
    moves = c["live"] * (c["pages"] - c["live"]) // c["pages"]
    return {"bytes": 2 * moves * page + 8 * c["B"] * width, "flops": 0}


# ------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    c, st = case, prepare(case, seed)
    if c["op"] in ("decode", "decode16"):
        return _exact_attention(c, st)
    if c["op"] == "append":
        return _exact_append(c, st)
    table = st["table"].tolist()
    if c["op"] == "fork":
        moves = _exact_fork(c, st, table)
    else:
        used = sorted({p for r in table for p in r if p >= 0})
        holes = sorted(set(range(len(used))) - set(used))
        moves = list(zip([p for p in used if p >= len(used)], holes))
    got = {}
    for name, t in _tensors(st).items():
        if t.dtype == torch.uint8:
            got[name] = None
            continue
        t = t.double()
        for s, d in moves:
            t[d] = t[s]
        got[name] = t
    return dict(got, **{n: None for n in (("table", "lens", "missing") if c["op"] == "fork" else ("table", "live"))})


def _exact_attention(c, st):
    lens, table = st["lens"].tolist(), st["table"].tolist()
    out = torch.zeros(c["B"], c["HQ"], c["D"], dtype=torch.float64, device=DEV)
    G = c["HQ"] // c["HKV"]
    for b, n in enumerate(lens):
        if n == 0:
            continue
        ids = torch.tensor(table[b][: _up(n, c["page"])], device=DEV)
        kv = []
        for a in ("k", "v"):
            if "x" in st[a]:
                x = st[a]["x"][ids].double()
            else:
                parts = [t[ids] for t in (st[a]["packed"], st[a]["scale"], st[a]["zero"])]
                byte = parts[0].long()
                code = torch.cat([byte // 2 ** (c["nbits"] * i) % 2 ** c["nbits"] for i in range(8 // c["nbits"])], -1).double()
                s, z = (t.double().repeat_interleave(c["group"], -1) for t in parts[1:])
                x = s * code + z
            kv.append(torch.cat(list(x), 1)[:, :n])  # (HKV, n, D)
        for h in range(c["HQ"]):
            s = kv[0][h // G] @ st["q"][b, h].double() / c["D"] ** 0.5
            out[b, h] = torch.softmax(s, 0) @ kv[1][h // G]
    return out


def _exact_append(c, st):
    lens, at, table = st["lens"].tolist(), st["at"].tolist(), st["table"].tolist()
    got = {n: (None if t.dtype == torch.uint8 else t.double()) for n, t in _tensors(st).items()}
    top = 2 ** c["nbits"] - 1
    for a in ("k", "v"):
        values = st[a + "_values"].double()
        for b, n in enumerate(lens):
            x = st[a + "_new"][b, :, :n].double()  # (HKV, n, D)
            groups = x.reshape(c["HKV"], n, -1, c["group"])
            low, high = groups.min(3).values, groups.max(3).values
            step = ((high - low) / top).half().double()
            step[high == low] = 1
            zero = low.half().double()
            code = torch.clamp(torch.round((groups - zero[..., None]) / step[..., None]), 0, top)
            values[b, :, :n] = (code * step[..., None] + zero[..., None]).reshape(c["HKV"], n, c["D"])
            where = [divmod(at[b] + t, c["page"]) for t in range(n)]
            pages = torch.tensor([table[b][i] for i, _ in where], device=DEV)
            rows = torch.tensor([r for _, r in where], device=DEV)
            got[a + "_scale"][pages, :, rows] = step.transpose(0, 1)
            got[a + "_zero"][pages, :, rows] = zero.transpose(0, 1)
        got[a + "_values"] = values
    return got


def _exact_fork(c, st, table):
    """(source, copy) pages, by walking the rows one after the other."""
    lens, parents, page = st["lens"].tolist(), st["parents"].tolist(), c["page"]
    used, seen = set(), set()
    parents = [p for p in parents if p >= 0]
    for p in parents:
        used.update(table[p][: lens[p] // page])
        if lens[p] % page:
            used.add(table[p][lens[p] // page])
    free = iter(sorted(set(range(next(iter(st["k"].values())).shape[0])) - used))
    moves = []
    for p in parents:
        n, copied = lens[p], False
        if n % page and p in seen:
            d = next(free, None)
            if d is not None:
                moves.append((table[p][n // page], d))
        seen.add(p)
        for _ in range(_up(n + c["reserve"], page) - _up(n, page)):
            next(free, None)
    return moves
