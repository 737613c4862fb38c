"""Paged KV cache: tokens of many sequences in one pool of equal pages.

A pool is a cache whose first axis is pages instead of sequences:

* packed -- a :class:`~tritonkv_b200.quantize.QuantizedTensor` with ``packed`` of shape
  ``(num_pages, HKV, page_size, head_dim*nbits/8)``, made with
  ``quantize.empty_cache(num_pages, HKV, page_size, head_dim, nbits, group_size, device)``;
* float16 -- a tensor ``(num_pages, HKV, page_size, head_dim)``.

Page ``i`` of sequence ``b`` is pool page ``block_table[b, i]`` (int32, -1 for none), so token
``n`` of sequence ``b`` lies in row ``n % page_size`` of page ``block_table[b, n // page_size]``.
An entry outside ``[0, num_pages)`` names no page: reading skips its tokens, writing drops them.
Which pages are in use is read off the table by every call; there is no other state.

Attention over such a cache: ``kernels.paged_decode_attention`` and
``kernels.paged_fp16_decode_attention``.  Every function here enqueues on the current stream of
the tensors' device and returns without waiting for it; none has a counterpart in the reference,
whose caches are contiguous.
"""

from __future__ import annotations

import ctypes
import struct

import torch

from . import _cabi
from .quantize import QuantizedTensor, check_cache_tensors

_U8, _F16, _I32 = torch.uint8, torch.float16, torch.int32


def pool_tensors(pool, what: str) -> tuple[torch.Tensor, ...]:
    """The contiguous 4-D tensors of a pool; the kernels use them in place."""
    if isinstance(pool, QuantizedTensor):
        p, s, z = pool.packed, pool.scale, pool.zero
        a, b = p.shape, s.shape
        # a well-formed pool passes here; a decode step is a few microseconds, so no more is spent on it
        if (len(a) == 4 and len(b) == 4 and p.dtype is _U8 and s.dtype is _F16 and z.dtype is _F16 and z.shape == b
                and a[0] == b[0] and a[1] == b[1] and a[2] == b[2] and a[3] * 8 == pool.head_dim * pool.nbits
                and b[3] * pool.group_size == pool.head_dim and p.is_contiguous() and s.is_contiguous()
                and z.is_contiguous() and p.get_device() == s.get_device() == z.get_device()):
            return p, s, z
        check_cache_tensors(pool, what, p.device)
        if len(a) != 4 or len(b) != 4 or b[:3] != a[:3] or z.shape != b:
            raise ValueError(f"{what}: a packed pool has packed (num_pages, HKV, page_size, bytes) and scale, zero "
                             f"(num_pages, HKV, page_size, groups); got {[tuple(x.shape) for x in (p, s, z)]}")
        if a[3] * 8 != pool.head_dim * pool.nbits or b[3] * pool.group_size != pool.head_dim:
            raise ValueError(f"{what}: rows of {a[3]} bytes and {b[3]} groups are not those of head_dim {pool.head_dim} "
                             f"at {pool.nbits} bits in groups of {pool.group_size}")
    elif isinstance(pool, torch.Tensor):
        if pool.dtype is not _F16:
            raise TypeError(f"{what} must be a QuantizedTensor or a float16 tensor, got {pool.dtype}")
        if pool.dim() != 4:
            raise ValueError(f"{what}: a float16 pool is (num_pages, HKV, page_size, head_dim), got {tuple(pool.shape)}")
        if pool.is_contiguous():
            return (pool,)
    else:
        raise TypeError(f"{what} must be a QuantizedTensor or a float16 tensor, got {type(pool).__name__}")
    raise ValueError(f"{what} must be contiguous: a pool is used in place")


def _on(where: int) -> str:
    return f"cuda:{where}" if where >= 0 else "the pools' device"


def check_table(block_table: torch.Tensor, B: int | None, where: int) -> tuple[int, int]:
    """(entries per row, row stride) of an int32 table (B, max_pages) on device ``where`` whose rows are contiguous."""
    shape = block_table.shape
    if len(shape) != 2 or block_table.dtype is not _I32 or block_table.get_device() != where:
        raise ValueError(f"block_table must be an int32 tensor (B, max_pages) on {_on(where)}")
    if B is not None and shape[0] != B:
        raise ValueError(f"block_table has {shape[0]} rows for {B} sequences")
    stride = block_table.stride()
    if shape[1] > 1 and stride[1] != 1:
        raise ValueError("block_table rows must be contiguous")
    return shape[1], stride[0]


def check_lens(lens: torch.Tensor, B: int, where: int, what: str) -> torch.Tensor:
    shape = lens.shape
    if len(shape) != 1 or shape[0] != B or lens.dtype is not _I32 or lens.get_device() != where:
        raise ValueError(f"{what} must be an int32 tensor of shape ({B},) on {_on(where)}")
    return lens if lens.is_contiguous() else lens.contiguous()


def _row_strides(x: torch.Tensor) -> tuple | None:
    """Strides of (B, HKV, T) of a 4-D tensor whose rows are contiguous and start on 16-byte boundaries."""
    b, h, t, d = x.stride()
    al = 16 // x.element_size() - 1
    if not (b | h | t) & al and d == 1 and not x.data_ptr() & 15:
        return b, h, t
    if x.shape[3] > 1 and d != 1 or x.data_ptr() & 15:
        return None
    kept = tuple(s if n > 1 else 0 for n, s in zip(x.shape, (b, h, t)))  # (an axis of one has no stride)
    return None if (kept[0] | kept[1] | kept[2]) & al else kept


_NO_STRIDES = (0, 0, 0)
_APPEND = _cabi.PAGED_APPEND_ARGS.pack


def _place(values: torch.Tensor, new: torch.Tensor, what: str) -> tuple[int, tuple]:
    """Address and strides of the tensor that the values of ``new`` go to."""
    if values.shape != new.shape or values.dtype != new.dtype or values.get_device() != new.get_device():
        raise ValueError(f"{what} must be a {new.dtype} tensor of shape {tuple(new.shape)} on {new.device}")
    strides = _row_strides(values)
    if strides is None:
        raise ValueError(f"{what} must have contiguous rows that start on 16-byte boundaries: it is written in place")
    if 0 in strides and any(s == 0 and n > 1 for s, n in zip(strides, values.shape)):
        raise ValueError(f"{what} must have a row for every token: it is written in place")
    return values.data_ptr(), strides


def append_kv_paged(kq, vq, k_new: torch.Tensor, v_new: torch.Tensor, block_table: torch.Tensor, positions,
                    lengths: torch.Tensor | None = None, k_values: torch.Tensor | None = None,
                    v_values: torch.Tensor | None = None):
    """Write new K and V tokens into the pages of a paged cache, one launch, no allocation.

    ``k_new``, ``v_new`` ``(B, HKV, T, head_dim)`` float16, bfloat16 or float32, of any strides
    that keep a row contiguous (the view ``x.transpose(1, 2)`` of a ``(B, T, HKV, head_dim)``
    projection is read in place).  Token ``t`` of sequence ``b`` goes to position
    ``positions[b] + t`` (``positions``: an int, or int32 ``(B,)`` on the device).  ``lengths``
    (int32 ``(B,)``): only the first ``lengths[b]`` of the T tokens are there, as in a padded
    batch of prompts.  Positions outside the table, and entries that name no page, drop their
    tokens; everything else in the pools stays as it was.

    Packed pools receive the bytes of ``quantize.quantize_groupwise`` on the same values.
    ``k_values`` / ``v_values`` (optional, shape and dtype of ``k_new``, rows contiguous): receive
    ``code * scale + zero`` of every written token -- what the cache now stands for, so that a
    prompt's own attention can see the same keys and values as the tokens that follow it.
    Two tokens that go to one place in the same call leave an undefined row there (in a packed pool even the
    codes of one beside the scale of the other), and undefined ``k_values`` / ``v_values`` where those overlap.
    Returns ``(kq, vq)``."""
    kt, vt = pool_tensors(kq, "kq"), pool_tensors(vq, "vq")
    packed = len(kt) == 3
    if len(vt) != len(kt) or kt[0].shape != vt[0].shape:
        raise ValueError("K and V pools must have the same format and shape")
    if packed and (kq.nbits != vq.nbits or kq.group_size != vq.group_size):
        raise ValueError("K and V must use the same nbits/group_size")
    NP, HKV, page, D = kt[0].shape
    if packed:
        D = kq.head_dim
    where = kt[0].get_device()
    shape, dtype = k_new.shape, k_new.dtype
    if len(shape) != 4 or shape != v_new.shape:
        raise ValueError(f"k_new and v_new must both be (B, HKV, T, head_dim), got {tuple(shape)} and {tuple(v_new.shape)}")
    B, H, T, Dn = shape
    if H != HKV or Dn != D:
        raise ValueError(f"k_new {tuple(shape)} does not match pools of {HKV} heads of {D}")
    if dtype != v_new.dtype:
        raise ValueError(f"k_new and v_new must have the same dtype, got {dtype} and {v_new.dtype}")
    if k_new.get_device() != where or v_new.get_device() != where or vt[0].get_device() != where:
        raise ValueError(f"the pools and the new tokens must be on one device, got {kt[0].device}, {vt[0].device}, "
                         f"{k_new.device}, {v_new.device}")
    W, stride = check_table(block_table, B, where)
    pos_ptr = pos0 = len_ptr = 0
    if isinstance(positions, torch.Tensor):
        positions = check_lens(positions, B, where, "positions")
        pos_ptr = positions.data_ptr()
    else:
        pos0 = int(positions)
        if pos0 < 0 or pos0 + T > min(W * page, 2 ** 30):  # the longest row of tokens a table may name
            raise ValueError(f"tokens [{pos0}, {pos0 + T}) do not fit a table of {W} pages of {page}")
    if lengths is not None:
        lengths = check_lens(lengths, B, where, "lengths")
        len_ptr = lengths.data_ptr()
    k_place, k_vs = (0, _NO_STRIDES) if k_values is None else _place(k_values, k_new, "k_values")
    v_place, v_vs = (0, _NO_STRIDES) if v_values is None else _place(v_values, v_new, "v_values")
    code = _cabi.dtype_code(k_new)
    _cabi.require_cuda(kt[0], "kq")
    lib = _cabi.load()
    if B == 0 or T == 0 or W == 0:
        return kq, vq
    k_strides, v_strides = _row_strides(k_new), _row_strides(v_new)
    if k_strides is None:
        k_new = k_new.clone(memory_format=torch.contiguous_format)
        k_strides = _row_strides(k_new)
    if v_strides is None:
        v_new = v_new.clone(memory_format=torch.contiguous_format)
        v_strides = _row_strides(v_new)
    kp, ks, kz = (t.data_ptr() for t in kt) if packed else (kt[0].data_ptr(), 0, 0)
    vp, vs, vz = (t.data_ptr() for t in vt) if packed else (vt[0].data_ptr(), 0, 0)
    dev = k_new.device
    with _cabi.on_device(dev):
        _cabi.check(lib.tkv_paged_append(
            _APPEND(k_new.data_ptr(), v_new.data_ptr(), kp, ks, kz, vp, vs, vz, k_place, v_place, block_table.data_ptr(),
                    pos_ptr, len_ptr, *k_strides, *v_strides, *k_vs, *v_vs, stride, code, pos0, B, HKV, T, NP, page, W, D,
                    kq.nbits if packed else 16, kq.group_size if packed else 0), _cabi.stream_ptr(dev)))
    return kq, vq


def _pool_list(pools) -> tuple[list[torch.Tensor], int, int, int]:
    """(tensors, num_pages, page_size, device index) of pools that share one block table."""
    if isinstance(pools, (QuantizedTensor, torch.Tensor)):
        pools = [pools]
    ts, shape, where = [], None, -1
    for i, p in enumerate(pools):
        t = pool_tensors(p, f"pools[{i}]")
        if shape is None:
            shape, where = t[0].shape, t[0].get_device()
        else:
            other = t[0].shape
            if other[0] != shape[0] or other[2] != shape[2] or t[0].get_device() != where:
                raise ValueError("pools that share a block table must have the same number and size of pages and one "
                                 "device")
        ts += t
    if not ts:
        raise ValueError("pools must name at least one pool")
    if ts[0].numel() == 0:
        raise ValueError("pools must have at least one page of at least one token")
    return ts, shape[0], shape[2], where


_FORK = _cabi.PAGES_FORK_ARGS.pack
_COMPACT = _cabi.PAGES_COMPACT_ARGS.pack
_pages_words: dict = {}


def _pages_workspace(ws: dict | None, B: int, NP: int, dev) -> torch.Tensor:
    """The plan's scratch, zero at first and kept in the caller's dict ``ws``, one for every number of pages on
    every device (its layout goes by the first, and its zero words are left zero for the next call).  What is made
    during a capture is the graph's own: it is cleared when the graph runs, so it is not kept for other calls."""
    need = _pages_words.get((B, NP))
    if need is None:
        n = ctypes.c_int64(0)
        _cabi.check(_cabi.load().tkv_pages_workspace(B, NP, ctypes.byref(n)))
        need = n.value
        if len(_pages_words) < 4096:
            _pages_words[(B, NP)] = need
    scratch = None if ws is None else ws.setdefault("pages", {})
    kept = None if scratch is None else scratch.get((NP, dev))
    if kept is None or kept.numel() < need:
        if scratch is None or _cabi.capturing():
            return torch.zeros(need, dtype=torch.int32, device=dev)
        if kept is not None:  # a captured graph may still use it
            ws.setdefault("outgrown", []).append(kept)
        # (2 words a row: room for twice the rows, so that rows added one by one leave few of them behind)
        kept = scratch[NP, dev] = torch.zeros(need + 2 * B, dtype=torch.int32, device=dev)
    return kept


def _pool_args(ts, NP: int):
    """(address, bytes per page) of every tensor as the C array, and how many."""
    words = []
    for t in ts:
        words += (t.data_ptr(), t.nbytes // NP)
    return struct.pack(f"{len(words)}q", *words), len(ts)


def _new_like(x, shape, like, what):
    if x is None:  # (empty_like is the cheaper call)
        return torch.empty_like(like) if like.shape == shape and like.is_contiguous() else like.new_empty(shape)
    if x.shape != shape or x.dtype is not _I32 or x.device != like.device or not x.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 tensor of shape {tuple(shape)} on {like.device}")
    return x


def _span(t: torch.Tensor) -> tuple[int, int]:
    """First and last + 1 byte of an int32 tensor; empty ones overlap nothing."""
    a, n = t.data_ptr(), t.numel()
    if n == 0:
        return 0, 0
    if not t.is_contiguous():
        n = 1 + sum((k - 1) * s for k, s in zip(t.shape, t.stride()))
    return a, a + 4 * n


def _no_overlap(outs, ins) -> None:
    ins = [_span(t) for t in ins]
    for i, t in enumerate(outs):
        a0, a1 = _span(t)
        for b0, b1 in ins:
            if a0 < b1 and b0 < a1:
                raise ValueError(f"out[{i}] must not share memory with a tensor it is made from or another out")
        ins.append((a0, a1))


def fork_pages(pools, block_table: torch.Tensor, seq_lens: torch.Tensor, parents: torch.Tensor, reserve=0,
               out: tuple | None = None, _workspace: dict | None = None):
    """The next round of sequences from the present ones: fork, keep, drop, and make room.

    Row ``b`` of the new table continues row ``parents[b]`` (int32 ``(B_new,)``) of
    ``block_table (B, max_pages)`` at its length ``seq_lens[parents[b]]``: full pages are shared,
    a partly filled page is kept by the first row that continues this parent and copied for every
    other one, in all ``pools`` (a pool or a list of pools -- K and V of every layer that uses
    this table).  A parent outside the old table gives an empty row; a row that nothing
    continues gives its pages back.  Then pages are added for ``reserve`` further tokens (an int,
    or int32 ``(B_new,)``).  So ``parents = arange(B)`` makes room, ``-1`` frees, and a beam search
    passes the winners.

    Fresh pages are the lowest ones that no kept entry names, in order of rows and positions.
    Entries behind a row's last page are -1.  Returns ``(table, lens, missing)``: int32
    ``(B_new, max_pages)``, ``(B_new,)``, and ``(1,)``, the number of pages that the pool was short of
    (their entries are -1, and what is appended there is dropped).  ``out``: these three
    tensors, supplied by the caller; they must not share memory with the inputs or each other.  The old
    table is not changed.  A partly filled page that two different rows name (which this
    function never makes) stays shared."""
    ts, NP, page, where = _pool_list(pools)
    W, stride = check_table(block_table, None, where)
    B_old = block_table.shape[0]
    seq_lens = check_lens(seq_lens, B_old, where, "seq_lens")
    if parents.dim() != 1:
        raise ValueError(f"parents must be an int32 tensor (B_new,) on {_on(where)}")
    B = parents.shape[0]
    parents = check_lens(parents, B, where, "parents")
    r_ptr = r0 = 0
    if isinstance(reserve, torch.Tensor):
        reserve = check_lens(reserve, B, where, "reserve")
        r_ptr = reserve.data_ptr()
    else:
        r0 = int(reserve)
        if not 0 <= r0 < 2 ** 31:
            raise ValueError(f"reserve must be a number of tokens, got {r0}")
    table, lens, missing = (None, None, None) if out is None else out
    table = _new_like(table, (B, W), block_table, "out[0]")
    lens = _new_like(lens, (B,), parents, "out[1]")
    missing = _new_like(missing, (1,), block_table, "out[2]")
    if out is not None:
        _no_overlap((table, lens, missing), (block_table, seq_lens, parents) + ((reserve,) if r_ptr else ()))
    _cabi.require_cuda(ts[0], "pools")
    lib, dev = _cabi.load(), block_table.device
    with _cabi.on_device(dev):
        ws = _pages_workspace(_workspace, B, NP, dev)
        _cabi.check(lib.tkv_pages_fork(
            _FORK(block_table.data_ptr(), seq_lens.data_ptr(), parents.data_ptr(), r_ptr, table.data_ptr(), lens.data_ptr(),
                  missing.data_ptr(), ws.data_ptr(), stride, B_old, r0, B, W, NP, page),
            *_pool_args(ts, NP), _cabi.stream_ptr(dev)))
    return table, lens, missing


def compact_pages(pools, block_table: torch.Tensor, out: tuple | None = None, _workspace: dict | None = None):
    """Move the pages that ``block_table (B, max_pages)`` names to the front of the ``pools``.

    With n different pages in use, the k-th used page at or above n moves to the k-th unused one
    below n (in order of page numbers), in all ``pools`` that share the table.  Returns
    ``(table, live)``: the table with the new numbers, and int32 ``(1,)`` holding n -- pages from n
    on are then unused.  The old table stays valid as long as the freed places are not written:
    pages are copied, and only into places that it did not name.  ``out``: these two tensors,
    supplied by the caller."""
    ts, NP, page, where = _pool_list(pools)
    W, stride = check_table(block_table, None, where)
    B = block_table.shape[0]
    table, live = (None, None) if out is None else out
    table = _new_like(table, (B, W), block_table, "out[0]")
    live = _new_like(live, (1,), block_table, "out[1]")
    if out is not None:
        _no_overlap((table, live), (block_table,))
    _cabi.require_cuda(ts[0], "pools")
    lib, dev = _cabi.load(), block_table.device
    with _cabi.on_device(dev):
        ws = _pages_workspace(_workspace, B, NP, dev)
        _cabi.check(lib.tkv_pages_compact(
            _COMPACT(block_table.data_ptr(), table.data_ptr(), live.data_ptr(), ws.data_ptr(), stride, B, W, NP),
            *_pool_args(ts, NP), _cabi.stream_ptr(dev)))
    return table, live
