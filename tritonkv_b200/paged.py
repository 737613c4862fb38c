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

import torch

from . import _cabi
from .quantize import QuantizedTensor, check_cache_tensors

Pool = "QuantizedTensor | torch.Tensor"


def pool_tensors(pool, what: str) -> tuple[torch.Tensor, ...]:
    """The contiguous 4-D tensors of a pool; the kernels use them in place."""
    if isinstance(pool, QuantizedTensor):
        t = (pool.packed, pool.scale, pool.zero)
        check_cache_tensors(pool, what, pool.packed.device)
        if pool.packed.dim() != 4 or t[1].shape[:3] != t[0].shape[:3] or t[2].shape != t[1].shape:
            raise ValueError(f"{what}: a packed pool has packed (num_pages, HKV, page_size, bytes) and scale, zero "
                             f"(num_pages, HKV, page_size, groups); got {[tuple(x.shape) for x in t]}")
        if t[0].shape[3] * 8 != pool.head_dim * pool.nbits or t[1].shape[3] * pool.group_size != pool.head_dim:
            raise ValueError(f"{what}: rows of {t[0].shape[3]} bytes and {t[1].shape[3]} groups are not those of "
                             f"head_dim {pool.head_dim} at {pool.nbits} bits in groups of {pool.group_size}")
    elif isinstance(pool, torch.Tensor):
        t = (pool,)
        if pool.dtype != torch.float16:
            raise TypeError(f"{what} must be a QuantizedTensor or a float16 tensor, got {pool.dtype}")
        if pool.dim() != 4:
            raise ValueError(f"{what}: a float16 pool is (num_pages, HKV, page_size, head_dim), got {tuple(pool.shape)}")
    else:
        raise TypeError(f"{what} must be a QuantizedTensor or a float16 tensor, got {type(pool).__name__}")
    for x in t:
        if not x.is_contiguous():
            raise ValueError(f"{what} must be contiguous: a pool is used in place")
    return t


def check_table(block_table: torch.Tensor, B: int | None, device) -> tuple[int, int]:
    """(entries per row, row stride) of an int32 table (B, max_pages) whose rows are contiguous."""
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.device != device:
        raise ValueError(f"block_table must be an int32 tensor (B, max_pages) on {device}")
    if B is not None and block_table.shape[0] != B:
        raise ValueError(f"block_table has {block_table.shape[0]} rows for {B} sequences")
    n = block_table.shape[1]
    if n > 1 and block_table.stride(1) != 1:
        raise ValueError("block_table rows must be contiguous")
    return n, block_table.stride(0)


def check_lens(lens: torch.Tensor, B: int, device, what: str) -> torch.Tensor:
    if lens.shape != (B,) or lens.dtype != torch.int32 or lens.device != device:
        raise ValueError(f"{what} must be an int32 tensor of shape ({B},) on {device}")
    return lens.contiguous()


def _rows16(x: torch.Tensor) -> torch.Tensor:
    """x itself where its rows are contiguous and start on 16-byte boundaries, else a copy."""
    al = 16 // x.element_size()
    ok = x.stride(3) == 1 and x.data_ptr() % 16 == 0
    for size, stride in zip(x.shape[:3], x.stride()[:3]):
        ok = ok and (size == 1 or stride % al == 0)
    return x if ok else x.clone(memory_format=torch.contiguous_format)


def _strides(x: torch.Tensor) -> list[int]:
    return [s if n > 1 else 0 for n, s in zip(x.shape[:3], x.stride()[:3])]


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
    Two tokens that go to one place in the same call leave either of them there.
    Returns ``(kq, vq)``."""
    kt, vt = pool_tensors(kq, "kq"), pool_tensors(vq, "vq")
    packed = isinstance(kq, QuantizedTensor)
    if len(kt) != len(vt) or any(a.shape != b.shape for a, b in zip(kt, vt)):
        raise ValueError("K and V pools must have the same format and shape")
    if packed and (kq.nbits, kq.group_size) != (vq.nbits, vq.group_size):
        raise ValueError("K and V must use the same nbits/group_size")
    NP, HKV, page, _ = kt[0].shape
    D = kq.head_dim if packed else kt[0].shape[3]
    dev = kt[0].device
    if k_new.dim() != 4 or k_new.shape != v_new.shape:
        raise ValueError(f"k_new and v_new must both be (B, HKV, T, head_dim), got {tuple(k_new.shape)} and {tuple(v_new.shape)}")
    B, H, T, Dn = k_new.shape
    if (H, Dn) != (HKV, D):
        raise ValueError(f"k_new {tuple(k_new.shape)} does not match pools of {HKV} heads of {D}")
    if k_new.dtype != v_new.dtype:
        raise ValueError(f"k_new and v_new must have the same dtype, got {k_new.dtype} and {v_new.dtype}")
    if k_new.device != dev or v_new.device != dev or vt[0].device != dev:
        raise ValueError(f"the pools and the new tokens must be on one device, got {dev}, {vt[0].device}, {k_new.device}")
    W, stride = check_table(block_table, B, dev)
    pos_ptr, pos0 = None, 0
    if isinstance(positions, torch.Tensor):
        positions = check_lens(positions, B, dev, "positions")
        pos_ptr = positions.data_ptr()
    else:
        pos0 = int(positions)
        if pos0 < 0 or pos0 + T > W * page:
            raise ValueError(f"tokens [{pos0}, {pos0 + T}) do not fit a table of {W} pages of {page}")
    if lengths is not None:
        lengths = check_lens(lengths, B, dev, "lengths")
    vstrides = [0] * 6
    for i, (val, new, what) in enumerate(((k_values, k_new, "k_values"), (v_values, v_new, "v_values"))):
        if val is None:
            continue
        if val.shape != new.shape or val.dtype != new.dtype or val.device != dev:
            raise ValueError(f"{what} must be a {new.dtype} tensor of shape {tuple(new.shape)} on {dev}")
        if _rows16(val) is not val:
            raise ValueError(f"{what} must have contiguous rows that start on 16-byte boundaries: it is written in place")
        vstrides[3 * i:3 * i + 3] = _strides(val)
    code = _cabi.dtype_code(k_new)
    _cabi.require_cuda(kt[0], "kq")
    lib = _cabi.load()
    if B == 0 or T == 0 or W == 0:
        return kq, vq
    k_new, v_new = _rows16(k_new), _rows16(v_new)
    ks, kz, vs, vz = (kt[1], kt[2], vt[1], vt[2]) if packed else (None,) * 4
    i6 = ctypes.c_int64 * 6
    with _cabi.on_device(dev):
        _cabi.check(lib.tkv_paged_append(
            k_new.data_ptr(), v_new.data_ptr(), code, i6(*_strides(k_new), *_strides(v_new)), kt[0].data_ptr(),
            _cabi.ptr(ks), _cabi.ptr(kz), vt[0].data_ptr(), _cabi.ptr(vs), _cabi.ptr(vz), _cabi.ptr(k_values),
            _cabi.ptr(v_values), i6(*vstrides), block_table.data_ptr(), stride, pos_ptr, pos0, _cabi.ptr(lengths), B,
            HKV, T, NP, page, W, D, kq.nbits if packed else 16, kq.group_size if packed else 0,
            _cabi.stream_ptr(dev)))
    return kq, vq


def _pool_list(pools) -> tuple[list[torch.Tensor], int, int, torch.device]:
    """(tensors, num_pages, page_size, device) of pools that share one block table."""
    if isinstance(pools, (QuantizedTensor, torch.Tensor)):
        pools = [pools]
    ts = [t for i, p in enumerate(pools) for t in pool_tensors(p, f"pools[{i}]")]
    if not ts:
        raise ValueError("pools must name at least one pool")
    NP, _, page, _ = ts[0].shape
    for t in ts:
        if (t.shape[0], t.shape[2]) != (NP, page) or t.device != ts[0].device:
            raise ValueError("pools that share a block table must have the same number and size of pages and one device")
    if NP == 0 or page == 0:
        raise ValueError("pools must have at least one page of at least one token")
    return ts, NP, page, ts[0].device


_pages_words: dict = {}


def _pages_workspace(ws: dict | None, B: int, NP: int, dev) -> torch.Tensor:
    """The plan's scratch, zero at first and kept in the caller's dict ``ws`` for one number of pages."""
    need = _pages_words.get((B, NP))
    if need is None:
        n = ctypes.c_int64(0)
        _cabi.check(_cabi.load().tkv_pages_workspace(B, NP, ctypes.byref(n)))
        need = n.value
        if len(_pages_words) < 4096:
            _pages_words[(B, NP)] = need
    kept, t = (None, None) if ws is None else ws.get("pages", (None, None))
    if kept != NP or t.numel() < need or t.device != dev:
        t = torch.zeros(need, dtype=torch.int32, device=dev)
        if ws is not None:
            ws["pages"] = (NP, t)
    return t


def _pool_args(ts):
    ptrs = (ctypes.c_void_p * len(ts))(*(t.data_ptr() for t in ts))
    sizes = (ctypes.c_int64 * len(ts))(*(t.numel() // t.shape[0] * t.element_size() for t in ts))
    return ptrs, sizes, len(ts)


def _new_like(x, shape, dev, what):
    if x is None:
        return torch.empty(shape, dtype=torch.int32, device=dev)
    if x.shape != shape or x.dtype != torch.int32 or x.device != dev or not x.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 tensor of shape {tuple(shape)} on {dev}")
    return x


def _no_overlap(a: torch.Tensor, b: torch.Tensor, what: str) -> None:
    if a.numel() and b.numel():
        span = lambda t: (t.data_ptr(), t.data_ptr() + 4 * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))))
        (a0, a1), (b0, b1) = span(a), span(b)
        if a0 < b1 and b0 < a1:
            raise ValueError(f"{what} must not share memory with the tensor it is made from")


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
    tensors, supplied by the caller; they must not share memory with the inputs.  The old
    table is not changed.  A partly filled page that two different rows name (which this
    function never makes) stays shared."""
    ts, NP, page, dev = _pool_list(pools)
    W, stride = check_table(block_table, None, dev)
    B_old = block_table.shape[0]
    seq_lens = check_lens(seq_lens, B_old, dev, "seq_lens")
    if parents.dim() != 1:
        raise ValueError(f"parents must be an int32 tensor (B_new,) on {dev}")
    B = parents.shape[0]
    parents = check_lens(parents, B, dev, "parents")
    r_ptr, r0 = None, 0
    if isinstance(reserve, torch.Tensor):
        reserve = check_lens(reserve, B, dev, "reserve")
        r_ptr = reserve.data_ptr()
    else:
        r0 = int(reserve)
        if not 0 <= r0 < 2 ** 31:
            raise ValueError(f"reserve must be a number of tokens, got {r0}")
    table, lens, missing = (None, None, None) if out is None else out
    table = _new_like(table, (B, W), dev, "out[0]")
    lens = _new_like(lens, (B,), dev, "out[1]")
    missing = _new_like(missing, (1,), dev, "out[2]")
    if out is not None:
        for x in (block_table, seq_lens, parents) + ((reserve,) if r_ptr is not None else ()):
            for i, y in enumerate((table, lens, missing)):
                _no_overlap(y, x, f"out[{i}]")
    _cabi.require_cuda(ts[0], "pools")
    lib = _cabi.load()
    with _cabi.on_device(dev):
        ws = _pages_workspace(_workspace, B, NP, dev)
        _cabi.check(lib.tkv_pages_fork(
            block_table.data_ptr(), stride, seq_lens.data_ptr(), B_old, parents.data_ptr(), r_ptr, r0, B, W, NP, page,
            table.data_ptr(), lens.data_ptr(), missing.data_ptr(), ws.data_ptr(), *_pool_args(ts), _cabi.stream_ptr(dev)))
    return table, lens, missing


def compact_pages(pools, block_table: torch.Tensor, out: tuple | None = None, _workspace: dict | None = None):
    """Move the pages that ``block_table (B, max_pages)`` names to the front of the ``pools``.

    With n different pages in use, the k-th used page at or above n moves to the k-th unused one
    below n (in order of page numbers), in all ``pools`` that share the table.  Returns
    ``(table, live)``: the table with the new numbers, and int32 ``(1,)`` holding n -- pages from n
    on are then unused.  The old table stays valid as long as the freed places are not written:
    pages are copied, and only into places that it did not name.  ``out``: these two tensors,
    supplied by the caller."""
    ts, NP, page, dev = _pool_list(pools)
    W, stride = check_table(block_table, None, dev)
    B = block_table.shape[0]
    table, live = (None, None) if out is None else out
    table = _new_like(table, (B, W), dev, "out[0]")
    live = _new_like(live, (1,), dev, "out[1]")
    if out is not None:
        _no_overlap(table, block_table, "out[0]")
        _no_overlap(live, block_table, "out[1]")
    _cabi.require_cuda(ts[0], "pools")
    lib = _cabi.load()
    with _cabi.on_device(dev):
        ws = _pages_workspace(_workspace, B, NP, dev)
        _cabi.check(lib.tkv_pages_compact(
            block_table.data_ptr(), stride, B, W, NP, table.data_ptr(), live.data_ptr(), ws.data_ptr(), *_pool_args(ts),
            _cabi.stream_ptr(dev)))
    return table, live
