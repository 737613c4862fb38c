"""Decode attention over a paged KV cache: packed 2/4-bit pages and float16 pages.

The paged counterparts of ``fused_decode_attention`` and ``fp16_decode_attention`` (see
:mod:`tritonkv_b200.paged` for the pools and the block table).  No reference counterpart: its
caches are one contiguous tensor per batch.
"""

from __future__ import annotations

import torch

from .. import _cabi
from ..paged import check_lens, check_table, pool_tensors
from ..quantize import QuantizedTensor
from ._launch import q_for_kernel

__all__ = ["paged_decode_attention", "paged_fp16_decode_attention"]


_CODE = {torch.float16: _cabi.DTYPE_F16, torch.bfloat16: _cabi.DTYPE_BF16, torch.float32: _cabi.DTYPE_F32}
_PACK = _cabi.PAGED_DECODE_ARGS.pack


def _attend(q, k, v, nbits, group_size, block_table, seq_lens, sm_scale, out, workspace):
    kt, vt = pool_tensors(k, "k"), pool_tensors(v, "v")
    shape = kt[0].shape
    if len(kt) != len(vt) or vt[0].shape != shape:
        raise ValueError("K and V pools must have the same shape")
    if q.dim() != 3:
        raise ValueError(f"q must be (B, HQ, head_dim), got {tuple(q.shape)}")
    B, HQ, D = q.shape
    NP, HKV, page, row = shape
    if D != (row if nbits == 16 else k.head_dim):
        raise ValueError(f"q {tuple(q.shape)} is incompatible with pools of {tuple(shape)}")
    if HKV == 0 or HQ == 0 or HQ % HKV != 0:
        raise ValueError(f"HQ={HQ} must be a multiple of HKV={HKV}")
    where = q.get_device()
    if kt[0].get_device() != where or vt[0].get_device() != where:
        raise ValueError(f"the pools are on {kt[0].device} and {vt[0].device}, q on {q.device}")
    W, stride = check_table(block_table, B, where)
    seq_lens = check_lens(seq_lens, B, where, "seq_lens")
    if out is None:
        out = torch.empty((B, HQ, D), device=q.device, dtype=torch.float32)
    elif out.shape != q.shape or out.dtype not in _CODE or out.get_device() != where or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous float32, float16 or bfloat16 tensor of shape {(B, HQ, D)} on {q.device}")
    _cabi.require_cuda(q, "q")
    lib = _cabi.load()
    if B == 0:
        return out
    q = q_for_kernel(q)
    if nbits == 16:
        k, v, ks, kz, vs, vz = kt[0].data_ptr(), vt[0].data_ptr(), 0, 0, 0, 0
    else:
        k, ks, kz = [t.data_ptr() for t in kt]
        v, vs, vz = [t.data_ptr() for t in vt]
    with _cabi.on_device(q.device):
        ws = _cabi.paged_workspace(workspace, (B, HQ, HKV, page, D, nbits, group_size, where), q.device)
        _cabi.check(lib.tkv_paged_decode(
            _PACK(q.data_ptr(), k, ks, kz, v, vs, vz, block_table.data_ptr(), seq_lens.data_ptr(), out.data_ptr(), ws[1],
                  ws[3], stride, ws[2], _CODE[q.dtype], _CODE[out.dtype], B, HQ, HKV, NP, page, W, D, nbits, group_size,
                  D ** -0.5 if sm_scale is None else sm_scale), _cabi.stream_ptr(q.device)))
    return out


def paged_decode_attention(
    q: torch.Tensor,
    kq: QuantizedTensor,
    vq: QuantizedTensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    sm_scale: float | None = None,
    out: torch.Tensor | None = None,
    _workspace: dict | None = None,
) -> torch.Tensor:
    """Single decode step of attention over packed pages.

    q ``(B, HQ, D)`` (rounded to float16 in the kernel); ``kq``, ``vq`` packed pools of
    ``(num_pages, HKV, page_size, ...)``, page_size a multiple of 16; ``block_table`` int32
    ``(B, max_pages)`` with contiguous rows; ``seq_lens`` int32 ``(B,)``.  Sequence ``b`` attends its
    first ``seq_lens[b]`` tokens (clamped to the table's), without those whose table entry names no
    page; with none left its output is zero.  Returns ``(B, HQ, D)`` float32, or ``out``, which may
    also be float16 or bfloat16 (rounded once, at the end).  With ``out`` and ``_workspace`` (a dict
    that the caller keeps, as long as a graph that was captured with it; one for each stream or
    graph that may run at the same time)
    supplied, the call allocates nothing after its first use and can be captured."""
    if not isinstance(kq, QuantizedTensor) or not isinstance(vq, QuantizedTensor):
        raise TypeError("paged_decode_attention reads packed pools (QuantizedTensor); see paged_fp16_decode_attention")
    if kq.nbits != vq.nbits or kq.group_size != vq.group_size:
        raise ValueError("K and V must use the same nbits/group_size")
    return _attend(q, kq, vq, kq.nbits, kq.group_size, block_table, seq_lens, sm_scale, out, _workspace)


def paged_fp16_decode_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    sm_scale: float | None = None,
    out: torch.Tensor | None = None,
    _workspace: dict | None = None,
) -> torch.Tensor:
    """Single decode step of attention over float16 pages ``k``, ``v``
    ``(num_pages, HKV, page_size, D)``; everything else as in :func:`paged_decode_attention`."""
    if not isinstance(k, torch.Tensor) or not isinstance(v, torch.Tensor):
        raise TypeError("paged_fp16_decode_attention reads float16 pools; see paged_decode_attention")
    return _attend(q, k, v, 16, 0, block_table, seq_lens, sm_scale, out, _workspace)
