"""Decode attention over a paged KV cache: packed 2/4-bit pages and float16 pages.

The paged counterparts of ``fused_decode_attention`` and ``fp16_decode_attention`` (see
:mod:`tritonkv_b200.paged` for the pools and the block table).  No reference counterpart: its
caches are one contiguous tensor per batch.
"""

from __future__ import annotations

import math

import torch

from .. import _cabi
from ..paged import check_lens, check_table, pool_tensors
from ..quantize import QuantizedTensor
from ._launch import q_for_kernel

__all__ = ["paged_decode_attention", "paged_fp16_decode_attention"]


_OUT = {torch.float32, torch.float16, torch.bfloat16}


def _check(q, k, v, block_table, seq_lens, out):
    """Checked arguments shared by the two forms: (k tensors, v tensors, q, seq_lens, out, sizes)."""
    kt, vt = pool_tensors(k, "k"), pool_tensors(v, "v")
    shape = kt[0].shape
    if len(kt) != len(vt) or vt[0].shape != shape:
        raise ValueError("K and V pools must have the same shape")
    if q.dim() != 3:
        raise ValueError(f"q must be (B, HQ, head_dim), got {tuple(q.shape)}")
    B, HQ, D = q.shape
    NP, HKV, page, row = shape
    if D != (k.head_dim if len(kt) == 3 else row):
        raise ValueError(f"q {tuple(q.shape)} is incompatible with pools of {tuple(shape)}")
    if HKV == 0 or HQ == 0 or HQ % HKV != 0:
        raise ValueError(f"HQ={HQ} must be a multiple of HKV={HKV}")
    dev = q.device
    if kt[0].device != dev or vt[0].device != dev:
        raise ValueError(f"the pools are on {kt[0].device} and {vt[0].device}, q on {dev}")
    W, stride = check_table(block_table, B, dev)
    seq_lens = check_lens(seq_lens, B, dev, "seq_lens")
    if out is None:
        out = torch.empty((B, HQ, D), device=dev, dtype=torch.float32)
    elif out.shape != q.shape or out.dtype not in _OUT or out.device != dev or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous float32, float16 or bfloat16 tensor of shape {(B, HQ, D)} on {dev}")
    return kt, vt, q_for_kernel(q), seq_lens, out, (B, HQ, HKV, NP, page, W, D), stride


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
    kt, vt, q, seq_lens, out, (B, HQ, HKV, NP, page, W, D), stride = _check(q, kq, vq, block_table, seq_lens, out)
    _cabi.require_cuda(q, "q")
    lib = _cabi.load()
    if B == 0:
        return out
    dev = q.device
    with _cabi.on_device(dev):
        ws = _cabi.paged_workspace(_workspace, B, HQ, HKV, page, D, kq.nbits, kq.group_size, dev)
        _cabi.check(lib.tkv_paged_decode(
            q.data_ptr(), _cabi.dtype_code(q), kt[0].data_ptr(), kt[1].data_ptr(), kt[2].data_ptr(), vt[0].data_ptr(),
            vt[1].data_ptr(), vt[2].data_ptr(), block_table.data_ptr(), stride, seq_lens.data_ptr(), out.data_ptr(),
            _cabi.dtype_code(out), ws[0].data_ptr(), ws[1], ws[2], B, HQ, HKV, NP, page, W, D, kq.nbits, kq.group_size,
            1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale), _cabi.stream_ptr(dev)))
    return out


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
    kt, vt, q, seq_lens, out, (B, HQ, HKV, NP, page, W, D), stride = _check(q, k, v, block_table, seq_lens, out)
    _cabi.require_cuda(q, "q")
    lib = _cabi.load()
    if B == 0:
        return out
    dev = q.device
    with _cabi.on_device(dev):
        ws = _cabi.paged_workspace(_workspace, B, HQ, HKV, page, D, 16, 0, dev)
        _cabi.check(lib.tkv_paged_fp16_decode(
            q.data_ptr(), _cabi.dtype_code(q), kt[0].data_ptr(), vt[0].data_ptr(), block_table.data_ptr(), stride,
            seq_lens.data_ptr(), out.data_ptr(), _cabi.dtype_code(out), ws[0].data_ptr(), ws[1], ws[2], B, HQ, HKV, NP, page, W, D,
            1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale), _cabi.stream_ptr(dev)))
    return out
