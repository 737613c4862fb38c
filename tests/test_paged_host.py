"""What the paged-cache functions refuse, checked without a GPU."""

import os
import struct

import pytest
import torch

from tritonkv_b200 import _cabi
from tritonkv_b200.kernels import paged_decode_attention, paged_fp16_decode_attention
from tritonkv_b200.paged import append_kv_paged, compact_pages, fork_pages
from tritonkv_b200.quantize import QuantizedTensor, empty_cache


def pool(NP=6, HKV=2, page=16, D=64, nbits=4, gs=32):
    return empty_cache(NP, HKV, page, D, nbits, gs, "cpu")


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def args(**kw):
    d = dict(q=torch.zeros(3, 4, 64).half(), kq=pool(), vq=pool(), block_table=i32(3, 5), seq_lens=i32(3))
    d.update(kw)
    return d


@pytest.mark.parametrize("bad,err,text", [
    (dict(), RuntimeError, "CUDA"),
    (dict(vq=pool(gs=16)), ValueError, "same nbits/group_size"),
    (dict(vq=pool(NP=7)), ValueError, "same shape"),
    (dict(q=torch.zeros(3, 4, 128).half()), ValueError, "incompatible"),
    (dict(q=torch.zeros(3, 5, 64).half()), ValueError, "multiple of HKV"),
    (dict(q=torch.zeros(3, 0, 64).half()), ValueError, "multiple of HKV"),
    (dict(q=torch.zeros(3, 4).half()), ValueError, "q must be"),
    (dict(block_table=i32(2, 5)), ValueError, "rows for 3"),
    (dict(block_table=i32(3, 5).long()), ValueError, "int32"),
    (dict(block_table=i32(15)), ValueError, "int32"),
    (dict(block_table=i32(5, 3).T), ValueError, "contiguous"),
    (dict(seq_lens=i32(4)), ValueError, "seq_lens"),
    (dict(seq_lens=i32(3).long()), ValueError, "seq_lens"),
    (dict(out=torch.zeros(3, 4, 32)), ValueError, "out must"),
    (dict(out=torch.zeros(3, 4, 64).double()), ValueError, "out must"),
    (dict(out=torch.zeros(3, 64, 4).transpose(1, 2)), ValueError, "out must"),
    (dict(kq=torch.zeros(6, 2, 16, 64).half()), TypeError, "packed pools"),
])
def test_attention_refuses(bad, err, text):
    with pytest.raises(err, match=text):
        paged_decode_attention(**args(**bad))


@pytest.mark.parametrize("k,err,text", [
    (torch.zeros(6, 2, 16, 64).half(), RuntimeError, "CUDA"),
    (torch.zeros(6, 2, 16, 64), TypeError, "float16"),
    (torch.zeros(6, 2, 64).half(), ValueError, "num_pages"),
    (torch.zeros(6, 16, 2, 64).half().transpose(1, 2), ValueError, "contiguous"),
    (pool(), TypeError, "float16 pools"),
])
def test_fp16_attention_refuses(k, err, text):
    with pytest.raises(err, match=text):
        paged_fp16_decode_attention(torch.zeros(3, 4, 64).half(), k, k, i32(3, 5), i32(3))


def test_pools_that_do_not_fit_together():
    p = pool()
    for broken, err in ((QuantizedTensor(p.packed, p.scale.float(), p.zero, 4, 32, 64), TypeError),
                        (QuantizedTensor(p.packed.to(torch.int8), p.scale, p.zero, 4, 32, 64), TypeError),
                        (QuantizedTensor(p.packed, p.scale[:3], p.zero, 4, 32, 64), ValueError),
                        (QuantizedTensor(p.packed, p.scale, p.zero, 2, 32, 64), ValueError),
                        (QuantizedTensor(p.packed, p.scale, p.zero, 4, 16, 64), ValueError),
                        (QuantizedTensor(p.packed[:, :, ::2], p.scale[:, :, ::2], p.zero[:, :, ::2], 4, 32, 64), ValueError),
                        (QuantizedTensor(p.packed[0], p.scale[0], p.zero[0], 4, 32, 64), ValueError)):
        with pytest.raises(err):
            paged_decode_attention(**args(kq=broken, vq=broken))
        with pytest.raises(err):
            compact_pages([broken], i32(3, 5))
        with pytest.raises(err):
            append_kv_paged(broken, broken, torch.zeros(3, 2, 1, 64).half(), torch.zeros(3, 2, 1, 64).half(), i32(3, 5), 0)


@pytest.mark.parametrize("bad,err,text", [
    (dict(), RuntimeError, "CUDA"),
    (dict(v_new=torch.zeros(3, 2, 2, 64).half()), ValueError, "must both"),
    (dict(v_new=torch.zeros(3, 2, 1, 64)), ValueError, "same dtype"),
    (dict(k_new=torch.zeros(3, 1, 1, 64).half(), v_new=torch.zeros(3, 1, 1, 64).half()), ValueError, "does not match"),
    (dict(k_new=torch.zeros(3, 2, 1, 64).double(), v_new=torch.zeros(3, 2, 1, 64).double()), TypeError, "unsupported dtype"),
    (dict(vq=pool(nbits=2, gs=32)), ValueError, "same format"),
    (dict(positions=-1), ValueError, "do not fit"),
    (dict(positions=80), ValueError, "do not fit"),
    (dict(positions=i32(2)), ValueError, "positions"),
    (dict(lengths=i32(3).long()), ValueError, "lengths"),
    (dict(block_table=i32(4, 5)), ValueError, "rows for 3"),
    (dict(k_values=torch.zeros(3, 2, 1, 64)), ValueError, "k_values"),
    (dict(v_values=torch.zeros(3, 2, 1, 128).half()[..., ::2]), ValueError, "v_values"),
])
def test_append_refuses(bad, err, text):
    d = dict(kq=pool(), vq=pool(), k_new=torch.zeros(3, 2, 1, 64).half(), v_new=torch.zeros(3, 2, 1, 64).half(),
             block_table=i32(3, 5), positions=0)
    d.update(bad)
    with pytest.raises(err, match=text):
        append_kv_paged(**d)


@pytest.mark.parametrize("bad,err,text", [
    (dict(), RuntimeError, "CUDA"),
    (dict(pools=[]), ValueError, "at least one pool"),
    (dict(pools=[pool(), pool(NP=7)]), ValueError, "same number"),
    (dict(pools=[pool(), pool(page=32)]), ValueError, "same number"),
    (dict(pools=[3]), TypeError, "QuantizedTensor"),
    (dict(seq_lens=i32(2)), ValueError, "seq_lens"),
    (dict(parents=i32(2, 2)), ValueError, "parents"),
    (dict(parents=i32(2).long()), ValueError, "parents"),
    (dict(reserve=-1), ValueError, "reserve"),
    (dict(reserve=2 ** 31), ValueError, "reserve"),
    (dict(reserve=i32(3)), ValueError, "reserve"),
    (dict(out=(i32(2, 4), i32(2), i32(1))), ValueError, r"out\[0\]"),
    (dict(out=(i32(2, 5), i32(2), i32(2))), ValueError, r"out\[2\]"),
])
def test_fork_refuses(bad, err, text):
    d = dict(pools=[pool()], block_table=i32(3, 5), seq_lens=i32(3), parents=i32(2))
    d.update(bad)
    with pytest.raises(err, match=text):
        fork_pages(**d)


def test_compact_refuses():
    with pytest.raises(RuntimeError, match="CUDA"):
        compact_pages(pool(), i32(3, 5))
    with pytest.raises(ValueError, match="int32"):
        compact_pages(pool(), i32(3, 5).float())
    t = i32(3, 5)
    with pytest.raises(ValueError, match="share memory"):
        compact_pages(pool(), t, out=(t, i32(1)))


def test_paged_graphed_step_refuses():
    from tritonkv_b200 import GraphedDecodeStep

    for kw in (dict(), dict(seq_lens=i32(3), zero_copy=True), dict(seq_lens=i32(3), num_splits=2)):
        with pytest.raises(ValueError, match="paged step"):
            GraphedDecodeStep(pool(), pool(), 4, block_table=i32(3, 5), **kw)
    with pytest.raises(RuntimeError, match="CUDA"):
        GraphedDecodeStep(pool(), pool(), 4, block_table=i32(3, 5), seq_lens=i32(3))


def test_c_entries_refuse():
    """Argument errors of the C ABI come back before any launch."""
    lib, P = _cabi.load(), 4096  # a pointer that nothing follows: every call fails before that

    def decode(q=P, out=P, B=1, HQ=4, HKV=2, NP=8, page=16, W=4, D=64, nbits=4, gs=32, dt=0, scale=P, v=P):
        return lib.tkv_paged_decode(_cabi.PAGED_DECODE_ARGS.pack(q, P, scale, P, v, P, P, P, P, out, P, 0, W, 1 << 30, dt, 0, B,
                                                                 HQ, HKV, NP, page, W, D, nbits, gs, 1.0), None)

    I, U, A = _cabi.TKV_ERR_INVALID, _cabi.TKV_ERR_UNSUPPORTED, _cabi.TKV_ERR_ALIGN
    for rc, kw in ((I, dict(q=0)), (I, dict(B=0)), (I, dict(HQ=5)), (I, dict(NP=0)), (I, dict(nbits=3)), (I, dict(dt=7)),
                   (I, dict(NP=1 << 27)), (I, dict(W=1 << 27)), (U, dict(page=24)), (U, dict(D=96)), (U, dict(gs=8)),
                   (U, dict(gs=128)), (A, dict(q=P + 8)), (A, dict(scale=P + 2)), (A, dict(out=P + 4)), (I, dict(scale=0)),
                   (I, dict(nbits=16, v=0)), (A, dict(nbits=16, v=P + 2)), (U, dict(nbits=16, D=32))):
        assert decode(**kw) == rc, (kw, _cabi.last_error())
    assert lib.tkv_paged_decode(None, None) == I

    def append(k=P, st=64, B=1, T=1, D=64, nbits=4, gs=32, dt=0, val=0, vst=64, scale=P):
        return lib.tkv_paged_append(_cabi.PAGED_APPEND_ARGS.pack(k, P, P, scale, P, P, P, P, val, 0, P, 0, 0, *[st] * 6,
                                                                 *[vst] * 6, 4, dt, 0, B, 2, T, 8, 16, 4, D, nbits, gs), None)

    for rc, kw in ((I, dict(k=0)), (I, dict(nbits=3)), (I, dict(B=-1)), (I, dict(dt=5)), (I, dict(scale=0)),
                   (U, dict(D=48)), (U, dict(gs=4)), (U, dict(gs=128)), (U, dict(D=16, gs=16, nbits=2)), (A, dict(st=63)),
                   (A, dict(val=P, vst=63)), (A, dict(k=P + 2)), (I, dict(T=1 << 30, B=4))):
        assert append(**kw) == rc, (kw, _cabi.last_error())
    assert append(B=0) == 0 and append(T=0) == 0 and lib.tkv_paged_append(None, None) == I
    one = struct.pack("2q", P, 64)

    def fork(B=2, Bo=2, W=4, NP=8, page=16, par=P, ws=P, pools=one, n=1):
        return lib.tkv_pages_fork(_cabi.PAGES_FORK_ARGS.pack(P, P, par, 0, P, P, P, ws, W, Bo, 0, B, W, NP, page), pools, n, None)

    for kw in (dict(par=0), dict(ws=0), dict(NP=0), dict(page=0), dict(B=-1), dict(W=1 << 29), dict(pools=None), dict(n=-1),
               dict(pools=struct.pack("2q", 0, 64)), dict(pools=struct.pack("2q", P, 0))):
        assert fork(**kw) == I, (kw, _cabi.last_error())
    assert lib.tkv_pages_fork(None, one, 1, None) == I

    def compact(B=2, W=4, NP=8, live=P, n=1):
        return lib.tkv_pages_compact(_cabi.PAGES_COMPACT_ARGS.pack(P, P, live, P, W, B, W, NP), one, n, None)

    for kw in (dict(B=-1), dict(NP=0), dict(live=0), dict(W=1 << 29), dict(n=-1)):
        assert compact(**kw) == I, (kw, _cabi.last_error())
    assert lib.tkv_pages_compact(None, one, 1, None) == I


def test_argument_structs_match_the_header(tmp_path):
    """The packed layouts of the binding against the compiler's, field by field."""
    import shutil
    import subprocess

    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler")
    fields = {"tkv_paged_decode_args": ("workspace", "tickets", "table_stride", "workspace_bytes", "q_dtype", "gs", "sm_scale"),
              "tkv_paged_append_args": ("k", "lengths", "strides", "value_strides", "table_stride", "in_dtype", "gs"),
              "tkv_pages_fork_args": ("reserve", "workspace", "table_stride", "B_old", "page_size"),
              "tkv_pages_compact_args": ("workspace", "table_stride", "B", "num_pages")}
    src = tmp_path / "t.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "tritonkv_b200.h"\nint main(void) {\n' + "".join(
        f'printf("%zu\\n", offsetof({t}, {f}));\n' for t, fs in fields.items() for f in fs) + "return 0; }\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = tmp_path / "t"
    subprocess.run([gcc, "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    at = lambda form: struct.calcsize("@" + form)  # the offset of what follows `form`
    want = [at("10P"), at("11P"), at("12P"), at("12Pq"), at("12P2q"), at("12P2q10i"), at("12P2q11i"),
            0, at("12P"), at("13P"), at("13P6q"), at("13P12q"), at("13P13q"), at("13P13q10i"),
            at("3P"), at("7P"), at("8P"), at("8Pq"), at("8Pq5i"), at("3P"), at("4P"), at("4Pq"), at("4Pq2i")]
    assert got == want
    assert _cabi.PAGED_DECODE_ARGS.size == at("12P2q11if") and _cabi.PAGED_APPEND_ARGS.size == at("13P13q11i")
    assert _cabi.PAGES_FORK_ARGS.size == at("8Pq6i") and _cabi.PAGES_COMPACT_ARGS.size == at("4Pq3i")
