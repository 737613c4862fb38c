"""Outputs of the paged-cache functions that overlap one another are refused, without a GPU."""

import pytest
import torch

from tritonkv_b200.paged import append_kv_paged, compact_pages, fork_pages
from tritonkv_b200.quantize import empty_cache


def pool():
    return empty_cache(6, 2, 16, 64, 4, 32, "cpu")


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_fork_and_compact():
    one, row = i32(1), i32(6)
    for out in ((i32(1, 5), one, one), (row[:5].view(1, 5), row[4:5], one), (row[:5].view(1, 5), one, row[:1])):
        with pytest.raises(ValueError, match="share memory"):
            fork_pages(pool(), i32(3, 5), i32(3), i32(1), out=out)
    with pytest.raises(ValueError, match="share memory"):
        compact_pages(pool(), i32(1, 5), out=(row[:5].view(1, 5), row[4:5]))
    for call in (lambda: fork_pages(pool(), i32(3, 5), i32(3), i32(1), out=(row[:5].view(1, 5), row[5:], one)),
                 lambda: compact_pages(pool(), i32(1, 5), out=(row[:5].view(1, 5), row[5:])),
                 lambda: fork_pages(pool(), i32(3, 5), i32(3), i32(0), out=(i32(0, 5), i32(0), one))):
        with pytest.raises(RuntimeError, match="CUDA"):  # (there is no CPU path: the checks are passed)
            call()


@pytest.mark.parametrize("axis", [0, 1, 2])
def test_values_of_an_append(axis):
    """A values tensor that is expanded along an axis has one row for several tokens."""
    shape = [3, 2, 4, 64]
    shape[axis] = 1
    x, val = torch.zeros(3, 2, 4, 64).half(), torch.zeros(*shape).half().expand(3, 2, 4, 64)
    for kw in (dict(k_values=val), dict(v_values=val)):
        with pytest.raises(ValueError, match="row for every token"):
            append_kv_paged(pool(), pool(), x, x, i32(3, 5), 0, **kw)
    y = x[:, :, :1]
    with pytest.raises(RuntimeError, match="CUDA"):
        append_kv_paged(pool(), pool(), y, y, i32(3, 5), 0, k_values=torch.zeros(3, 2, 64).half()[:, :, None])
