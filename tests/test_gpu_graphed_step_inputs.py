"""The captured step reads the tensors that it was made with: they live as long as it does."""

import gc
import weakref

import pytest
import torch

from tritonkv_b200 import GraphedDecodeStep
from tritonkv_b200.quantize import empty_cache

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("paged", [False, True])
def test_inputs_live_as_long_as_the_step(paged):
    k, v = (empty_cache(6, 2, 32, 64, 4, 32, DEV) for _ in range(2))
    lens = torch.tensor([20] * (3 if paged else 6), dtype=torch.int32, device=DEV)
    table = torch.arange(6, dtype=torch.int32, device=DEV).view(3, 2) if paged else None
    refs = [weakref.ref(t) for t in (k.packed, k.scale, k.zero, v.packed, v.scale, v.zero, lens) + ((table,) if paged else ())]
    step = GraphedDecodeStep(k, v, 4, seq_lens=lens, block_table=table)
    del k, v, lens, table
    gc.collect()
    assert all(r() is not None for r in refs)
    del step
    gc.collect()
    assert all(r() is None for r in refs)
