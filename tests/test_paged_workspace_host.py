"""What the paged-cache functions keep in a caller's `_workspace`, without a GPU."""

import pytest
import torch

from tritonkv_b200 import _cabi, paged

CPU, META = torch.device("cpu"), torch.device("meta")


def kept_tensors(x):
    if isinstance(x, torch.Tensor):
        return [x]
    if isinstance(x, dict):
        x = list(x.values())
    return [t for y in x for t in kept_tensors(y)] if isinstance(x, (list, tuple)) else []


def kept_bytes(ws):
    return sum({id(t): t.nbytes for t in kept_tensors(ws)}.values())


def test_page_scratch_of_two_pools_in_turn():
    """One dict used for pools of different sizes: an earlier scratch is found again, with what it holds."""
    ws, first = {}, {}
    for i in range(60):
        NP, dev = ((8000, CPU), (2000, CPU), (2000, META))[i % 3]
        t = paged._pages_workspace(ws, 16, NP, dev)
        assert t.device == dev and t.numel() >= 4 + 2 * (-(-NP // 32)) + 3 * NP + 2 * 16
        if dev == CPU and i < 3:
            assert not t.any()
            t[-1] = NP
        assert first.setdefault((NP, dev), t) is t
    assert int(first[8000, CPU][-1]) == 8000 and int(first[2000, CPU][-1]) == 2000
    assert len({id(t) for t in kept_tensors(ws)}) == 3


def test_page_scratch_of_a_growing_batch():
    ws = {}
    for B in range(1, 513):
        t = paged._pages_workspace(ws, B, 100, CPU)
        assert t.numel() >= 4 + 2 * 4 + 300 + 2 * B
    assert len({id(t) for t in kept_tensors(ws)}) <= 12
    assert paged._pages_workspace(ws, 3, 100, CPU) is t
