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


@pytest.fixture(autouse=True)
def sizes(monkeypatch):
    """(the library's sizes need a device: stand-ins for the time of a test)"""
    monkeypatch.setattr(_cabi, "_paged_bytes", {})


def decode_key(B, dev=0):
    key = (B, 8, 8, 16, 128, 4, 32, dev)
    _cabi._paged_bytes[key] = (min(B, 512) * 8 + 444) * 8 * 130 * 4
    return key


def test_partials_of_a_growing_batch():
    """A batch that climbs by ones: what is outgrown stays for the graphs that may use it, and is bounded."""
    ws, tickets = {}, None
    for B in range(1, 513):
        key = decode_key(B)
        kept = _cabi.paged_workspace(ws, key, CPU)
        assert kept[0] == key and kept[4].numel() == kept[2] >= _cabi._paged_bytes[key] and kept[1] == kept[4].data_ptr()
        tickets = kept[5] if tickets is None else tickets
        assert kept[5] is tickets and kept[3] == tickets.data_ptr()
    assert kept_bytes(ws) <= 4 * _cabi._paged_bytes[key] + tickets.nbytes
    assert _cabi.paged_workspace(ws, key, CPU) is kept
    assert _cabi.paged_workspace(ws, decode_key(5), CPU)[4] is kept[4]


def test_partials_of_two_devices_in_turn():
    """One dict used on two devices: each finds its own buffers again."""
    ws, first = {}, {}
    for i in range(40):
        dev = i % 3
        kept = _cabi.paged_workspace(ws, decode_key(16, dev), CPU if dev else META)
        assert first.setdefault(dev, kept[4]) is kept[4] and kept[0][7] == dev
    assert len({id(t) for t in kept_tensors(ws)}) == 6


def test_without_a_dict_nothing_is_kept():
    a, b = (_cabi.paged_workspace(None, decode_key(2), CPU) for _ in range(2))
    assert a[4] is not b[4] and not a[5].any() and not b[5].any()


def test_what_a_capture_makes_is_its_own(monkeypatch):
    """Memory that is cleared by a node of a graph holds anything until the graph has run: neither another call nor
    another graph may find it."""
    ws = {}
    monkeypatch.setattr(_cabi, "capturing", lambda: True)
    seen = [paged._pages_workspace(ws, 4, 100, CPU), _cabi.paged_workspace(ws, decode_key(4), CPU)[5]]
    assert not kept_tensors(ws)
    monkeypatch.setattr(_cabi, "capturing", lambda: False)
    mine = [paged._pages_workspace(ws, 4, 100, CPU), _cabi.paged_workspace(ws, decode_key(4), CPU)]
    assert mine[0] is not seen[0] and mine[1][5] is not seen[1]
    monkeypatch.setattr(_cabi, "capturing", lambda: True)  # what was there before the capture serves it
    assert paged._pages_workspace(ws, 3, 100, CPU) is mine[0]
    assert _cabi.paged_workspace(ws, decode_key(3), CPU)[4] is mine[1][4]
    more = _cabi.paged_workspace(ws, decode_key(300), CPU)  # (cleared tickets are there; partials need no clearing)
    assert more[4] is not mine[1][4] and more[5] is mine[1][5] and ws["paged"][4] is mine[1][4]
    assert paged._pages_workspace(ws, 300, 100, CPU) is not mine[0] and len(kept_tensors(ws)) == 3
