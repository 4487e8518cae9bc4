"""The workspace of a stream under capture, with the library's allocation and the capture
state faked; no device is touched."""
import ctypes

import pytest
import torch


@pytest.fixture
def faked(hyperion, monkeypatch):
    """(capturing flag, blocks the library gave): the current stream is number 77."""
    h, state, given = hyperion, {"capturing": False}, []

    def alloc(nbytes, ptr):
        given.append(ctypes.create_string_buffer(nbytes))
        ctypes.cast(ptr, ctypes.POINTER(ctypes.c_void_p))[0] = ctypes.addressof(given[-1])
        return 0

    zeros = torch.zeros

    def torch_zeros(*args, device=None, **kw):
        assert not state["capturing"]  # it would be the graph's memory and the graph's fill
        return zeros(*args, **kw)

    monkeypatch.setattr(h._capi.lib, "hyperion_workspace_alloc", alloc)
    monkeypatch.setattr(h, "_raw_stream", lambda idx: 77)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    monkeypatch.setattr(torch, "zeros", torch_zeros)
    for name in ("_workspaces", "_captured", "_retired"):
        monkeypatch.setattr(h, name, type(getattr(h, name))())
    return h, state, given


DEV = torch.device("cuda", 0)


def test_a_block_first_needed_under_capture_is_the_librarys(faked):
    h, state, given = faked
    state["capturing"] = True
    ws = h._workspace(DEV, 100)
    assert len(given) == 1 and ws.data_ptr() == ctypes.addressof(given[0]) and ws.numel() == 1 << 16
    assert h._workspace(DEV, 1 << 16) is ws
    state["capturing"] = False
    assert h._workspace(DEV, 300) is ws  # eager calls of the stream go on with it
    big = h._workspace(DEV, 1 << 17)
    assert isinstance(big, torch.Tensor) and h._retired == {(0, 77): [ws]}  # a graph holds the first


def test_a_block_outgrown_under_capture_stays_with_its_flags(faked):
    h, state, given = faked
    ws = h._workspace(DEV, 100)
    ws[64] = 2
    state["capturing"] = True
    assert h._workspace(DEV, 100) is ws and not given
    big = h._workspace(DEV, 1 << 17)
    assert big.numel() == 1 << 17 and h._retired == {(0, 77): [ws]}
    assert ws[64] == 2 and bytes(given[0].raw[:256]) == bytes(256)  # read where they were raised


def test_a_block_no_graph_has_seen_is_replaced_with_its_flags(faked):
    h, state, given = faked
    ws = h._workspace(DEV, 100)
    ws[64] = 2
    big = h._workspace(DEV, 1 << 17)
    assert big[64] == 2 and not h._retired and not given


def test_a_workspace_of_no_room_is_refused(hyperion):
    capi = hyperion._capi
    ptr = ctypes.c_void_p()
    assert capi.lib.hyperion_workspace_alloc(255, ctypes.byref(ptr)) == capi.HYPERION_ERR_INVALID_ARG
    assert capi.lib.hyperion_workspace_alloc(256, None) == capi.HYPERION_ERR_INVALID_ARG
    assert not ptr.value and capi.last_error()
