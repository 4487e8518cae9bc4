"""The workspace of a stream whose calls are captured: its error word is sticky until read,
whatever has been replayed, and no block that a graph uses is given back."""
import numpy as np
import pytest
import torch

from cache_ops_reference import make_table
from hyperion_b200 import glue

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
i32 = torch.int32


def _new_stream(h):
    """A stream without a workspace yet (torch hands the same few out again)."""
    s = torch.cuda.Stream(DEV)
    h._workspaces.pop((0, s.cuda_stream), None)
    s.wait_stream(torch.cuda.current_stream())
    return s


def _flags(h, s, clear=True):
    with torch.cuda.stream(s):
        return h.read_device_errors(DEV, clear=clear)


class _Call:
    """Key weights of one query a row; a page of the table can be spoilt in place."""

    def __init__(self, h):
        rng = np.random.default_rng(1)
        self.h, self.table = h, make_table(2, 4, 0).to(DEV)
        self.good = int(self.table[1, 2])
        words = lambda n: torch.from_numpy(rng.integers(-2**31, 2**31, (n, 4), dtype=np.int64).astype(np.int32)).to(DEV)  # noqa: E731
        self.q, self.k = words(2), words(2 * 4 * 16)
        self.ctx = torch.tensor([64, 50], dtype=i32, device=DEV)
        self.w = torch.zeros(2, 64, device=DEV)
        self.out = torch.zeros_like(self.w)
        torch.cuda.synchronize()

    def spoil(self, bad):
        self.table[1, 2] = -1 if bad else self.good
        torch.cuda.synchronize()

    def __call__(self):
        self.h.accumulate_key_weights(self.q, self.k, self.ctx, self.table, self.w, 1, 128, 16, 4, 0.1, False, out=self.out)

    def captured(self, s, before=None):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            if before:
                before()
            self()
        return g


def _replay(g, s):
    with torch.cuda.stream(s):
        g.replay()
    s.synchronize()


def test_a_replays_flags_last_until_they_are_read(hyperion):
    h, call = hyperion, _Call(hyperion)
    call()
    s, other = _new_stream(h), torch.cuda.Stream(DEV)
    g = call.captured(s)  # the first call on this stream is a captured one
    call.spoil(True)
    _replay(g, s)
    call.spoil(False)
    _replay(g, s)
    assert _flags(h, s, clear=False) == h.DEVERR_BAD_BLOCK  # of the first replay
    assert _flags(h, s) == h.DEVERR_BAD_BLOCK
    _replay(g, s)
    assert _flags(h, s) == 0
    call.spoil(True)
    _replay(g, other)  # a replay flags where its call was captured
    assert _flags(h, s) == h.DEVERR_BAD_BLOCK and _flags(h, other) == 0


def test_a_workspace_first_used_under_capture_holds_no_flags_of_its_own(hyperion):
    h, call = hyperion, _Call(hyperion)
    call()
    s = _new_stream(h)

    def scratch_of_the_graph():  # every replay writes over what this gives back
        x = torch.full((1 << 16,), 0xFF, dtype=torch.uint8, device=DEV)
        del x

    g = call.captured(s, scratch_of_the_graph)
    assert _flags(h, s) == 0  # before any replay
    with torch.cuda.stream(s):
        call()
    assert _flags(h, s) == 0
    for _ in range(3):
        _replay(g, s)
        assert _flags(h, s) == 0


def test_two_graphs_of_one_stream_keep_each_others_flags(hyperion):
    h, call = hyperion, _Call(hyperion)
    call()
    s = _new_stream(h)
    first, second = call.captured(s), call.captured(s)
    call.spoil(True)
    _replay(second, s)
    call.spoil(False)
    _replay(first, s)
    assert _flags(h, s) == h.DEVERR_BAD_BLOCK
    del first
    torch.cuda.synchronize()
    call.spoil(True)
    _replay(second, s)
    assert _flags(h, s) == h.DEVERR_BAD_BLOCK


def _forward(h, call):
    """A forward whose split-KV partials outgrow the workspace of the other calls."""
    rows, D = 64, 128
    g = torch.Generator().manual_seed(0)
    q = torch.randint(-2**31, 2**31, (rows, D // 32), generator=g).to(i32).to(DEV)
    k = torch.randint(-2**31, 2**31, (rows * 256, D // 32), generator=g).to(i32).to(DEV)
    v = torch.randint(0, 0x7F, (rows * 256, D), generator=g).to(torch.uint8).to(DEV)
    ctx = torch.full((rows,), 256, dtype=i32, device=DEV)
    wl = glue.build_worklist(torch.ones(1, dtype=i32, device=DEV), rows)
    scale = torch.ones(1, device=DEV)

    def run(splits):
        o = torch.zeros(rows, D, dtype=torch.float32, device=DEV)
        h.hyperion_apex_kernel(wl, rows, q, None, k, None, v, scale, ctx, None, o, 1, D, D // 8, 256, 1, 0.1, False, path="row",
                               num_splits=splits)
        return o

    return run


@pytest.mark.parametrize("grown_under_capture", [False, True])
def test_growing_a_workspace_keeps_what_a_graph_uses_and_every_flag(hyperion, grown_under_capture):
    h, call = hyperion, _Call(hyperion)
    forward = _forward(h, call)
    want = forward(8)  # on a stream of its own, once
    s = _new_stream(h)
    with torch.cuda.stream(s):
        call()
        small = h._workspace(DEV, 1 << 16)
    first = call.captured(s)
    with torch.cuda.stream(s):
        call.spoil(True)
        call()  # an eager flag, not read yet
        call.spoil(False)
    if grown_under_capture:
        second = torch.cuda.CUDAGraph()
        with torch.cuda.graph(second, stream=s):
            o = forward(8)
    else:
        with torch.cuda.stream(s):
            o = forward(8)
    with torch.cuda.stream(s):
        assert h._workspace(DEV, 1 << 16).numel() > small.numel()
    address = small.data_ptr()
    del small
    # what a freed block would be given to
    with torch.cuda.stream(s):
        taken = [torch.full((1 << 16,), 0xEE, dtype=torch.uint8, device=DEV) for _ in range(8)]
    assert all(t.data_ptr() != address for t in taken)
    s.synchronize()
    assert _flags(h, s) == h.DEVERR_BAD_BLOCK  # the eager call's
    call.spoil(True)
    _replay(first, s)
    assert all(bool((t == 0xEE).all()) for t in taken)
    assert _flags(h, s) == h.DEVERR_BAD_BLOCK  # of a graph on the outgrown block
    assert _flags(h, s) == 0
    if grown_under_capture:
        for _ in range(2):
            o.zero_()
            torch.cuda.synchronize()
            _replay(second, s)
            assert torch.equal(o, want)
    s.synchronize()
    assert torch.equal(o, want) and _flags(h, s) == 0
