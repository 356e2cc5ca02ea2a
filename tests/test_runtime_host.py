"""CPU tier: a runtime over a stand-in for the library — what a workspace frees and when, and in which order the calls of a
batch scope reach the engine."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from k100lc_kernels import Runtime, Workspace


class _Engine:
    """Stands in for the library: allocations, graphs and the order in which launches reach the engine."""

    def __init__(self):
        self.next, self.freed, self.graphs, self.order = 0, [], 0, []

    def fm_alloc(self, n):
        self.next += 4096
        return self.next

    def fm_free(self, p):
        self.freed.append(int(p.value))

    def fm_graph_begin(self):
        return 0

    def fm_graph_end(self):
        self.graphs += 1
        return self.graphs - 1

    def fm_graph_free(self, graph):
        return 0

    def fm_kernel_id(self, name):
        return len(name)

    def fm_launch_batch(self, buf, n):
        at = 0
        for _ in range(n):
            self.order.append(buf[at + 4])               # the first argument names the launch
            at += 4 + buf[at + 3]
        return n

    def fm_launch2d(self, name, gx, gy, wx, wy, argv, n):
        self.order.append(argv[0])
        return 0

    def fm_launch_dyn(self, name, gx, gy, wx, wy, layout, n, group, private, kernarg, argv, nargv):
        self.order.append(argv[0])
        return 0

    def _other(self, name):
        def call(*args):
            self.order.append(name)
            return 0
        return call

    def __getattr__(self, name):
        if name in ("fm_upload", "fm_download", "fm_copy", "fm_memset", "fm_sync", "fm_upload_async", "fm_download_async", "fm_graph_launch"):
            return self._other(name)
        raise AttributeError(name)


def _runtime(engine):
    """A Runtime over the stand-in (no library, no device)."""
    rt = Runtime.__new__(Runtime)
    rt._lib, rt._pending, rt._argv, rt._enc, rt._ids, rt._names_by_id = engine, None, (ctypes.c_uint64 * 32)(), {}, {}, {}
    rt._graphs, rt.catalog = set(), {"kernels": [{"name": "k", "args": []}]}
    return rt


def test_workspace_keeps_what_a_captured_graph_holds():
    """A block that has to grow is freed at once while no captured graph is alive, and otherwise kept: the graph's kernels
    have its address."""
    eng = _Engine()
    rt = _runtime(eng)
    with Workspace(rt) as ws:
        a = ws.buffer("a", 100)
        b = ws.buffer("a", 200)
        assert eng.freed == [a]
        rt.graph_begin()
        assert ws.buffer("a", 150) == b
        one = rt.graph_end()
        rt.graph_begin()
        two = rt.graph_end()
        c = ws.buffer("a", 300)
        assert c != b and eng.freed == [a]
        rt.graph_free(one)
        d = ws.buffer("a", 400)
        assert eng.freed == [a]
        rt.graph_free(two)
        e = ws.buffer("a", 500)
        assert sorted(eng.freed) == [a, b, c, d]
    assert sorted(eng.freed) == [a, b, c, d, e]


def test_workspace_forgets_a_block_that_it_could_not_replace():
    eng = _Engine()
    rt = _runtime(eng)
    ws = Workspace(rt)
    a = ws.buffer("a", 100)
    eng.fm_alloc = lambda n: 0
    with pytest.raises(MemoryError):
        ws.buffer("a", 200)
    assert eng.freed == [a] and ws.size("a") == 0
    ws.free()
    assert eng.freed == [a]


def test_batch_scope_keeps_the_order_of_the_calls():
    """Launches are recorded; any other call that works on the device comes after those in front of it."""
    eng = _Engine()
    rt = _runtime(eng)
    x = np.zeros(4, np.float32)
    with rt.batch():
        rt.launch("k", 1, 1, [1])
        rt.launch("k", 1, 1, [2])
        assert eng.order == []
        rt.launch2d("k", 1, 1, 1, 1, [3])
        assert eng.order == [1, 2, 3]
        for call in (lambda: rt.upload(64, x), lambda: rt.download(64, 4, np.float32), lambda: rt.copy_dev(64, 128, 16), lambda: rt.memset(64, 0, 16),
                     rt.sync, lambda: rt.upload_async(64, x), lambda: rt.download_async(x, 64), lambda: rt.graph_launch(0),
                     lambda: rt.launch_dyn("k", 1, 1, 1, 1, [5]), lambda: rt.launch_any("k", 1, 1, [5])):
            eng.order.clear()
            rt.launch("k", 1, 1, [4])
            call()
            assert eng.order[0] == 4 and len(eng.order) == 2
        eng.order.clear()
        rt.launch("k", 1, 1, [6])
    assert eng.order == [6]
    with rt.batch():
        rt.launch2d("k", 1, 1, 1, 1, [7])
    assert eng.order == [6, 7]
