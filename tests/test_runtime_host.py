"""CPU tier: a runtime over a stand-in for the library — what a workspace frees, and when."""
from __future__ import annotations

import ctypes

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


def _runtime(engine):
    """A Runtime over the stand-in (no library, no device)."""
    rt = Runtime.__new__(Runtime)
    rt._lib, rt._pending, rt._argv, rt._enc, rt._ids, rt._names_by_id = engine, None, (ctypes.c_uint64 * 32)(), {}, {}, {}
    rt._graphs = set()
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
