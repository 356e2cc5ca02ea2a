"""CPU tier: argument checks and launch sequences of the routing and epilogue-product classes, the plan of the plain
form against the host routing of MoEExperts, and the plain forms against themselves."""
from __future__ import annotations

import numpy as np
import pytest

import moe_plain as P
from k100lc_kernels import ExpertLinear, FusedLinear, MoEExperts, MoEMLP, MoEPlan, MoERouter, catalog
from test_host_logic import _RecordingRuntime


class Recorder(_RecordingRuntime):
    def __init__(self):
        super().__init__(set())
        self.uploads = []

    def upload(self, ptr, data):
        self.uploads.append((ptr, np.asarray(data).nbytes))

    def memset(self, ptr, value, nbytes):
        self.launches.append(("memset", value, nbytes, 0))


def test_router_refuses():
    rt = Recorder()
    for kw in (dict(n_exp=0, topk=1), dict(n_exp=1025, topk=1), dict(n_exp=8, topk=9), dict(n_exp=64, topk=33),
               dict(n_exp=8, topk=0), dict(n_exp=8, topk=1, n_group=3), dict(n_exp=66, topk=1, n_group=33),
               dict(n_exp=8, topk=1, n_group=4, topk_group=5), dict(n_exp=8, topk=3, n_group=4, topk_group=1),
               dict(n_exp=8, topk=1, group_top=3), dict(n_exp=8, topk=1, score="linear"), dict(n_exp=8, topk=1, dtype="f64"),
               dict(n_exp=8, topk=1, bias=np.zeros(7, np.float32)), dict(n_exp=8, topk=1, topk_group=0)):
        with pytest.raises(ValueError):
            MoERouter(rt, **kw)
    r = MoERouter(rt, 8, 2)
    with pytest.raises(ValueError):
        r.forward_device(64, -1)
    with pytest.raises(ValueError):
        r.forward(np.zeros((3, 7), np.float32))
    with pytest.raises(ValueError):
        MoERouter(rt, 8, 2, dtype="bf16").forward(np.zeros((3, 8), np.float32))
    assert not rt.launches


def test_products_refuse():
    rt = Recorder()
    for kw in (dict(n=0, k=128), dict(n=4, k=64), dict(n=4, k=192), dict(n=4, k=128, act="tanh"),
               dict(n=4, k=128, bias=np.zeros(5, np.float32)), dict(n=4, k=128, gated=True, bias=np.zeros(4, np.float32))):
        with pytest.raises(ValueError):
            FusedLinear(rt, wq=64, ws_scale=128, **kw)
        with pytest.raises(ValueError):
            ExpertLinear(rt, 1, wq=64, ws_scale=128, **kw)
    with pytest.raises(ValueError):
        ExpertLinear(rt, 0, 4, 128, 64, 128)
    lin = FusedLinear(rt, 4, 128, 64, 128)
    for kw in (dict(rows=-1), dict(rows=1, ldy=3), dict(rows=1, ldr=3)):
        with pytest.raises(ValueError):
            lin.forward_codes_device((1, 2, 3, 4), **kw)
    with pytest.raises(ValueError):
        lin.forward(np.zeros((2, 256), np.float32))
    with pytest.raises(ValueError):
        lin.forward(np.zeros((2, 128), np.float32), np.zeros((1, 4), np.float32))
    plan = MoEPlan(rows=3, topk=2, n_exp=5, ids=1, weights=1, bucket_rows=1, base=1, offsets=1)
    with pytest.raises(ValueError):
        ExpertLinear(rt, 4, 4, 128, 64, 128).forward_codes_device((1, 2, 3, 4), plan)
    router = MoERouter(rt, 4, 2)
    gate, plain = ExpertLinear(rt, 4, 128, 256, 1, 2, gated=True), ExpertLinear(rt, 4, 256, 128, 1, 2)
    MoEMLP(rt, router, gate, plain)
    for g, d, r in ((plain, plain, router), (gate, gate, router), (gate, plain, MoERouter(rt, 5, 2)),
                    (gate, ExpertLinear(rt, 4, 128, 128, 1, 2), router)):
        with pytest.raises(ValueError):
            MoEMLP(rt, r, g, d)
    assert not rt.launches


def test_launch_sequence_and_argument_counts():
    """The block queues its launches without a synchronisation or a download, each with as many arguments as the
    library's table names."""
    rt = Recorder()
    router = MoERouter(rt, 4, 2, bias=np.zeros(4, np.float32))
    block = MoEMLP(rt, router, ExpertLinear(rt, 4, 128, 256, 1, 2, act="silu", gated=True), ExpertLinear(rt, 4, 256, 128, 1, 2))
    block.forward_device(64, 128, 5)
    names = [l[0] for l in rt.launches]
    assert names == ["moe_route_plan_k", "memset", "quant_act", "moe_linear_w4a8_k", "quant_act", "moe_linear_w4a8_k",
                     "moe_combine_gather_k"]
    FusedLinear(rt, 4, 128, 64, 128, bias=77).forward_device(64, 3, residual_dev=4096)
    for name, _grid, _wg, nargs in rt.launches:
        if name != "memset":
            assert len(catalog.info(name)["args"]) == nargs, name
    rt.launches.clear()
    block.forward_device(64, 128, 0)
    assert rt.launches == []
    FusedLinear(rt, 4, 128, 64, 128).forward_device(64, 70000)
    assert [l[:2] for l in rt.launches] == [("quant_act", (1, 65535)), ("quant_act", (1, 4465)), ("linear_w4a8_k", 1)]


def test_plain_plan_is_the_host_routing():
    rng = np.random.default_rng(3)
    ids = rng.integers(-1, 7, size=(9, 3))
    w = rng.random((9, 3)).astype(np.float32)
    w[2, 1] = 0
    moe = MoEExperts(Recorder(), [None] * 6, 9, 4, 4, 3)
    for a, b in zip(moe.route(ids, w), P.plan(ids, w, 6)):
        assert np.array_equal(a, b)


def test_plain_route_by_hand():
    x = np.array([[1.0, 3.0, 3.0, -np.inf], [np.nan, -np.inf, -np.inf, -np.inf], [0.0, 0.0, 0.0, 0.0]], np.float32)
    ids, w = P.route(x, 2)
    assert ids.tolist() == [[1, 2], [-1, -1], [0, 1]]
    assert np.allclose(w, [[0.5, 0.5], [0, 0], [0.5, 0.5]])
    ids, w = P.route(np.array([[2.0, 0.0, 1.0, 0.9]], np.float32), 1, "sigmoid", n_group=2, topk_group=1, group_top=2, renorm=False)
    assert ids.tolist() == [[2]]                       # 0.73 + 0.71 against 0.88 + 0.5
    assert np.allclose(w, 1 / (1 + np.exp(-1.0)))
