"""GPU tier: the W4A8 products with an epilogue (dense and per expert) against the plain 64-bit form, element by element
within the error of their fp32 sums, the whole mixture-of-experts block, and the calls that are refused."""
from __future__ import annotations

import numpy as np
import pytest

import moe_plain as P
from gpu_util import Bufs
from k100lc_kernels import ExpertLinear, FusedLinear, MoEExperts, MoEMLP, MoEPlan, MoERouter, RT4Linear, Workspace

pytestmark = pytest.mark.gpu


def _within(got, want, bound):
    assert np.all(np.isfinite(got))
    bad = np.abs(got - want) > bound
    assert not bad.any(), (int(bad.sum()), float((np.abs(got - want) / bound).max()), np.argwhere(bad)[:5].tolist())


def _dense(rt, m, n, k, act="none", gated=False, bias=False, residual=False, seed=0, ldy=None, ldr=None, in_place=False):
    rng = np.random.default_rng(seed + m * 7 + n * 3 + k)
    wq, ws, w = P.layer(rng, 1, n * (2 if gated else 1), k)
    cd, q = P.codes(rng, m, k)
    b = rng.standard_normal(w.shape[1]).astype(np.float32) if bias else None
    r = (rng.standard_normal((m, n)) * 3).astype(np.float32) if residual else None
    ldy, ldr = ldy or n, ldr or n
    with Bufs(rt) as bf:
        lin = FusedLinear(rt, n, k, bf.put(wq), bf.put(ws), bias=b, act=act, gated=gated)
        pad = np.full((m, ldr), np.nan, np.float32)
        if residual:
            pad[:, :n] = r
        pr = bf.put(pad) if residual else None
        out = pr if in_place else bf.zeros(m * ldy, np.float32, -777.0)
        lin.forward_codes_device([bf.put(c) for c in cd], m, residual_dev=pr, out_dev=out, ldy=ldy, ldr=ldr)
        got = bf.get(out, m * ldy).reshape(m, ldy)
        assert rt.gemm_status() == 0
        lin.ws.free()
    if not in_place:
        assert np.all(got[:, n:] == -777.0)
    want, bound = P.epilogue(*P.product(w[0], ws[0], q, cd[2]), act, gated, b, r)
    _within(got[:, :n], want, bound)


@pytest.mark.parametrize("m", [1, 2, 5, 8, 9, 16, 17, 31, 64, 100, 129, 300])
@pytest.mark.parametrize("n,k", [(1, 128), (40, 256), (129, 1152), (1000, 640)])
def test_dense_sizes(rt, m, n, k):
    _dense(rt, m, n, k)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 72, 1024), (3, 7, 384), (40, 200, 512), (150, 65, 256)])
def test_dense_epilogue(rt, act, gated, m, n, k):
    _dense(rt, m, n, k, act, gated, bias=True, residual=True)
    _dense(rt, m, n, k, act, gated, bias=True, seed=1)
    _dense(rt, m, n, k, act, gated, residual=True, seed=2)


@pytest.mark.parametrize("m", [1, 20, 200])
def test_dense_row_strides_and_residual_in_place(rt, m):
    _dense(rt, m, 130, 256, "silu", bias=True, residual=True, ldy=200, ldr=135)
    _dense(rt, m, 130, 256, "silu", residual=True, in_place=True)
    _dense(rt, m, 130, 256, "silu", residual=True, in_place=True, ldy=133, ldr=133, gated=True)


@pytest.mark.parametrize("m,n,k", [(1, 17408, 5120), (4, 5120, 17408), (77, 1024, 5120), (2, 6144, 6144)])
def test_dense_model_shapes(rt, m, n, k):
    _dense(rt, m, n, k, "gelu", bias=True)


# From here to the experts: enough rows and weights for the tensor-core tiles.  One group and odd numbers of groups, rows of
# weights and of x that end inside a tile, more tiles than an SM (so that a CTA walks several).
@pytest.mark.parametrize("m,n,k", [(300, 1000, 5120), (700, 1000, 1152), (4100, 129, 1152), (3000, 1000, 128), (129, 17408, 1152), (65, 17407, 1280),
                                   (2049, 1300, 384), (300, 1000, 25728)])
def test_tiles_sizes(rt, m, n, k):
    _dense(rt, m, n, k)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("gated", [False, True])
def test_tiles_epilogue(rt, act, gated):
    _dense(rt, 1030, 700, 1152, act, gated, bias=True, residual=True)
    _dense(rt, 1030, 700, 1152, act, gated, bias=True, seed=1)
    _dense(rt, 1030, 700, 1152, act, gated, residual=True, seed=2)


def test_tiles_row_strides_and_residual_in_place(rt):
    _dense(rt, 1030, 700, 1152, "silu", bias=True, residual=True, ldy=711, ldr=705)
    _dense(rt, 1030, 700, 1152, residual=True, in_place=True)
    _dense(rt, 1030, 700, 1152, "silu", residual=True, in_place=True)
    _dense(rt, 1030, 700, 1152, "silu", residual=True, in_place=True, ldy=703, ldr=703, gated=True)


@pytest.mark.parametrize("m,n,k,gated", [(513, 5000, 640, False), (513, 2500, 640, True), (1000, 5000, 128, False), (300, 17408, 5120, False)])
def test_tiles_repeat_bit_for_bit(rt, m, n, k, gated):
    """Forty calls in a row: a role that gets ahead of another would show as another sum or as a wait that ran out."""
    rng = np.random.default_rng(m)
    wq, ws, _ = P.layer(rng, 1, n * (2 if gated else 1), k)
    cd, _ = P.codes(rng, m, k)
    with Bufs(rt) as b:
        lin = FusedLinear(rt, n, k, b.put(wq), b.put(ws), act="silu", gated=gated)
        dev, outs = [b.put(c) for c in cd], [b.zeros(m * n) for _ in range(2)]
        lin.forward_codes_device(dev, m, out_dev=outs[0])
        first = b.get(outs[0], m * n)
        for i in range(40):
            lin.forward_codes_device(dev, m, out_dev=outs[1])
            if i % 8 == 7:
                assert np.array_equal(b.get(outs[1], m * n), first)
        assert rt.gemm_status() == 0


def test_tiles_and_placement_in_graphs(rt):
    """Two captured runs of a router of many tokens and of products on tiles, replayed in turn with other inputs: the graphs
    share the engine's workspace, and each holds launches that begin while the one in front ends."""
    rng = np.random.default_rng(6)
    rows, n_exp, n, k = 900, 6, 600, 1152
    wq, ws, w = P.layer(rng, n_exp, n, k)
    with Bufs(rt) as b:
        router = [MoERouter(rt, n_exp, 2) for _ in range(2)]
        experts = ExpertLinear(rt, n_exp, n, k, b.put(wq), b.put(ws))
        dense = FusedLinear(rt, n, k, experts.wq, experts.ws_scale, act="silu")
        px, pl = b.zeros(rows * k), b.zeros(rows * n_exp)
        pe, pd = [b.zeros(rows * 2 * n) for _ in range(2)], [b.zeros(rows * n) for _ in range(2)]

        def queue(i):
            plan = router[i].forward_device(pl, rows)
            experts.forward_device(px, plan, out_dev=pe[i])
            dense.forward_device(px, rows, out_dev=pd[i])
            return plan

        plans = [queue(i) for i in range(2)]                       # sizes the workspaces
        graphs = []
        for i in range(2):
            rt.graph_begin()
            queue(i)
            graphs.append(rt.graph_end())
        for _ in range(3):
            rt.upload(px, rng.standard_normal((rows, k)).astype(np.float32))
            logits = rng.standard_normal((rows, n_exp)).astype(np.float32)
            rt.upload(pl, logits)
            for g in graphs:
                rt.graph_launch(g)
            got = [(b.get(pe[i], rows * 2 * n), b.get(pd[i], rows * n), b.get(plans[i].offsets, n_exp + 1, np.int32)) for i in range(2)]
            for x, y in zip(*got):
                assert np.array_equal(x, y)
            assert np.array_equal(got[0][2], P.plan(*P.route(logits, 2), n_exp)[3])
            queue(0)
            assert np.array_equal(b.get(pe[0], rows * 2 * n), got[0][0]) and np.array_equal(b.get(pd[0], rows * n), got[0][1])
        assert rt.gemm_status() == 0
        for g in graphs:
            rt.graph_free(g)


def test_dense_is_the_by_name_layer(rt):
    """Without an epilogue the layer is RT4Linear's: both sum the same exact integers, in another order."""
    rng = np.random.default_rng(8)
    wq, ws, w = P.layer(rng, 1, 512, 5120)
    x = rng.standard_normal((4, 5120)).astype(np.float32)
    with Bufs(rt) as b:
        pq, ps = b.put(wq), b.put(ws)
        one, other = RT4Linear(rt, 512, 5120, pq, ps).forward(x), FusedLinear(rt, 512, 5120, pq, ps).forward(x)
        part = FusedLinear(rt, 512, 5120, pq, ps).forward(x[1:2])
    assert np.abs(one - other).max() <= 1e-5 * np.abs(one).max()
    assert np.abs(part - other[1:2]).max() <= 1e-5 * np.abs(one).max()


def _experts(rt, rows, n_exp, topk, n, k, act="none", gated=False, bias=False, gather=True, ids=None, seed=0):
    rng = np.random.default_rng(seed + rows * 5 + n_exp + n + k)
    wq, ws, w = P.layer(rng, n_exp, n * (2 if gated else 1), k)
    if ids is None:
        ids = np.stack([rng.permutation(n_exp)[:topk] for _ in range(rows)]) if rows else np.zeros((0, topk))
    ids = ids.astype(np.int32)
    bucket, base, wz, offsets = P.plan(ids, np.ones(ids.shape, np.float32), n_exp)
    total = bucket.size
    bucket = np.concatenate([bucket, np.full(rows * topk - total, 2 ** 31 - 1, np.int32)])     # slots behind the last bucket
    cd, q = P.codes(rng, rows if gather else rows * topk, k)
    b = rng.standard_normal((n_exp, w.shape[1])).astype(np.float32) if bias else None
    with Bufs(rt) as bf:
        lin = ExpertLinear(rt, n_exp, n, k, bf.put(wq), bf.put(ws), bias=b, act=act, gated=gated)
        plan = MoEPlan(rows=rows, topk=topk, n_exp=n_exp, ids=bf.put(ids), weights=bf.put(wz), bucket_rows=bf.put(bucket), base=bf.put(base),
                       offsets=bf.put(offsets))
        out = bf.zeros(max(1, rows * topk * n), np.float32, -777.0)
        lin.forward_codes_device([bf.put(c) for c in cd], plan, gather=gather, out_dev=out)
        got = bf.get(out, rows * topk * n).reshape(rows * topk, n)
        assert rt.gemm_status() == 0
        lin.ws.free()
    assert np.all(got[total:] == -777.0)
    for e in range(n_exp):
        lo, hi = offsets[e], offsets[e + 1]
        if hi > lo:
            at = bucket[lo:hi] if gather else np.arange(lo, hi)
            want, bound = P.epilogue(*P.product(w[e], ws[e], q[at], cd[2][at]), act, gated, None if b is None else b[e], None)
            _within(got[lo:hi], want, bound)


@pytest.mark.parametrize("rows,n_exp,topk,n,k", [(1, 4, 2, 40, 256), (1, 64, 8, 100, 1024), (9, 6, 2, 33, 384), (33, 3, 3, 70, 128), (50, 130, 4, 24, 256),
                                                 (200, 5, 2, 130, 512), (400, 2, 2, 64, 256), (300, 16, 4, 257, 384)])
@pytest.mark.parametrize("gather", [False, True])
def test_experts_sizes(rt, rows, n_exp, topk, n, k, gather):
    _experts(rt, rows, n_exp, topk, n, k, gather=gather)
    _experts(rt, rows, n_exp, topk, n, k, "silu", True, True, gather)


@pytest.mark.parametrize("rows,n_exp,topk,n,k", [(2000, 5, 2, 130, 1152), (1500, 16, 4, 257, 1152), (1999, 24, 4, 600, 640)])
@pytest.mark.parametrize("gather", [False, True])
def test_experts_tiles(rt, rows, n_exp, topk, n, k, gather):
    _experts(rt, rows, n_exp, topk, n, k, gather=gather)
    _experts(rt, rows, n_exp, topk, n // 2, k, "silu", True, True, gather)


def test_experts_tiles_most_experts(rt):
    _experts(rt, 20000, 1024, 2, 129, 640, bias=True)


def test_experts_tiles_uneven_buckets(rt):
    """Empty experts at both ends and between, buckets of one row and of hundreds, pairs without an expert."""
    rng = np.random.default_rng(3)
    ids = rng.choice([-1, 2, 3, 7, 38], p=[0.1, 0.6, 0.001, 0.199, 0.1], size=(3000, 1))
    for gather in (False, True):
        _experts(rt, 3000, 40, 1, 300, 1152, "gelu", bias=True, gather=gather, ids=ids)
    _experts(rt, 3000, 40, 1, 300, 1152, ids=np.full((3000, 1), -1))


@pytest.mark.parametrize("rows,n,k", [(16, 40, 256), (3000, 300, 1152)])
def test_experts_damaged_plan_writes_nothing(rt, rows, n, k):
    rng = np.random.default_rng(rows)
    wq, ws, _ = P.layer(rng, 3, n, k)
    cd, _ = P.codes(rng, rows, k)
    with Bufs(rt) as b:
        lin = ExpertLinear(rt, 3, n, k, b.put(wq), b.put(ws))
        codes, none = [b.put(c) for c in cd], b.zeros(rows, np.int32)
        for bounds in ([0, 9, 4, rows], [-1, 3, 5, rows], [0, 3, 5, rows + 1], [0, -2 ** 31, 2 ** 31 - 1, rows], [7, 7, 7, 7]):
            plan = MoEPlan(rows=rows, topk=1, n_exp=3, ids=0, weights=0, bucket_rows=none, base=0, offsets=b.put(np.array(bounds, np.int32)))
            for gather in (False, True):
                out = b.zeros(rows * n, np.float32, -777.0)
                lin.forward_codes_device(codes, plan, gather=gather, out_dev=out)
                assert np.all(b.get(out, rows * n) == -777.0)
        assert rt.gemm_status() == 0


def test_experts_uneven_buckets(rt):
    """One expert with every token, experts without any, pairs without an expert, the same expert twice for a token."""
    rng = np.random.default_rng(2)
    ids = np.full((150, 2), 3)
    ids[:, 1] = rng.integers(-1, 6, 150)
    _experts(rt, 150, 5, 2, 70, 256, "gelu", ids=ids)
    _experts(rt, 150, 5, 2, 70, 256, "gelu", gather=False, ids=ids)
    _experts(rt, 4, 5, 2, 70, 256, ids=np.full((4, 2), -1))          # nothing routed: nothing written
    _experts(rt, 0, 5, 2, 70, 256)
    _experts(rt, 64, 1000, 1, 8, 128, ids=np.full((64, 1), 999))


def _block(rt, b, rng, n_exp, topk, dim, ffn, **kw):
    wg, sg, _ = P.layer(rng, n_exp, 2 * ffn, dim)
    wd, sd, _ = P.layer(rng, n_exp, dim, ffn)
    gate = ExpertLinear(rt, n_exp, ffn, dim, b.put(wg), b.put(sg), act="silu", gated=True)
    down = ExpertLinear(rt, n_exp, dim, ffn, b.put(wd), b.put(sd))
    return MoEMLP(rt, MoERouter(rt, n_exp, topk, **kw), gate, down)


@pytest.mark.parametrize("rows", [1, 13, 260])
def test_whole_block_is_its_parts(rt, rows):
    """Router, buckets, gated product, quantiser, down product and combine against the host routing of MoEExperts over one
    FusedLinear per expert: the same integers, so the results agree to fp32's sums wherever the codes of h do."""
    rng = np.random.default_rng(rows)
    n_exp, topk, dim, ffn = 6, 2, 256, 384
    x = rng.standard_normal((rows, dim)).astype(np.float32)
    logits = rng.standard_normal((rows, n_exp)).astype(np.float32)
    with Bufs(rt) as b, Workspace(rt) as ws:
        block = _block(rt, b, rng, n_exp, topk, dim, ffn)
        got = block.forward(x, logits)
        again = block.forward(x, logits)
        assert np.array_equal(got, again)
        ids, w = block.router.forward(logits)

        class Expert:                                      # gate/up, quantiser and down of one expert
            def __init__(self, e):
                g, d = block.gate_up, block.down
                self.up = FusedLinear(rt, ffn, dim, g.wq + e * ffn * dim, g.ws_scale + e * 2 * ffn * (dim // 128) * 2, act="silu", gated=True, ws=ws, tag=f"u{e}")
                self.down = FusedLinear(rt, dim, ffn, d.wq + e * dim * ffn // 2, d.ws_scale + e * dim * (ffn // 128) * 2, ws=ws, tag=f"d{e}")

            def forward_device(self, x_dev, n, out_dev=None, sync=False):
                return self.down.forward_device(self.up.forward_device(x_dev, n), n, out_dev=out_dev)

        ref = MoEExperts(rt, [Expert(e) for e in range(n_exp)], rows, dim, dim, topk, ws).forward(x, ids, w)
    # a code of h that falls on the other side of a rounding moves an output by one step of its group: amax / 127 of h
    # times a weight, about 1e-3 of the output's size
    assert np.abs(got - ref).max() <= 4e-3 * np.abs(ref).max()
    assert np.linalg.norm(got - ref) <= 1e-3 * np.linalg.norm(ref)


def test_block_without_any_expert_is_zero(rt):
    rng = np.random.default_rng(1)
    with Bufs(rt) as b:
        block = _block(rt, b, rng, 4, 2, 128, 128)
        rt.upload(block.ws.buffer(block.tag + ".d", 3 * 2 * 128 * 4), np.full(3 * 2 * 128, np.nan, np.float32))
        y = block.forward(rng.standard_normal((3, 128)).astype(np.float32), np.full((3, 4), -np.inf, np.float32))
    assert np.array_equal(y, np.zeros((3, 128), np.float32))


def test_block_in_a_graph(rt):
    """Captured once, replayed with other inputs and another routing; a second captured block shares the engine's
    workspace."""
    rng = np.random.default_rng(4)
    rows, dim = 70, 256
    with Bufs(rt) as b:
        blocks = [_block(rt, b, rng, 5, 2, dim, 128, score="sigmoid", bias=np.linspace(0, 0.1, 5).astype(np.float32)) for _ in range(2)]
        px, pl, py = b.zeros(rows * dim), b.zeros(rows * 5), [b.zeros(rows * dim) for _ in range(2)]
        for blk, y in zip(blocks, py):
            blk.forward_device(px, pl, rows, out_dev=y, sync=True)     # sizes the workspaces
        graphs = []
        for blk, y in zip(blocks, py):
            rt.graph_begin()
            blk.forward_device(px, pl, rows, out_dev=y)
            graphs.append(rt.graph_end())
        for _ in range(3):
            x, logits = rng.standard_normal((rows, dim)).astype(np.float32), rng.standard_normal((rows, 5)).astype(np.float32)
            rt.upload(px, x)
            rt.upload(pl, logits)
            for g in graphs:
                rt.graph_launch(g)
            got = [b.get(y, rows * dim).reshape(rows, dim) for y in py]
            for blk, y in zip(blocks, got):
                assert np.array_equal(y, blk.forward(x, logits))
        for g in graphs:
            rt.graph_free(g)


def test_products_refuse(rt):
    n, k, m = 16, 256, 3
    with Bufs(rt) as b:
        wq, ws, ae, ao = b.zeros(n * k // 2, np.uint8), b.zeros(n * 2, np.float16), b.zeros(m * k // 2, np.int8), b.zeros(m * k // 2, np.int8)
        asc, asu, bias, res, y = b.zeros(m * 2), b.zeros(m * 2, np.int32), b.zeros(n), b.zeros(m * n), b.zeros(m * n)
        ok = [wq, ws, ae, ao, asc, asu, bias, res, y, m, n, k, n, n, 0, 0]
        rt.launch("linear_w4a8_k", 1, 1, ok)
        for at, bad in ((0, wq + 8), (0, wq + 16), (0, 0), (1, ws + 1), (1, ws + 2), (2, ae + 4), (2, ae + 16), (3, ao + 16), (4, asc + 4), (5, asu + 4),
                        (6, bias + 4), (7, res + 4), (8, y + 4), (9, -1), (9, m + 1), (10, 0), (10, n + 1), (11, 0), (11, 64), (11, 384), (12, n - 1),
                        (12, 2 * n), (13, n - 1), (13, 2 * n), (14, 5), (14, -1), (15, 1), (15, 2)):
            with pytest.raises(RuntimeError, match="rejected"):
                rt.launch("linear_w4a8_k", 1, 1, ok[:at] + [bad] + ok[at + 1:])
        both = b.zeros(2 * m * n)                          # a residual that overlaps y without being y
        for r, ldr in ((both + 64, n), (both, n + 1), (both + 4 * (m * n - 1), n)):
            with pytest.raises(RuntimeError, match="overlap"):
                rt.launch("linear_w4a8_k", 1, 1, ok[:7] + [r, both] + ok[9:13] + [ldr, 0, 0])
        rt.launch("linear_w4a8_k", 1, 1, ok[:7] + [both + 4 * m * n, both] + ok[9:])
        off, rows = b.zeros(3, np.int32), b.zeros(4, np.int32)
        w2, s2 = b.zeros(2 * n * k // 2, np.uint8), b.zeros(2 * n * 2, np.float16)
        out = b.zeros(4 * n)
        ok = [w2, s2, ae, ao, asc, asu, 0, rows, off, out, 2, 4, m, n, k, n, 0, 0]
        rt.launch("moe_linear_w4a8_k", 1, 1, ok)
        for at, bad in ((0, wq), (1, ws), (6, bias), (7, 0), (7, rows + 4), (8, off + 4), (8, 0), (9, out + 4), (10, 0), (10, 3), (10, 1025), (11, 5),
                        (11, -1), (12, 0), (12, m + 1), (13, n + 1), (15, n - 1), (16, 9), (17, 3), (17, 1)):
            with pytest.raises(RuntimeError, match="rejected"):
                rt.launch("moe_linear_w4a8_k", 1, 1, ok[:at] + [bad] + ok[at + 1:])
        rt.sync()


@pytest.mark.parametrize("rows", [4, 260])
def test_block_keeps_one_token_s_infinity_from_the_others(rt, rows):
    """Token 0, which has the first slot of the buckets, overflows in the down product (values of 1e18 through weights of
    60000; a quantiser in front of an infinity gives zeros); the others have choices without an expert."""
    rng = np.random.default_rng(rows)
    n_exp, dim, ffn = 5, 256, 128
    x = rng.standard_normal((rows, dim)).astype(np.float32)
    logits = rng.standard_normal((rows, n_exp)).astype(np.float32)
    logits[0] = [9, 8, 0, 0, 0]
    logits[1:, 1:] = -np.inf                               # one expert for two choices
    wg, sg, _ = P.layer(rng, n_exp, 2 * ffn, dim)
    wd, sd, _ = P.layer(rng, n_exp, dim, ffn)
    with Bufs(rt) as b:
        gate = ExpertLinear(rt, n_exp, ffn, dim, b.put(wg), b.put(sg), act="silu", gated=True)
        down = ExpertLinear(rt, n_exp, dim, ffn, b.put(wd), b.put(np.full_like(sd, 60000)))
        block = MoEMLP(rt, MoERouter(rt, n_exp, 2), gate, down)
        want = block.forward(x, logits)
        x[0] *= 1e18
        got = block.forward(x, logits)
    assert np.all(np.isfinite(want)) and not np.all(np.isfinite(got[0]))
    assert np.array_equal(got[1:], want[1:])


@pytest.mark.parametrize("rows,n,k", [(16, 40, 256), (5, 100, 1152), (16, 700, 1024), (3000, 300, 1152)])
@pytest.mark.parametrize("gated", [False, True])
def test_experts_slot_without_a_row_of_x(rt, rows, n, k, gated):
    """A row index outside of x stands for a row of zeros, with few rows and on tiles."""
    rng = np.random.default_rng(rows + n)
    wq, ws, w = P.layer(rng, 2, n * (2 if gated else 1), k)
    cd, q = P.codes(rng, rows, k)
    bias = rng.standard_normal((2, w.shape[1])).astype(np.float32)
    bucket = rng.integers(0, rows, rows).astype(np.int32)
    for i, bad in enumerate((-1, rows, 2 ** 31 - 1, -2 ** 31)):
        bucket[i::5] = bad
    offsets = np.array([0, rows // 3, rows], np.int32)
    with Bufs(rt) as b:
        lin = ExpertLinear(rt, 2, n, k, b.put(wq), b.put(ws), bias=bias, act="silu", gated=gated)
        plan = MoEPlan(rows=rows, topk=1, n_exp=2, ids=0, weights=0, bucket_rows=b.put(bucket), base=0, offsets=b.put(offsets))
        out = b.zeros(rows * n, np.float32, -777.0)
        lin.forward_codes_device([b.put(c) for c in cd], plan, out_dev=out)
        got = b.get(out, rows * n).reshape(rows, n)
        assert rt.gemm_status() == 0
        lin.ws.free()
    known = (bucket >= 0) & (bucket < rows)
    at = np.where(known, bucket, 0)
    q, asc = np.where(known[:, None], q[at], 0), np.where(known[:, None], cd[2][at], 0).astype(np.float32)
    for e in range(2):
        lo, hi = offsets[e], offsets[e + 1]
        want, bound = P.epilogue(*P.product(w[e], ws[e], q[lo:hi], asc[lo:hi]), "silu", gated, bias[e], None)
        _within(got[lo:hi], want, bound)


@pytest.mark.parametrize("m", [3, 3000])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_activations_in_their_tails(rt, m, act):
    """Codes of zero leave the bias, here from -30 to 30, as the activation's argument v.
    2^-20 |v| everywhere: the erf formula is within 1.5e-7, the roundings of its reciprocal (times a slope of 3.5 at most),
    five steps and exp within 1.3e-6, half of both times |v|; the logistic forms have a reciprocal, an exp whose argument's
    error is damped by s (1 - s) |t| < 1/4, and three products.
    Left of 0 the result is a small number of its own: v / 2 times erfc, whose formula is within 3.9 % of it up to
    |v| = 13.3 (compared in 64 bits), or v / (1 + exp(t)) with t within 2^-21 of its value, t <= 88.  Behind that
    it is below 2^-126 |v|, where the reciprocal and exp give 0."""
    from scipy.special import erfc
    n, k = 600, 1152
    v = np.linspace(-30, 30, n).astype(np.float32)
    wq, ws, _ = P.layer(np.random.default_rng(1), 1, n, k)
    zero = np.zeros((m, k // 2), np.int8)
    with Bufs(rt) as b:
        lin = FusedLinear(rt, n, k, b.put(wq), b.put(ws), bias=v, act=act)
        out = b.zeros(m * n)
        lin.forward_codes_device([b.put(zero), b.put(zero), b.zeros(m * k // 128), b.zeros(m * k // 128, np.int32)], m, out_dev=out)
        got = b.get(out, m * n).reshape(m, n)
        lin.ws.free()
    x = v.astype(np.float64)
    with np.errstate(over="ignore"):
        want = {"gelu": x / 2 * erfc(-x / np.sqrt(2)), "silu": x / (1 + np.exp(-x)),
                "gelu_tanh": x / (1 + np.exp(-2 * np.sqrt(2 / np.pi) * (x + 0.044715 * x ** 3)))}[act]
    assert np.all(np.abs(got - want) <= 2.0 ** -20 * np.abs(v))
    left = v < 0
    assert np.all(np.abs(got - want)[:, left] <= (0.05 * np.abs(want) + 2.0 ** -125 * np.abs(v))[left])
    assert np.all(got == got[0])


def test_block_in_a_graph_outlives_a_larger_call(rt):
    """A graph of few rows is replayed after a call of many, for which every buffer of the block grew."""
    rng = np.random.default_rng(7)
    dim, few, many = 256, 5, 700
    with Bufs(rt) as b:
        block = _block(rt, b, rng, 5, 2, dim, 128)
        px, pl, py = b.zeros(few * dim), b.zeros(few * 5), b.zeros(few * dim)
        block.forward_device(px, pl, few, out_dev=py, sync=True)
        rt.graph_begin()
        block.forward_device(px, pl, few, out_dev=py)
        graph = rt.graph_end()
        for _ in range(2):
            x, logits = rng.standard_normal((few, dim)).astype(np.float32), rng.standard_normal((few, 5)).astype(np.float32)
            want = block.forward(x, logits)
            block.forward(rng.standard_normal((many, dim)).astype(np.float32), rng.standard_normal((many, 5)).astype(np.float32))
            many *= 2
            rt.upload(px, x)
            rt.upload(pl, logits)
            rt.graph_launch(graph)
            assert np.array_equal(b.get(py, few * dim).reshape(few, dim), want)
        rt.graph_free(graph)


@pytest.mark.parametrize("rows", [6, 40])
def test_block_in_a_batch_scope(rt, rows):
    """Two blocks behind each other, and a layer on their output: the quantisers between the recorded launches take their
    turn."""
    rng = np.random.default_rng(rows)
    dim = 256
    x, logits = rng.standard_normal((rows, dim)).astype(np.float32), rng.standard_normal((rows, 5)).astype(np.float32)
    with Bufs(rt) as b:
        block = _block(rt, b, rng, 5, 2, dim, 128)
        wq, ws, _ = P.layer(rng, 1, dim, dim)
        lin = FusedLinear(rt, dim, dim, b.put(wq), b.put(ws), act="gelu")
        px, pl, pa, pb, pc = b.put(x), b.put(logits), b.zeros(rows * dim), b.zeros(rows * dim), b.zeros(rows * dim)

        def run():
            block.forward_device(px, pl, rows, out_dev=pa)
            block.forward_device(pa, pl, rows, out_dev=pb)
            return lin.forward_device(pb, rows, out_dev=pc)

        run()
        want = b.get(pc, rows * dim)
        for p in (pa, pb, pc):
            rt.memset(p, 0, rows * dim * 4)
        with rt.batch():
            run()
        assert np.any(want) and np.array_equal(b.get(pc, rows * dim), want)
