"""GPU tier: moe_route_k and moe_plan_k against the plain 64-bit forms — whole numbers equal, weights within fp32's
error — and the calls that they refuse."""
from __future__ import annotations

import numpy as np
import pytest

import moe_plain as P
from gpu_util import Bufs
from k100lc_kernels import MoERouter, Workspace

pytestmark = pytest.mark.gpu


def _rounded(x, dtype):
    """(bits for the device, the values they stand for)"""
    if dtype == "f32":
        return x.astype(np.float32), x.astype(np.float32)
    if dtype == "f16":
        return x.astype(np.float16), x.astype(np.float16).astype(np.float32)
    bits = (x.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)
    return bits, (bits.astype(np.uint32) << 16).view(np.float32)


def _run(rt, x, dtype="f32", **kw):
    rows, n_exp = x.shape
    bits, values = _rounded(x, dtype)
    topk = kw["topk"]
    with Workspace(rt) as ws:
        router = MoERouter(rt, n_exp, dtype=dtype, ws=ws, **kw)
        plan = router.forward_device(ws.upload("x", bits) if rows else 0, rows, sync=True)
        get = lambda p, n, t: rt.download(p, n, t)  # noqa: E731
        got = dict(ids=get(plan.ids, rows * topk, np.int32).reshape(rows, topk), w=get(plan.weights, rows * topk, np.float32).reshape(rows, topk),
                   bucket=get(plan.bucket_rows, rows * topk, np.int32), base=get(plan.base, rows * topk, np.int32).reshape(rows, topk),
                   offsets=get(plan.offsets, n_exp + 1, np.int32))
    return got, values


def _check(got, values, **kw):
    ids, w = P.route(values, **kw)
    assert np.array_equal(got["ids"], ids)
    assert np.all(np.abs(got["w"] - w) <= P.ROUTE_REL * np.abs(w) + 2.0 ** -126)
    bucket, base, _w, offsets = P.plan(got["ids"], got["w"], values.shape[1])
    assert np.array_equal(got["offsets"], offsets) and np.array_equal(got["base"], base)
    assert np.array_equal(got["bucket"][: bucket.size], bucket)


@pytest.mark.parametrize("rows,n_exp,topk", [(1, 1, 1), (1, 8, 2), (3, 33, 5), (7, 60, 4), (64, 128, 8), (5, 1024, 32), (257, 513, 3),
                                             (1000, 256, 8), (4099, 64, 6)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_route_sizes(rt, rows, n_exp, topk, score, biased):
    rng = np.random.default_rng(rows * 1000 + n_exp)
    x = (rng.standard_normal((rows, n_exp)) * 2).astype(np.float32)
    kw = dict(topk=topk, score=score, bias=(rng.standard_normal(n_exp) * 0.1).astype(np.float32) if biased else None)
    got, values = _run(rt, x, **kw)
    _check(got, values, **kw)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n_exp,n_group,topk_group,group_top", [(256, 8, 4, 2), (60, 4, 2, 1), (36, 12, 5, 2), (32, 32, 8, 2), (1024, 2, 1, 2), (40, 1, 1, 1)])
@pytest.mark.parametrize("biased", [False, True])
def test_route_groups_and_types(rt, dtype, n_exp, n_group, topk_group, group_top, biased):
    rng = np.random.default_rng(n_exp + n_group)
    x = rng.standard_normal((301, n_exp)) * 1.5
    kw = dict(topk=min(8, n_exp // n_group * topk_group), score="sigmoid", n_group=n_group, topk_group=topk_group, group_top=group_top,
              bias=(rng.standard_normal(n_exp) * 0.05).astype(np.float32) if biased else None, scale=2.5)
    got, values = _run(rt, x, dtype, **kw)
    _check(got, values, **kw)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
def test_route_masks_ties_and_infinities(rt, score, renorm):
    inf, nan = np.inf, np.nan
    x = np.zeros((9, 40), np.float32)
    x[0] = -inf                                            # nothing to choose
    x[1] = nan
    x[2, 3:] = -inf                                        # three candidates for five choices
    x[3] = np.finfo(np.float32).min                        # the type's lowest value is a number
    x[4, 5], x[4, 6] = inf, inf
    x[5, ::2] = -0.0                                       # -0 and +0 tie
    x[6] = np.arange(40) % 7
    x[7, 11] = nan
    x[8, 39] = 30
    if score == "sigmoid":
        x[3] = -80
    for bias in (None, np.zeros(40, np.float32), np.where(np.arange(40) == 0, -inf, 0).astype(np.float32)):
        kw = dict(topk=5, score=score, renorm=renorm, bias=bias)
        got, values = _run(rt, x, **kw)
        _check(got, values, **kw)


def test_route_resolves_keys_that_fp32_cannot(rt):
    """Logits one step apart and large biases: many keys agree in 32 bits and differ in 64."""
    rng = np.random.default_rng(5)
    step = np.float32(1.0)
    row = []
    for _ in range(64):
        row.append(step)
        step = np.nextafter(step, np.float32(2))
    x = np.stack([rng.permutation(np.array(row, np.float32)) for _ in range(200)])
    for score in ("softmax", "sigmoid"):
        for b in (np.zeros(64), np.full(64, 3.0), np.where(np.arange(64) < 32, 100.0, 100.0 + 2.0 ** -17)):
            kw = dict(topk=8, score=score, bias=b.astype(np.float32))
            got, values = _run(rt, x, **kw)
            _check(got, values, **kw)
            kw |= dict(n_group=8, topk_group=3, group_top=2)
            got, values = _run(rt, x, **kw)
            _check(got, values, **kw)


@pytest.mark.parametrize("rows", [5, 128, 129, 600])
@pytest.mark.parametrize("n_exp", [16, 300])
def test_route_alone_is_route_with_plan(rt, rows, n_exp):
    """moe_route_k, then moe_plan_k: what the one call gives on either side of its choice of one launch or two."""
    x = np.random.default_rng(rows).standard_normal((rows, n_exp)).astype(np.float32)
    got, values = _run(rt, x, topk=8, score="sigmoid")
    _check(got, values, topk=8, score="sigmoid")
    with Bufs(rt) as b:
        ids, w, slot, base, off = b.zeros(rows * 8, np.int32), b.zeros(rows * 8), b.zeros(rows * 8, np.int32), b.zeros(rows * 8, np.int32), b.zeros(n_exp + 1, np.int32)
        rt.launch("moe_route_k", 1, 1, [b.put(x), 0, ids, w, rows, n_exp, 8, 1, 1, 1, 1, 1, 1.0, 0])
        rt.launch("moe_plan_k", 1, 1, [ids, w, slot, base, off, rows, n_exp, 8])
        assert np.array_equal(b.get(ids, rows * 8, np.int32), got["ids"].reshape(-1)) and np.array_equal(b.get(w, rows * 8), got["w"].reshape(-1))
        assert np.array_equal(b.get(slot, rows * 8, np.int32), got["bucket"]) and np.array_equal(b.get(base, rows * 8, np.int32), got["base"].reshape(-1))
        assert np.array_equal(b.get(off, n_exp + 1, np.int32), got["offsets"])


def test_routes_back_to_back(rt):
    """Routers of both kinds in turn, without a wait between them: they share the engine's workspace and a counter."""
    rng = np.random.default_rng(9)
    xs = [rng.standard_normal((r, 24)).astype(np.float32) for r in (1, 700, 40, 1999, 3, 512)]
    with Workspace(rt) as ws:
        routers = [MoERouter(rt, 24, 2, ws=ws, tag=f"r{i}") for i in range(len(xs))]
        px = [ws.upload(f"x{i}", x) for i, x in enumerate(xs)]
        for _ in range(20):
            plans = [r.forward_device(p, x.shape[0]) for r, p, x in zip(routers, px, xs)]
        rt.sync()
        for plan, x in zip(plans, xs):
            n = x.shape[0] * 2
            got = dict(ids=rt.download(plan.ids, n, np.int32).reshape(-1, 2), w=rt.download(plan.weights, n, np.float32).reshape(-1, 2),
                       bucket=rt.download(plan.bucket_rows, n, np.int32), base=rt.download(plan.base, n, np.int32).reshape(-1, 2),
                       offsets=rt.download(plan.offsets, 25, np.int32))
            _check(got, x, topk=2)


def test_route_no_rows(rt):
    got, _ = _run(rt, np.zeros((0, 8), np.float32), topk=2)
    assert np.array_equal(got["offsets"], np.zeros(9, np.int32))


@pytest.mark.parametrize("rows,n_exp,topk", [(1, 1, 1), (1, 1024, 32), (33, 5, 3), (2048, 8, 1), (2049, 8, 1), (5000, 300, 7), (40000, 64, 8)])
def test_plan_of_given_pairs(rt, rows, n_exp, topk):
    """Ids out of range, repeated experts and zero weights; slots behind the last bucket stay as they were."""
    rng = np.random.default_rng(rows)
    ids = rng.integers(-2, n_exp + 2, size=(rows, topk)).astype(np.int32)
    w = rng.random((rows, topk)).astype(np.float32)
    w[rng.random((rows, topk)) < 0.1] = 0
    with Bufs(rt) as b:
        pw, pr, pb, po = b.put(w), b.zeros(rows * topk, np.int32, -7), b.zeros(rows * topk, np.int32, -7), b.zeros(n_exp + 1, np.int32, -7)
        rt.launch("moe_plan_k", 1, 1, [b.put(ids), pw, pr, pb, po, rows, n_exp, topk])
        got = [b.get(pr, rows * topk, np.int32), b.get(pb, rows * topk, np.int32).reshape(rows, topk), b.get(pw, rows * topk).reshape(rows, topk),
               b.get(po, n_exp + 1, np.int32)]
    bucket, base, wz, offsets = P.plan(ids, w, n_exp)
    assert np.array_equal(got[0][: bucket.size], bucket) and np.all(got[0][bucket.size:] == -7)
    assert np.array_equal(got[1], base) and np.array_equal(got[2], wz) and np.array_equal(got[3], offsets)


def test_route_and_plan_refuse(rt):
    with Bufs(rt) as b:
        x, ids, w = b.zeros(64), b.zeros(16, np.int32), b.zeros(16)
        ok = [x, 0, ids, w, 8, 8, 2, 1, 1, 1, 0, 1, 1.0, 0]
        rt.launch("moe_route_k", 1, 1, ok)
        for at, bad in ((4, -1), (4, 9), (5, 0), (5, 1025), (5, 9), (6, 0), (6, 9), (7, 3), (8, 2), (9, 0), (10, 2), (11, 2), (13, 3), (0, x + 2),
                        (0, x + 4), (1, x + 240), (2, ids + 4), (3, w + 4), (0, 0)):
            with pytest.raises(RuntimeError, match="rejected"):
                rt.launch("moe_route_k", 1, 1, ok[:at] + [bad] + ok[at + 1:])
        bucket, base, off = b.zeros(16, np.int32), b.zeros(16, np.int32), b.zeros(9, np.int32)
        both = ok[:4] + [bucket, base, off] + ok[4:]
        rt.launch("moe_route_plan_k", 1, 1, both)
        for at, bad in ((7, -1), (7, 9), (8, 0), (8, 1025), (8, 9), (9, 0), (9, 9), (10, 3), (11, 2), (12, 0), (13, 2), (14, 2), (16, 3), (0, x + 2),
                        (0, x + 4), (1, x + 240), (2, ids + 4), (3, w + 4), (4, bucket + 4), (4, 0), (5, base + 2), (6, off + 4)):
            with pytest.raises(RuntimeError, match="rejected"):
                rt.launch("moe_route_plan_k", 1, 1, both[:at] + [bad] + both[at + 1:])
        ok = [ids, w, bucket, base, off, 8, 8, 2]
        rt.launch("moe_plan_k", 1, 1, ok)
        for at, bad in ((5, -1), (5, 9), (6, 0), (6, 9), (6, 1025), (7, 0), (7, 33), (0, ids + 4), (1, 0), (2, bucket + 4), (3, base + 2), (4, off + 4)):
            with pytest.raises(RuntimeError, match="rejected"):
                rt.launch("moe_plan_k", 1, 1, ok[:at] + [bad] + ok[at + 1:])
        rt.sync()


def _tie_at_the_cut(rng, rows, n_exp, topk, kind):
    """topk - 1 clear winners, `ties` equal inputs at the cut, and larger keys that fp32 does not tell from them, all at
    random places -> logits, bias"""
    x, bias = np.full((rows, n_exp), -5.0), None
    if kind != "logits":
        # the bias belongs to the expert: one order of the experts for all rows, the places of ties and larger keys differ
        bias = np.full(n_exp, -1.0, np.float32)
    order = rng.permutation(n_exp)
    for r in range(rows):
        winners, rest = order[: topk - 1], rng.permutation(order[topk - 1: topk + 15])
        ties, more = rest[: 2 + r % 3], rest[4: 5 + r % 2]
        if kind == "logits":
            x[r, winners] = 2 + np.arange(topk - 1)
            x[r, ties], x[r, more] = 1.0, np.nextafter(np.float32(1), np.float32(2))
            continue
        bias[winners], bias[order[topk - 1: topk + 15]] = 2 + np.arange(topk - 1), 0.25
        x[r, winners], x[r, ties], x[r, more] = 5.0, *((20.0, 21.0) if kind == "sigmoid" else (-12.0, -11.0))
    return x, bias


@pytest.mark.parametrize("kind,dtype", [("logits", "f32"), ("sigmoid", "f32"), ("sigmoid", "bf16"), ("sigmoid", "f16"), ("softmax", "f32"), ("softmax", "bf16")])
@pytest.mark.parametrize("topk", [1, 2, 8, 31])
def test_route_larger_key_behind_a_tie_at_the_cut(rt, kind, dtype, topk):
    rng = np.random.default_rng(topk)
    for n_exp in (64, 256, 1000):
        x, bias = _tie_at_the_cut(rng, 48, n_exp, topk, kind)
        kw = dict(topk=topk, score="sigmoid" if kind == "sigmoid" else "softmax", bias=bias)
        got, values = _run(rt, x, dtype, **kw)
        _check(got, values, **kw)
        # the same for one token, whose plan is made by the launch that routes
        got, values = _run(rt, x[:1], dtype, **kw)
        _check(got, values, **kw)


def test_route_by_hand_behind_a_tie_at_the_cut(rt):
    x = np.full((1, 256), -5, np.float32)
    x[0, 0] = x[0, 8] = 1
    x[0, 16] = np.nextafter(np.float32(1), np.float32(2))
    assert _run(rt, x, topk=1)[0]["ids"].tolist() == [[16]]
    x[0, 0] = x[0, 8] = 20
    x[0, 16] = 21
    assert _run(rt, x, topk=1, score="sigmoid", bias=np.zeros(256, np.float32))[0]["ids"].tolist() == [[16]]


@pytest.mark.parametrize("n_exp,groups", [(32, 1), (60, 4), (256, 1), (256, 8)])
@pytest.mark.parametrize("score,biased", [("softmax", False), ("softmax", True), ("sigmoid", True)])
def test_route_of_few_levels(rt, n_exp, groups, score, biased):
    """Logits of four levels, each moved by 0..2 steps of fp32: equal inputs and neighbours everywhere, at the cut too."""
    rng = np.random.default_rng(n_exp + groups)
    base = rng.integers(0, 4, size=(400, n_exp)) * 0.5 + 0.5
    x = (base * (1 + rng.integers(0, 3, size=base.shape) * 2.0 ** -23)).astype(np.float32)
    bias = np.full(n_exp, 0.5, np.float32) if biased else None
    for topk in (1, 3, 8):
        kw = dict(topk=topk, score=score, bias=bias, n_group=groups, topk_group=max(1, groups // 2), group_top=2 if groups > 1 else 1)
        got, values = _run(rt, x, **kw)
        _check(got, values, **kw)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_route_weights_of_scores_that_underflow(rt, dtype):
    """Chosen scores below fp32's range have an ordinary quotient.  (The logits differ by less than 64, so their difference
    rounds by 2^-19 at most, which the weights' tolerance holds twice over.)"""
    x = np.full((8, 16), -np.inf)
    for r, v in enumerate(((-90, -91), (-100, -104), (-200, -201, -202.5), (-600, -600), (-16, -60), (-60, -90, -100), (-3, -63), (-63.5, -64.5, -88, -120))):
        x[r, 3: 3 + len(v)] = v
    kw = dict(topk=4, score="sigmoid", scale=2.5)
    got, values = _run(rt, x, dtype, **kw)
    _check(got, values, **kw)
    assert np.allclose(got["w"][0, :2], [2.5 * 0.7310586, 2.5 * 0.2689414], rtol=1e-6)
    # softmax: the bias takes the largest logit out of the choice
    x = np.random.default_rng(1).standard_normal((40, 16)) * 3
    x[:, 5] = np.linspace(60, 300, 40)
    bias = np.linspace(0, 1, 16).astype(np.float32)
    bias[5] = -np.inf
    kw = dict(topk=4, bias=bias)
    got, values = _run(rt, x, dtype, **kw)
    _check(got, values, **kw)
    # and so do the groups: one large expert alone against two of its size less something
    x = np.random.default_rng(2).standard_normal((40, 16))
    x[:, 0], x[:, 1:4] = 300, -np.inf
    kw = dict(topk=2, n_group=4, topk_group=1, group_top=2, bias=np.where(np.arange(16) < 4, -2.0, 0).astype(np.float32))
    got, values = _run(rt, x, dtype, **kw)
    _check(got, values, **kw)


def test_route_weights_at_the_type_s_lowest_value(rt):
    """Equal scores have equal weights, however small; an infinite logit that the bias excludes leaves nothing to the others."""
    x = np.full((2, 40), np.finfo(np.float32).min, np.float32)
    x[1, 7] = 1.5
    for score in ("softmax", "sigmoid"):
        got, _ = _run(rt, x, topk=5, score=score)
        assert got["ids"].tolist() == [[0, 1, 2, 3, 4], [7, 0, 1, 2, 3]]
        assert np.allclose(got["w"], [[0.2] * 5, [1, 0, 0, 0, 0]], rtol=1e-6, atol=0)
        assert got["offsets"][40] == 6
    x = np.zeros((1, 8), np.float32)
    x[0, 2] = np.inf
    got, _ = _run(rt, x, topk=2, bias=np.where(np.arange(8) == 2, -5, 0).astype(np.float32))
    assert got["ids"].tolist() == [[0, 1]] and not got["w"].any()


def test_route_sigmoid_weights_below_the_normal_numbers(rt):
    """Without renormalisation the weight is the score itself, a subnormal number between logits of -87 and -103: within two
    steps of 2^-149 of its value, and a pair with a slot."""
    x = np.array([[-80, -87, -88, -89, -95, -100, -102, -110]], np.float32)
    got, _ = _run(rt, x, topk=8, score="sigmoid", renorm=False)
    want = 1 / (1 + np.exp(-x.astype(np.float64)))
    assert got["ids"].tolist() == [[0, 1, 2, 3, 4, 5, 6, 7]]
    assert np.all(np.abs(got["w"] - want) <= P.ROUTE_REL * want + 3 * 2.0 ** -149)
    assert got["offsets"][8] == 7                          # the score at -110 is 0 in fp32
