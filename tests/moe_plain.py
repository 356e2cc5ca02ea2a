"""Plain NumPy forms in 64 bits of the routing, its plan and the W4A8 products with an epilogue, and how far fp32
kernels may be from them."""
from __future__ import annotations

import numpy as np
from scipy.special import erf

EPS = 2.0 ** -24                        # half a step of fp32, relative


# ------------------------------------------------------------------------------------------------------ routing
def scores(logits, score):
    x = np.where(np.isnan(logits), -np.inf, logits).astype(np.float64)
    if score == "sigmoid":
        with np.errstate(over="ignore"):
            return 1 / (1 + np.exp(-x))
    m = x.max(-1, keepdims=True)
    with np.errstate(invalid="ignore"):
        e = np.where(x == m, 1.0, np.exp(x - m))
    e = np.where(np.isneginf(x), 0.0, e)
    z = e.sum(-1, keepdims=True)
    return e / np.where(z == 0, 1, z)


def route(logits, topk, score="softmax", bias=None, n_group=1, topk_group=1, group_top=1, renorm=True, scale=1.0):
    x = np.where(np.isnan(logits), -np.inf, logits).astype(np.float64)
    rows, n_exp = x.shape
    s = scores(logits, score)
    worth_of = s if bias is None else s + bias.astype(np.float64)
    key = x if bias is None else worth_of
    dead = np.isneginf(x) | np.isneginf(key) | np.isnan(key)
    key = np.where(dead, -np.inf, key)
    if n_group > 1:
        v = (key if bias is None and group_top == 1 else np.where(dead, -np.inf, worth_of)).reshape(rows, n_group, -1)
        best = -np.sort(-v, -1)[..., :group_top]
        worth = best[..., 0]
        if group_top == 2 and v.shape[-1] > 1:
            worth = worth + np.where(np.isneginf(best[..., 1]), 0.0, best[..., 1])
        keep = np.argsort(-worth, -1, kind="stable")[:, :topk_group]
        mask = np.zeros((rows, n_group), bool)
        np.put_along_axis(mask, keep, True, 1)
        key = np.where(np.repeat(mask, n_exp // n_group, 1), key, -np.inf)
    ids = np.argsort(-key, -1, kind="stable")[:, :topk]
    none = np.isneginf(np.take_along_axis(key, ids, 1))
    w = np.where(none, 0.0, np.take_along_axis(s, ids, 1))
    if renorm:
        t = w.sum(-1, keepdims=True)
        w = np.where(t > 0, w / np.where(t > 0, t, 1), 0.0)
    return np.where(none, -1, ids).astype(np.int32), w * scale


# exp is within 2^-22 of its value and its argument |x| <= 32 moves it by 32 * 2^-24; a softmax sum of up to 1024 terms
# adds 37 roundings, renormalising another 6 and the divisions and products 4: (4 + 32 + 37 + 6 + 4) * 2^-24 < 2^-17.6,
# twice that because a sum errs with its terms
ROUTE_REL = 2.0 ** -16


def plan(ids, weights, n_exp):
    rows, topk = ids.shape
    w = np.array(weights, np.float32)
    ok = (ids >= 0) & (ids < n_exp) & (w != 0)
    w[~ok] = 0
    pair = np.flatnonzero(ok.reshape(-1))
    order = pair[np.argsort(ids.reshape(-1)[pair], kind="stable")]
    offsets = np.concatenate([[0], np.cumsum(np.bincount(ids.reshape(-1)[pair], minlength=n_exp))]).astype(np.int32)
    base = np.zeros(rows * topk, np.int32)
    base[order] = np.arange(order.size)
    return (order // topk).astype(np.int32), base.reshape(rows, topk), w, offsets


# ----------------------------------------------------------------------------------------------------- products
def layer(rng, stack, n, k):
    """-> (wq bytes [stack, n, k/2], f16 scales, the int8 weights they stand for)"""
    w = rng.integers(-8, 8, size=(stack, n, k), dtype=np.int8)
    wq = ((w[..., 0::2] & 15) | ((w[..., 1::2] & 15) << 4)).astype(np.uint8)
    ws = (np.abs(rng.standard_normal((stack, n, k // 128))) * 0.01 + 1e-3).astype(np.float16)
    return wq, ws, w


def codes(rng, rows, k):
    """Activation codes of random rows, extremes among them: (ae, ao, asc, asu), q"""
    q = rng.integers(-127, 128, size=(rows, k)).astype(np.int8)
    if rows:
        q[0, : min(k, 256)] = 127
        q[-1, : min(k, 128)] = -128
    asc = (np.abs(rng.standard_normal((rows, k // 128))) * 0.02 + 1e-3).astype(np.float32)
    asu = q.reshape(rows, k // 128, 128).astype(np.int32).sum(-1).astype(np.int32)
    return (np.ascontiguousarray(q[:, 0::2]), np.ascontiguousarray(q[:, 1::2]), asc, asu), q


def act(name, v):
    with np.errstate(over="ignore"):
        return {"none": lambda: v, "relu": lambda: np.maximum(v, 0), "silu": lambda: v / (1 + np.exp(-v)),
                "gelu": lambda: 0.5 * v * (1 + erf(v / np.sqrt(2))),
                "gelu_tanh": lambda: 0.5 * v * (1 + np.tanh(np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)))}[name]()


def product(w, ws, q, asc):
    """-> (v, error bound of an fp32 sum over the groups): v[m, n] = sum_g ws * asc * I"""
    n, k = w.shape
    g = k // 128
    integers = np.einsum("mgk,ngk->mng", q.reshape(-1, g, 128).astype(np.float64), w.reshape(n, g, 128).astype(np.float64))
    term = integers * ws.astype(np.float64)[None] * asc.astype(np.float64)[:, None]
    # the scale product rounds once, the fused multiply-adds and the joining of partial sums once per group at most
    return term.sum(-1), (g + 2) * EPS * np.abs(term).sum(-1)


def epilogue(v, err, name, gated, bias, residual):
    """-> (y, bound).  Each activation's slope is below 1.13; its own evaluation (an exp or erfc within 2^-20 of its
    value with the argument's error, a division, products) stays within 2^-18 of |v| for |v| < 64."""
    if bias is not None:
        v = v + bias.astype(np.float64)
        err = err + EPS * np.abs(v)
    n = v.shape[1] // 2 if gated else v.shape[1]

    def acted(u, e):
        return act(name, u), 1.13 * e + (0 if name in ("none", "relu") else 2.0 ** -18 * np.abs(u))

    if gated:
        a, ea = acted(v[:, :n], err[:, :n])
        up, eu = v[:, n:], err[:, n:]
        y, err = a * up, ea * np.abs(up) + np.abs(a) * eu + ea * eu + EPS * np.abs(a * up)
    else:
        y, err = acted(v, err)
    if residual is not None:
        y = y + residual.astype(np.float64)
    return y, 1.01 * err + 2 * EPS * np.abs(y) + 1e-30
