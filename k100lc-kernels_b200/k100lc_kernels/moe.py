"""Routing to experts and W4A8 products with an epilogue, on the device from the router's logits to the rows.

``FusedLinear``    y = act(x . W^T + bias) + residual, optionally gated (act(gate) * up from stacked gate and up rows);
``MoERouter``      logits -> ``MoEPlan``: every token's experts and weights, and the pairs sorted into buckets;
``ExpertLinear``   the product of ``FusedLinear`` for every expert's bucket of a plan;
``MoEMLP``         router, gated product, quantiser, down product and weighted combine without a host round trip.

The classes keep the contract of ``model.py``: weights are on the device already or uploaded once, intermediate
buffers come from a ``Workspace``, ``forward_device`` queues kernels on the engine's stream and returns device
pointers.  ``MoEExperts`` stays the form for routing decided on the host and experts of any layer class.
"""
from __future__ import annotations

import dataclasses

import numpy as np

from .model import Workspace, _as_rows
from .runtime import Runtime, _bits

__all__ = ["ACTIVATIONS", "FusedLinear", "MoEPlan", "MoERouter", "ExpertLinear", "MoEMLP"]

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
SCORES = {"softmax": 0, "sigmoid": 1}
LOGIT_TYPES = {"f32": 0, "bf16": 1, "f16": 2}
GROUP = 128


def _quantise(rt: Runtime, ws: Workspace, tag: str, x_dev: int, rows: int, k: int):
    """``quant_act`` over all rows -> (ae, ao, asc, asu); a launch covers at most 65535 rows."""
    half, ng4 = k // 2, (k // GROUP) * 4
    codes = [ws.buffer(f"{tag}.q{i}", rows * n) for i, n in enumerate((half, half, ng4, ng4))]
    for r in range(0, rows, 65535):
        m = min(65535, rows - r)
        rt.launch2d("quant_act", k // GROUP, m, 32, 1,
                    [int(x_dev) + r * k * 4] + [c + r * n for c, n in zip(codes, (half, half, ng4, ng4))] + [m, k])
    return tuple(codes)


class _Product:
    """What the dense and the per-expert product share: the shapes, the weights and the epilogue."""

    def __init__(self, rt: Runtime, n_exp: int, n: int, k: int, wq: int, ws_scale: int, bias, act: str, gated: bool,
                 ws: Workspace | None, tag: str | None, kind: str):
        if act not in ACTIVATIONS:
            raise ValueError(f"unknown activation {act!r}; built here: {sorted(ACTIVATIONS)}")
        if n < 1 or k < GROUP or k % GROUP:
            raise ValueError(f"N={n} must be positive and K={k} a positive multiple of {GROUP}")
        if n_exp < 1:
            raise ValueError(f"n_exp={n_exp} must be positive")
        self.rt, self.n_exp, self.n, self.k = rt, int(n_exp), int(n), int(k)
        self.act, self.gated, self.path = act, bool(gated), "w4a8"
        self.tag = tag or f"{kind}_{id(self):x}"
        self._own_ws = ws is None
        self.ws = ws or Workspace(rt)
        self.wq, self.ws_scale = int(wq), int(ws_scale)
        self.bias = 0
        if bias is not None and not isinstance(bias, (int, np.integer)):
            rows = self.n_exp * self.n * (2 if self.gated else 1)
            bias = np.ascontiguousarray(bias, dtype=np.float32)
            if bias.size != rows:
                raise ValueError(f"bias has {bias.size} values, the weights have {rows} rows")
            self.bias = self.ws.upload(self.tag + ".bias", bias)
        elif bias is not None:
            self.bias = int(bias)
        self._epilogue = (ACTIVATIONS[act], int(self.gated))


class FusedLinear(_Product):
    """W4A8 layer with its epilogue in the product: ``y = act(x . W^T + bias) + residual`` in one launch, any number
    of rows.  ``wq`` / ``ws_scale``: an RT4 layer on the device (``RT4Linear``'s pointers) of ``n`` rows, or with
    ``gated`` of ``2n`` rows, ``n`` gate rows before ``n`` up rows, for ``y = act(gate) * up + residual``.  ``bias``: an
    array (uploaded once) or a device pointer of one f32 per weight row.  ``act``: one of ``ACTIVATIONS``."""

    def __init__(self, rt: Runtime, n: int, k: int, wq: int, ws_scale: int, bias=None, act: str = "none",
                 gated: bool = False, ws: Workspace | None = None, tag: str | None = None):
        super().__init__(rt, 1, n, k, wq, ws_scale, bias, act, gated, ws, tag, "fused")

    def forward_codes_device(self, codes, rows: int, residual_dev: int | None = None, out_dev: int | None = None,
                             ldy: int | None = None, ldr: int | None = None, sync: bool = False) -> int:
        """``codes`` = (ae, ao, asc, asu) as ``quant_act`` / ``rmsnorm_quant_k`` leave them.  ``ldy`` / ``ldr``: values
        between the rows of the output / the residual (default: ``n``).  ``residual_dev`` may be ``out_dev``."""
        ldy, ldr = int(ldy or self.n), int(ldr or self.n)
        if rows < 0 or ldy < self.n or ldr < self.n:
            raise ValueError(f"rows={rows}, ldy={ldy}, ldr={ldr}: rows of {self.n} values")
        out = int(out_dev) if out_dev is not None else self.ws.buffer(self.tag + ".y", max(1, rows) * ldy * 4)
        ae, ao, asc, asu = codes
        self.rt.launch("linear_w4a8_k", 1, 1, [self.wq, self.ws_scale, ae, ao, asc, asu, self.bias, residual_dev or 0, out,
                                               rows, self.n, self.k, ldy, ldr, *self._epilogue])
        if sync:
            self.rt.sync()
        return out

    def forward_device(self, x_dev: int, rows: int, sync: bool = False, out_dev: int | None = None,
                       residual_dev: int | None = None) -> int:
        """f32 rows in: ``quant_act``, then the product."""
        codes = _quantise(self.rt, self.ws, self.tag, x_dev, rows, self.k) if rows else (0, 0, 0, 0)
        return self.forward_codes_device(codes, rows, residual_dev, out_dev, sync=sync)

    def forward(self, x: np.ndarray, residual: np.ndarray | None = None) -> np.ndarray:
        x = _as_rows(x)
        if x.shape[1] != self.k:
            raise ValueError(f"x has {x.shape[1]} columns, the layer K={self.k}")
        px = self.ws.upload(self.tag + ".x", x)
        pr = None
        if residual is not None:
            residual = _as_rows(residual)
            if residual.shape != (x.shape[0], self.n):
                raise ValueError(f"residual {residual.shape} does not match ({x.shape[0]}, {self.n})")
            pr = self.ws.upload(self.tag + ".r", residual)
        out = self.forward_device(px, x.shape[0], sync=True, residual_dev=pr)
        return self.rt.download(out, x.shape[0] * self.n, np.float32).reshape(x.shape[0], self.n)


@dataclasses.dataclass(frozen=True)
class MoEPlan:
    """Device pointers of a routing decision: ``ids`` / ``weights`` / ``base`` are ``[rows, topk]`` (i32, f32, i32),
    ``bucket_rows`` holds the token of every bucket slot (``rows * topk`` i32, used up to ``offsets[n_exp]``),
    ``offsets`` the ``n_exp + 1`` bucket bounds."""
    rows: int
    topk: int
    n_exp: int
    ids: int
    weights: int
    bucket_rows: int
    base: int
    offsets: int


class MoERouter:
    """Router logits ``[rows, n_exp]`` -> experts, weights and buckets.

    ``score``: "softmax" over the experts or "sigmoid" of each.  ``bias`` (one f32 per expert) is added to the scores
    for the choice only.  ``n_group`` > 1: only the experts of the ``topk_group`` best groups of neighbours are
    eligible, a group being worth its best expert (``group_top=1``) or its two best (2).  ``renorm`` divides the
    chosen scores by their sum; ``scale`` multiplies the result.  Equal keys go to the lowest index; an expert whose
    logit (or bias) is -inf or NaN is never chosen, and a choice without a candidate gets id -1 and weight 0.
    ``dtype``: type of the logits, "f32", "bf16" or "f16"."""

    def __init__(self, rt: Runtime, n_exp: int, topk: int, score: str = "softmax", bias=None, n_group: int = 1,
                 topk_group: int = 1, group_top: int = 1, renorm: bool = True, scale: float = 1.0, dtype: str = "f32",
                 ws: Workspace | None = None, tag: str | None = None):
        if score not in SCORES or dtype not in LOGIT_TYPES:
            raise ValueError(f"score={score!r} dtype={dtype!r}; built here: {sorted(SCORES)}, {sorted(LOGIT_TYPES)}")
        if not 1 <= n_exp <= 1024 or not 1 <= n_group <= 32 or n_exp % n_group:
            raise ValueError(f"n_exp={n_exp}: 1..1024 experts in 1..32 groups of one size (n_group={n_group})")
        if not 1 <= topk_group <= n_group or not 1 <= topk <= min(32, n_exp // n_group * topk_group):
            raise ValueError(f"topk={topk}, topk_group={topk_group}: at most 32 choices, of the experts of the kept groups")
        if group_top not in (1, 2):
            raise ValueError(f"group_top={group_top}: a group is worth its best expert (1) or its two best (2)")
        self.rt, self.n_exp, self.topk, self.dtype = rt, int(n_exp), int(topk), dtype
        self.tag = tag or f"router_{id(self):x}"
        self._own_ws = ws is None
        self.ws = ws or Workspace(rt)
        self.bias = 0
        if bias is not None:
            bias = np.ascontiguousarray(bias, dtype=np.float32)
            if bias.shape != (self.n_exp,):
                raise ValueError(f"bias {bias.shape} does not match the {self.n_exp} experts")
            self.bias = self.ws.upload(self.tag + ".bias", bias)
        self._key, self._last = self.tag + ".plan", None
        self._tail = (int(n_group), int(topk_group), int(group_top), SCORES[score], int(bool(renorm)), _bits(float(scale)),
                      LOGIT_TYPES[dtype])

    def forward_device(self, logits_dev: int, rows: int, sync: bool = False) -> MoEPlan:
        """Queues the routing; the plan's buffers belong to the router and hold until its next call."""
        if rows < 0:
            raise ValueError(f"rows={rows}")
        # plan and arguments of the last call are used again while the row count and the block of memory are the same
        if self._last is None or self._last[0] != rows or self.ws._bufs.get(self._key) is not self._last[1]:
            array = -(-max(1, rows * self.topk) * 4 // 256) * 256
            at = self.ws.buffer(self._key, 4 * array + (self.n_exp + 1) * 4)
            plan = MoEPlan(rows, self.topk, self.n_exp, ids=at, weights=at + array, bucket_rows=at + 2 * array, base=at + 3 * array,
                           offsets=at + 4 * array)
            self._last = (rows, self.ws._bufs[self._key], plan,
                          [0, self.bias, plan.ids, plan.weights, plan.bucket_rows, plan.base, plan.offsets, rows, self.n_exp,
                           self.topk, *self._tail])
        plan, argv = self._last[2:]
        argv[0] = int(logits_dev)
        self.rt.launch("moe_route_plan_k", 1, 1, argv)
        if sync:
            self.rt.sync()
        return plan

    def forward(self, logits: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
        """f32 logits on the host -> (ids, weights) as ``MoEExperts.forward`` takes them."""
        if self.dtype != "f32":
            raise ValueError("forward takes f32 logits; use forward_device for 16-bit ones")
        logits = _as_rows(logits)
        if logits.shape[1] != self.n_exp:
            raise ValueError(f"logits have {logits.shape[1]} columns, the router {self.n_exp} experts")
        plan = self.forward_device(self.ws.upload(self.tag + ".x", logits), logits.shape[0], sync=True)
        shape = (logits.shape[0], self.topk)
        return (self.rt.download(plan.ids, shape[0] * shape[1], np.int32).reshape(shape),
                self.rt.download(plan.weights, shape[0] * shape[1], np.float32).reshape(shape))


class ExpertLinear(_Product):
    """``FusedLinear`` for a stack of experts (``wq [n_exp, n or 2n, k/2]``, ``ws_scale``, ``bias`` likewise): every
    bucket of a plan runs through its expert's weights, one launch for all of them."""

    def __init__(self, rt: Runtime, n_exp: int, n: int, k: int, wq: int, ws_scale: int, bias=None, act: str = "none",
                 gated: bool = False, ws: Workspace | None = None, tag: str | None = None):
        super().__init__(rt, n_exp, n, k, wq, ws_scale, bias, act, gated, ws, tag, "experts")

    def forward_codes_device(self, codes, plan: MoEPlan, gather: bool = True, out_dev: int | None = None,
                             sync: bool = False) -> int:
        """-> ``[plan.rows * plan.topk, n]`` f32 in bucket order.  ``gather``: the codes are those of the tokens and a
        slot takes its token's row (a row index outside of them: a row of zeros); otherwise they are in bucket order
        already.  Rows behind the last bucket are left as they were."""
        if plan.n_exp != self.n_exp:
            raise ValueError(f"the plan is for {plan.n_exp} experts, the layer has {self.n_exp}")
        pairs = plan.rows * plan.topk
        out = int(out_dev) if out_dev is not None else self.ws.buffer(self.tag + ".y", max(1, pairs) * self.n * 4)
        ae, ao, asc, asu = codes
        self.rt.launch("moe_linear_w4a8_k", 1, 1,
                       [self.wq, self.ws_scale, ae, ao, asc, asu, self.bias, plan.bucket_rows if gather else 0, plan.offsets,
                        out, self.n_exp, pairs, plan.rows if gather else pairs, self.n, self.k, self.n, *self._epilogue])
        if sync:
            self.rt.sync()
        return out

    def forward_device(self, x_dev: int, plan: MoEPlan, gather: bool = True, out_dev: int | None = None, sync: bool = False) -> int:
        """f32 rows in: ``quant_act``, then the product.  (Rows in bucket order behind the last bucket are quantised
        as well, whatever they hold, and not used.)"""
        rows = plan.rows if gather else plan.rows * plan.topk
        codes = _quantise(self.rt, self.ws, self.tag, x_dev, rows, self.k) if rows else (0, 0, 0, 0)
        return self.forward_codes_device(codes, plan, gather, out_dev, sync)


class MoEMLP:
    """Mixture-of-experts feed-forward block ``y[t] = sum_j w[t, j] * down_e(act(gate_e(x_t)) * up_e(x_t))`` with
    e = ids[t, j]: router, one gated product over all buckets, quantiser, one down product, weighted combine — seven
    launches for a few tokens, ten for many, whatever the number of experts, none of them waiting for the host, so
    that the block can be captured into a graph (after a first call with as many rows, which sizes the buffers).  ``gate_up`` is a gated ``ExpertLinear``, ``down`` a plain one."""

    def __init__(self, rt: Runtime, router: MoERouter, gate_up: ExpertLinear, down: ExpertLinear, ws: Workspace | None = None,
                 tag: str | None = None):
        if not gate_up.gated or gate_up.n != down.k or down.n != gate_up.k or down.n % 4:
            raise ValueError("gate_up must be gated, its outputs the inputs of down, and down's outputs as many as its "
                             "inputs (a multiple of 4)")
        if not router.n_exp == gate_up.n_exp == down.n_exp:
            raise ValueError("router, gate_up and down have different numbers of experts")
        self.rt, self.router, self.gate_up, self.down = rt, router, gate_up, down
        self.dim = down.n
        self.tag = tag or f"moe_mlp_{id(self):x}"
        self._own_ws = ws is None
        self.ws = ws or Workspace(rt)

    def forward_device(self, x_dev: int, logits_dev: int, rows: int, sync: bool = False, out_dev: int | None = None) -> int:
        """x ``[rows, dim]`` f32 and the router's logits -> y ``[rows, dim]`` f32."""
        rt, pairs = self.rt, rows * self.router.topk
        y = int(out_dev) if out_dev is not None else self.ws.buffer(self.tag + ".y", max(1, rows) * self.dim * 4)
        if rows:
            plan = self.router.forward_device(logits_dev, rows)
            h = self.ws.buffer(self.tag + ".h", pairs * self.gate_up.n * 4)
            d = self.ws.buffer(self.tag + ".d", pairs * self.dim * 4)
            # a pair without a slot names row 0 of the buckets: written even if no pair has a slot (the combine drops it, its weight is 0)
            rt.memset(d, 0, self.dim * 4)
            self.gate_up.forward_device(x_dev, plan, out_dev=h)
            self.down.forward_device(h, plan, gather=False, out_dev=d)
            rt.launch("moe_combine_gather_k", rows, 64, [y, d, plan.weights, plan.base, plan.topk, rows, self.dim])
        if sync:
            rt.sync()
        return y

    def forward(self, x: np.ndarray, logits: np.ndarray) -> np.ndarray:
        x, logits = _as_rows(x), _as_rows(logits)
        if x.shape[1] != self.dim or logits.shape != (x.shape[0], self.router.n_exp) or self.router.dtype != "f32":
            raise ValueError(f"x {x.shape} and f32 logits {logits.shape} for {self.dim} values and {self.router.n_exp} experts")
        out = self.forward_device(self.ws.upload(self.tag + ".x", x), self.ws.upload(self.tag + ".logits", logits), x.shape[0], sync=True)
        return self.rt.download(out, x.shape[0] * self.dim, np.float32).reshape(x.shape[0], self.dim)
