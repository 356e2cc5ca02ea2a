"""Performance cases of the mixture-of-experts routing and of the W4A8 products with an epilogue.

Three operators of a quantised decoder layer:

``route``    router logits -> experts and weights of every token, and the plan that sorts the (token, expert) pairs
             into one contiguous bucket per expert;
``linear``   y = act(x . W^T + bias) + residual with int4 weights and int8 activations, one scale per 128 k on both
             sides (optionally gated: act(gate) * up from stacked gate and up rows);
``experts``  the same product for every expert's bucket of a plan.

``run`` computes them from elementary torch operations in 32 bits (64 where the order of nearly equal scores is
decided) while ``own`` is false, and through the package's public classes while it is true.
"""
import pathlib
import sys

import numpy as np
import torch

own = False

ROOT = pathlib.Path(__file__).resolve().parents[1]
GROUP = 128
LARGEST = 2048 * 17408 * 5120          # multiply-adds of the largest listed case


# ------------------------------------------------------------------------------------------------------- cases
def _route(name, rows, experts, topk, score, dtype="f32", bias=False, groups=1, kept=1, top=1, scale=1.0):
    return {"name": name, "op": "route", "rows": rows, "experts": experts, "topk": topk, "score": score, "dtype": dtype,
            "bias": bias, "groups": groups, "kept": kept, "group_top": top, "scale": scale}


def _linear(name, rows, n, k, act="none", gated=False, bias=False, residual=False):
    return {"name": name, "op": "linear", "rows": rows, "n": n, "k": k, "act": act, "gated": gated, "bias": bias,
            "residual": residual}


def _experts(name, rows, experts, topk, n, k, act="none", gated=False, bias=False, gather=True):
    return {"name": name, "op": "experts", "rows": rows, "experts": experts, "topk": topk, "n": n, "k": k, "act": act,
            "gated": gated, "bias": bias, "gather": gather}


def listed():
    return [
        # one decoded token, plain softmax router: launch latency
        _route("route one token", 1, 128, 8, "softmax"),
        # a decode batch with group-limited sigmoid routing and a balance bias
        _route("route decode batch", 48, 256, 8, "sigmoid", bias=True, groups=8, kept=4, top=2, scale=2.5),
        # prefill with an expert count that is no power of two and an odd token count
        _route("route odd prefill", 3001, 60, 4, "softmax"),
        # a long prefill, 16-bit logits (many equal ones), balance bias and groups
        _route("route long prefill", 16384, 256, 8, "sigmoid", dtype="bf16", bias=True, groups=8, kept=4, top=2, scale=2.5),
        # one decoded token through the wide projection of the feed-forward block
        _linear("linear one token", 1, 17408, 5120, act="silu", bias=True),
        # five sequences through the down projection, added to the residual stream
        _linear("linear decode down", 5, 5120, 17408, residual=True),
        # a short prompt through stacked gate and up projections
        _linear("linear gated prompt", 77, 6144, 5120, act="silu", gated=True),
        # prefill through the wide projection
        _linear("linear prefill", 2048, 17408, 5120, act="gelu", bias=True),
        # one decoded token through its eight experts' gate and up projections
        _experts("experts one token", 1, 64, 8, 1024, 5120, act="silu", gated=True),
        # a decode batch through the experts' down projections (the rows are in bucket order already)
        _experts("experts decode down", 33, 64, 8, 5120, 1024, gather=False),
        # an odd prefill through few experts, row count of the weights no multiple of any tile
        _experts("experts odd", 301, 24, 4, 1000, 2048, act="relu", bias=True),
        # prefill through all experts' gate and up projections
        _experts("experts prefill", 1999, 64, 8, 1024, 5120, act="silu", gated=True),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["route", "linear", "experts"])
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * _log(rng, 8, 256 // groups)
        kept = max(1, groups // 2)
        topk = rng.randint(1, min(8, kept * (experts // groups)))
        biased = rng.random() < 0.5
        return _unnamed(_route("", _log(rng, 1, 16384), experts, topk, rng.choice(["softmax", "sigmoid"]),
                               rng.choice(["f32", "bf16", "f16"]), biased, groups, kept, 2 if biased and groups > 1 else 1,
                               rng.choice([1.0, 2.5])))
    act = rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"])
    gated = act != "none" and rng.random() < 0.5
    if op == "linear":
        n, k = _log(rng, 200, 17408 // (1 + gated)), 128 * _log(rng, 1, 136)
        rows = min(_log(rng, 1, 4096), max(1, LARGEST // (n * (1 + gated) * k)))
        return _unnamed(_linear("", rows, n, k, act, gated, rng.random() < 0.5, rng.random() < 0.5))
    experts, n, k = _log(rng, 4, 64), _log(rng, 100, 5120 // (1 + gated)), 128 * _log(rng, 2, 40)
    topk = rng.randint(1, min(8, experts))
    rows = min(_log(rng, 1, 2048), max(1, LARGEST // (topk * n * (1 + gated) * k)))
    return _unnamed(_experts("", rows, experts, topk, n, k, act, gated, rng.random() < 0.5, rng.random() < 0.7))


def _unnamed(case):
    del case["name"]
    return case


def work(case):
    rows = case["rows"]
    if case["op"] == "route":
        e, k = case["experts"], case["topk"]
        size = 4 if case["dtype"] == "f32" else 2
        # logits in; experts, weights, positions and bucket rows of every pair and the bucket bounds out
        return {"bytes": rows * e * size + (4 * e if case["bias"] else 0) + rows * k * 16 + 4 * (e + 1), "flops": 10 * rows * e}
    n_out, k = case["n"], case["k"]
    n = n_out * (2 if case["gated"] else 1)
    weights = n * k // 2 + n * (k // GROUP) * 2 + (4 * n if case["bias"] else 0)
    codes = k + (k // GROUP) * 8
    if case["op"] == "linear":
        return {"bytes": weights + rows * codes + 4 * rows * n_out * (2 if case["residual"] else 1), "flops": 2 * rows * n * k}
    e, topk = case["experts"], case["topk"]
    pairs = rows * topk
    hit = e * (1 - (1 - topk / e) ** rows)              # experts that some token chose, were all equally popular
    return {"bytes": hit * weights + (rows if case["gather"] else pairs) * codes + 4 * pairs * n_out + 4 * pairs,
            "flops": 2 * pairs * n * k}


# ------------------------------------------------------------------------------------------------------ inputs
def _quantise(x):
    """The int8 activation codes of x [rows, k]: even and odd k apart, a scale and the sum of the codes per 128 k."""
    rows, k = x.shape
    g = x.view(rows, k // GROUP, GROUP)
    scale = g.abs().amax(-1) / 127
    q = torch.clamp(torch.round(g / scale[..., None]), -128, 127).to(torch.int8).view(rows, k)
    return {"ae": q[:, 0::2].contiguous(), "ao": q[:, 1::2].contiguous(), "asc": scale.contiguous(),
            "asu": q.view(rows, k // GROUP, GROUP).sum(-1, dtype=torch.int32).contiguous()}


def _plan(logits, topk):
    """Experts chosen by the largest logits, and their buckets."""
    rows, experts = logits.shape
    values, ids = torch.topk(logits, topk, dim=-1)
    weights = torch.softmax(values, -1)
    flat = ids.reshape(-1)
    order = torch.argsort(flat, stable=True)
    base = torch.empty_like(order)
    base[order] = torch.arange(order.numel(), device=order.device)
    counts = torch.bincount(flat, minlength=experts)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=flat.device)
    offsets[1:] = counts.cumsum(0)
    return {"ids": ids.to(torch.int32), "weights": weights, "bucket_rows": (order // topk).to(torch.int32),
            "base": base.to(torch.int32).view(rows, topk), "offsets": offsets}, int(counts.max())


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    s = {"case": case}
    if case["op"] == "route":
        logits = normal(case["rows"], case["experts"]) * 1.5 + normal(case["experts"]) * 0.5
        s["logits"] = logits.to({"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[case["dtype"]])
        s["bias"] = normal(case["experts"]) * 0.05 if case["bias"] else None
    else:
        stack = case.get("experts", 1)
        n, k = case["n"] * (2 if case["gated"] else 1), case["k"]
        s["wq"] = torch.randint(0, 256, (stack, n, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
        s["ws"] = (normal(stack, n, k // GROUP).abs() * 0.01 + 1e-3).to(torch.float16)
        s["bias"] = normal(stack, n) if case["bias"] else None
        rows = case["rows"]
        if case["op"] == "experts":
            s["plan"], s["largest"] = _plan(normal(rows, stack) + normal(stack) * 0.5, case["topk"])
            rows = rows if case["gather"] else rows * case["topk"]
        s["codes"] = _quantise(normal(rows, k))
        s["residual"] = normal(rows, case["n"]) * 4 if case.get("residual") else None
    if own:
        s["engine"] = _Engine(s)
    return s


# -------------------------------------------------------------------------------------------------- plain forms
def _act(name, v):
    if name == "relu":
        return torch.clamp(v, min=0)
    if name == "silu":
        return v / (1 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * 0.7071067811865476))
    if name == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v)))
    return v


def _weights(wq, ws):
    """Two's-complement nibbles (low nibble first) times the scale of their group, in 32 bits."""
    low, high = (((wq & 15) ^ 8).to(torch.int8) - 8), (((wq >> 4) ^ 8).to(torch.int8) - 8)
    w = torch.stack((low, high), -1).view(*wq.shape[:-1], -1, GROUP)
    return (w.float() * ws.float()[..., None]).flatten(-2)


def _activations(codes):
    q = torch.stack((codes["ae"], codes["ao"]), -1).flatten(1)
    return (q.view(q.shape[0], -1, GROUP).float() * codes["asc"][..., None]).flatten(1)


def _epilogue(case, v, bias, residual):
    if bias is not None:
        v = v + bias
    if case["gated"]:
        gate, up = v[..., : case["n"]], v[..., case["n"]:]
        v = _act(case["act"], gate) * up
    else:
        v = _act(case["act"], v)
    return v if residual is None else v + residual


def _plain_route(s):
    case, logits = s["case"], s["logits"].double()
    rows, e = logits.shape
    if case["score"] == "softmax":
        score = torch.exp(logits - logits.amax(-1, keepdim=True))
        score = score / score.sum(-1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-logits))
    key = score if s["bias"] is None else score + s["bias"].double()
    if case["groups"] > 1:
        g = key.view(rows, case["groups"], -1)
        best = torch.sort(g, -1, descending=True)[0][..., : case["group_top"]].sum(-1)
        keep = torch.sort(best, dim=-1, descending=True, stable=True)[1][:, : case["kept"]]
        mask = torch.zeros_like(best, dtype=torch.bool).scatter_(1, keep, True)
        key = torch.where(mask[..., None], g, -torch.inf).view(rows, e)
    ids = torch.sort(key, dim=-1, descending=True, stable=True)[1][:, : case["topk"]]
    w = torch.gather(score, 1, ids)
    weights = (w / w.sum(-1, keepdim=True) * case["scale"]).float()
    flat = ids.reshape(-1)
    order = torch.sort(flat, dim=0, stable=True)[1]
    base = torch.empty_like(order)
    base[order] = torch.arange(order.numel(), device=order.device)
    counts = (flat[:, None] == torch.arange(e, device=flat.device)).sum(0)
    offsets = torch.cat((counts.new_zeros(1), counts.cumsum(0)))
    return {"ids": ids.int(), "weights": weights, "bucket_rows": (order // case["topk"]).int(),
            "base": base.view(rows, -1).int(), "offsets": offsets.int()}


def _plain_linear(s):
    v = _activations(s["codes"]) @ _weights(s["wq"][0], s["ws"][0]).T
    return _epilogue(s["case"], v, None if s["bias"] is None else s["bias"][0], s["residual"])


def _plain_experts(s):
    case, plan = s["case"], s["plan"]
    pairs = plan["bucket_rows"].numel()
    slot = torch.arange(pairs, device="cuda")
    expert = torch.searchsorted(plan["offsets"][1:].long(), slot, right=True)
    x = _activations(s["codes"])
    if case["gather"]:
        x = x[plan["bucket_rows"].long()]
    bias = None if s["bias"] is None else s["bias"][expert]
    if pairs <= case["experts"]:                                      # few pairs: each with its own expert's weights
        v = torch.bmm(_weights(s["wq"][expert], s["ws"][expert]), x[..., None])[..., 0]
    else:                                                             # buckets padded to the fullest one
        place = slot - plan["offsets"].long()[expert]
        padded = x.new_zeros(case["experts"], s["largest"], x.shape[1])
        padded[expert, place] = x
        v = torch.bmm(padded, _weights(s["wq"], s["ws"]).transpose(1, 2))[expert, place]
    return _epilogue(case, v, bias, None)


# ------------------------------------------------------------------------------------------- the package's calls
class _Buffers:
    """Device buffers of one state, freed when neither the state nor one of its outputs is in use any more."""

    def __init__(self, workspace):
        self.workspace = workspace

    def view(self, ptr, shape, typestr):
        return torch.as_tensor(_Memory(self, ptr, shape, typestr), device="cuda")

    def __del__(self):
        self.workspace.free()


class _Memory:
    """Names memory of the engine to torch; a tensor made from it keeps the buffers."""

    def __init__(self, owner, ptr, shape, typestr):
        self.owner = owner
        self.__cuda_array_interface__ = {"data": (ptr, False), "shape": tuple(shape), "typestr": typestr, "version": 3}


class _Engine:
    """The handles and device buffers that a user's program keeps between calls."""

    runtime = None

    def __init__(self, s):
        if str(ROOT / "k100lc-kernels_b200") not in sys.path:
            sys.path.insert(0, str(ROOT / "k100lc-kernels_b200"))
        import k100lc_kernels as kk
        if _Engine.runtime is None:
            _Engine.runtime = kk.Runtime()
        rt, case = _Engine.runtime, s["case"]
        ws = kk.Workspace(rt)
        self.buffers, self.views = _Buffers(ws), {}

        def put(name, t):
            if t is None:
                return None
            p = ws.buffer(name, t.numel() * t.element_size())
            self.buffers.view(p, (t.numel() * t.element_size(),), "|u1").copy_(t.contiguous().view(-1).view(torch.uint8))
            return p

        rows = case["rows"]
        if case["op"] == "route":
            bias = None if s["bias"] is None else s["bias"].cpu().numpy()
            self.op = kk.MoERouter(rt, case["experts"], case["topk"], score=case["score"], bias=bias, n_group=case["groups"],
                                   topk_group=case["kept"], group_top=case["group_top"], scale=case["scale"],
                                   dtype=case["dtype"], ws=ws)
            self.logits = put("logits", s["logits"])
            torch.cuda.synchronize()                                  # the engine has a stream of its own
            return
        wq, scales, bias = put("wq", s["wq"]), put("ws", s["ws"]), put("bias", s["bias"])
        self.codes = tuple(put(n, s["codes"][n]) for n in ("ae", "ao", "asc", "asu"))
        self.residual = put("residual", s["residual"])
        if case["op"] == "linear":
            self.op = kk.FusedLinear(rt, case["n"], case["k"], wq, scales, bias=bias, act=case["act"], gated=case["gated"], ws=ws)
        else:
            self.op = kk.ExpertLinear(rt, case["experts"], case["n"], case["k"], wq, scales, bias=bias, act=case["act"],
                                      gated=case["gated"], ws=ws)
            self.plan = kk.MoEPlan(rows=rows, topk=case["topk"], n_exp=case["experts"],
                                   **{n: put("plan." + n, t) for n, t in s["plan"].items()})
            rows = rows * case["topk"]
        self.out = ws.buffer("out", rows * case["n"] * 4)
        self.result = self.buffers.view(self.out, (rows, case["n"]), "<f4")
        torch.cuda.synchronize()

    def run(self, case):
        if case["op"] == "route":
            plan = self.op.forward_device(self.logits, case["rows"])
            if not self.views:                                        # the router's buffers, named once
                pairs, view = (case["rows"], case["topk"]), self.buffers.view
                self.views = {"ids": view(plan.ids, pairs, "<i4"), "weights": view(plan.weights, pairs, "<f4"),
                              "bucket_rows": view(plan.bucket_rows, (pairs[0] * pairs[1],), "<i4"),
                              "base": view(plan.base, pairs, "<i4"),
                              "offsets": view(plan.offsets, (case["experts"] + 1,), "<i4")}
            return self.views
        if case["op"] == "linear":
            self.op.forward_codes_device(self.codes, case["rows"], residual_dev=self.residual, out_dev=self.out)
        else:
            self.op.forward_codes_device(self.codes, self.plan, gather=case["gather"], out_dev=self.out)
        return self.result


def run(state):
    if own:
        return state["engine"].run(state["case"])
    return {"route": _plain_route, "linear": _plain_linear, "experts": _plain_experts}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(case, s)
    q = torch.empty(s["codes"]["ae"].shape[0], case["k"], dtype=torch.float64, device="cuda")
    q[:, 0::2], q[:, 1::2] = s["codes"]["ae"].double(), s["codes"]["ao"].double()
    a = q * s["codes"]["asc"].double().repeat_interleave(GROUP, dim=1)

    def layer(e, rows):
        b = s["wq"][e].to(torch.int16)
        w = torch.empty(b.shape[0], case["k"], dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = ((b % 16 + 8) % 16 - 8).double(), ((b // 16 + 8) % 16 - 8).double()
        w *= s["ws"][e].double().repeat_interleave(GROUP, dim=1)
        v = torch.mm(rows, w.t())
        if s["bias"] is not None:
            v += s["bias"][e].double()
        head = v[:, : case["n"]]
        act = {"none": lambda t: t, "relu": lambda t: torch.where(t > 0, t, torch.zeros_like(t)),
               "silu": lambda t: t * torch.sigmoid(t), "gelu": lambda t: t * torch.special.ndtr(t),
               "gelu_tanh": lambda t: t * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (t + 0.044715 * t ** 3))}[case["act"]]
        return act(head) * v[:, case["n"]:] if case["gated"] else act(head)

    if case["op"] == "linear":
        y = layer(0, a)
        return y if s["residual"] is None else y + s["residual"].double()
    bounds = s["plan"]["offsets"].tolist()
    a = a[s["plan"]["bucket_rows"].long()] if case["gather"] else a
    return torch.cat([layer(e, a[lo:hi]) for e, (lo, hi) in enumerate(zip(bounds, bounds[1:])) if hi > lo])


def _exact_route(case, s):
    x = s["logits"].double().cpu().numpy()
    rows, e = x.shape
    if case["score"] == "softmax":
        score = np.exp(x - np.log(np.exp(x - x.max(1, keepdims=True)).sum(1, keepdims=True)) - x.max(1, keepdims=True))
    else:
        score = np.reciprocal(1 + np.exp(-x))
    key = score if s["bias"] is None else score + s["bias"].double().cpu().numpy()
    if case["groups"] > 1:
        g = key.reshape(rows, case["groups"], -1)
        best = np.sort(g, axis=-1)[..., -case["group_top"]:].sum(-1)
        kept = np.argsort(-best, axis=-1, kind="stable")[:, : case["kept"]]
        out = np.full_like(g, -np.inf)
        np.put_along_axis(out, kept[..., None], np.take_along_axis(g, kept[..., None], 1), 1)
        key = out.reshape(rows, e)
    ids = np.argsort(-key, axis=-1, kind="stable")[:, : case["topk"]]
    w = np.take_along_axis(score, ids, 1)
    # the whole-number outputs have no value in 64 bits: they are compared with the plain form's
    return {"ids": None, "weights": torch.from_numpy(w / w.sum(1, keepdims=True) * case["scale"]), "bucket_rows": None,
            "base": None, "offsets": None}
