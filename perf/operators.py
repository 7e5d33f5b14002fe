"""The operators around the EXL3 experts of a layer, as timed cases: the general router gate, the 16-bit matrix product
with its epilogue, its gated form, and the two products together as the MLP of a dense layer or of a shared expert.

A case is a dict of plain values. kind:
  "route"  gfr_moe.route_gate: router logits [rows, routed] -> picks and weights [rows, topk + 1]
           score ("softmax" over all experts, "sigmoid"), bias (a per-expert bias of the choice), groups, kept (of these
           groups), group_score ("max", "top2"), renorm (weights divided by their sum), scale, type (of the logits)
  "dense"  gfr_moe.dense: out = act(x w^T + bias) + residual, x [rows, k], w [n, k]
  "gated"  gfr_moe.dense_gated: out = act(min(g, limit)) * clamp(u, -limit, limit), g and u the halves of x w^T,
           w [2 n, k]; limit 0: none
  "mlp"    the two one after the other: hidden k -> inter n -> hidden, with a residual

`own` false: the plain form, in elementary torch operations; true: the framework's entry points.
"""
import math
import os
import sys

import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ROUTE = dict(kind="route", bias=False, groups=1, kept=1, group_score="max", renorm=True, scale=1.0, type="fp32")
DENSE = dict(kind="dense", bias=False, act="none", residual="none", type="bf16", out="same", pad=0)
GATED = dict(kind="gated", act="silu", limit=0.0, type="bf16", out="same", pad=0)
MLP = dict(kind="mlp", act="silu", limit=0.0, type="bf16")
# the largest listed case's multiply-adds: no drawn one has more
MOST = 8192 * 5120 * 12288 * 3


def listed():
    return [
        # one token's routing in a layer of 288 experts: sigmoid scores, the bias for balance, half of the groups kept
        dict(ROUTE, name="route 1 row", rows=1, routed=288, topk=8, score="sigmoid", bias=True, groups=8, kept=4,
             group_score="top2", scale=2.5),
        # the tail of a prompt, 16-bit logits, softmax scores kept as they are, groups by their best expert
        dict(ROUTE, name="route 77 rows bf16", rows=77, routed=160, topk=6, score="softmax", groups=8, kept=3,
             renorm=False, type="bf16"),
        # a prefill chunk through a small layer: softmax with a bias for balance, no groups
        dict(ROUTE, name="route 8192 rows", rows=8192, routed=64, topk=4, score="softmax", bias=True),
        # the tokens of several prefill chunks at once, the gate of the first case
        dict(ROUTE, name="route 32768 rows", rows=32768, routed=256, topk=8, score="sigmoid", bias=True, groups=8,
             kept=4, group_score="top2", scale=2.5),
        # one token's down projection added to the residual stream
        dict(DENSE, name="dense 1 row", rows=1, k=1536, n=5120, residual="same"),
        # a tail of odd sizes: rows that end off every alignment, a bias and a GELU
        dict(DENSE, name="dense 77 rows odd", rows=77, k=1001, n=2077, bias=True, act="gelu", type="fp16"),
        # a prompt's down projection into a 32-bit residual stream
        dict(DENSE, name="dense 709 rows fp32 out", rows=709, k=12288, n=5120, bias=True, residual="fp32", out="fp32"),
        # one token through the gate and up matrices of a dense layer: the weights are read once
        dict(GATED, name="gated 1 row", rows=1, k=5120, n=12288),
        # a verify window through a 16-bit shared expert with the limited SwiGLU
        dict(GATED, name="gated 12 rows", rows=12, k=4096, n=512, limit=10.0),
        # a prefill window through the same, its rows a slice of a wider buffer
        dict(GATED, name="gated 4096 rows", rows=4096, k=4096, n=512, limit=10.0, pad=512),
        # a verify window of several streams through a small MLP
        dict(MLP, name="mlp 32 rows", rows=32, k=2048, n=1536),
        # the largest: a full prefill chunk through a dense layer
        dict(MLP, name="mlp 8192 rows", rows=8192, k=5120, n=12288),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["route", "dense", "gated", "mlp"])
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        routed = groups * rng.randint(max(4, 16 // groups), 512 // groups)
        kept = rng.randint(1, groups)
        return dict(kind=kind, rows=spread(1, 32768), routed=routed, topk=rng.randint(1, min(12, kept * routed // groups)),
                    score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.6, groups=groups, kept=kept,
                    group_score=rng.choice(["max", "top2"]), renorm=rng.random() < 0.6, scale=rng.choice([1.0, 2.5]),
                    type=rng.choice(["fp32", "fp32", "bf16", "fp16"]))
    # hidden sizes as models have them, or anything at all
    step = rng.choice([128, 128, 8, 1])
    k, n = step * (spread(256, 12288) // step), step * (spread(256, 12288) // step)
    halves = {"dense": 1, "gated": 2, "mlp": 3}[kind]
    rows = spread(1, max(1, min(8192, MOST // (halves * k * n))))
    case = dict(kind=kind, rows=rows, k=k, n=n, type=rng.choice(["bf16", "bf16", "fp16"]))
    if kind == "dense":
        case.update(bias=rng.random() < 0.5, act=rng.choice(["none", "none", "relu", "gelu", "gelu_tanh", "silu"]),
                    residual=rng.choice(["none", "same", "fp32"]))
    else:
        case.update(act=rng.choice(["silu", "silu", "gelu"]), limit=rng.choice([0.0, 10.0]))
    if kind != "mlp":
        case.update(out=rng.choice(["same", "same", "fp32"]), pad=rng.choice([0, 0, 8, 512]))
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _matrix(g, n, k, dtype, size=1.0):
    """Weights whose products with rows of N(0, 1) are of the order of `size`."""
    return (_randn(g, n, k) * (size / k ** 0.5)).to(dtype)


def prepare(case, seed):
    """Inputs from the seed alone: logits of a trained router's spread and a small bias for balance; activations of
    order one, weights that keep them there (the limit of the gated form is met now and then)."""
    g = _gen(seed)
    s = dict(case)
    dt = DTYPE[case["type"]]
    if case["kind"] == "route":
        s["logits"] = (_randn(g, case["rows"], case["routed"]) * 1.5).to(dt)
        s["bias"] = _randn(g, case["routed"]) * 0.02 if case["bias"] else None
        return s
    rows, k, n = case["rows"], case["k"], case["n"]
    s["x"] = _randn(g, rows, k + case.get("pad", 0)).to(dt)[:, :k]
    if case["kind"] == "dense":
        s["w"] = _matrix(g, n, k, dt)
        s["bias"] = _randn(g, n) * 0.5 if case["bias"] else None
        res = case["residual"]
        s["residual"] = None if res == "none" else _randn(g, rows, n).to(dt if res == "same" else DTYPE[res])
    else:
        s["w"] = _matrix(g, 2 * n, k, dt, 2.0)
        if case["kind"] == "mlp":
            s["down"] = _matrix(g, k, n, dt)
            s["residual"] = _randn(g, rows, k).to(dt)
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------
_module = None


def _gfr():
    global _module
    if _module is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "glm-flash-rs_amd"))
        import gfr_moe
        _module = gfr_moe
    return _module


def _out_dtype(s):
    return DTYPE[s["type"]] if s["out"] == "same" else DTYPE[s["out"]]


def run(state):
    s = state
    if own:
        gfr = _gfr()
        if s["kind"] == "route":
            gate = gfr.Gate(score=s["score"], bias=s["bias"], groups=s["groups"], kept_groups=s["kept"],
                            group_score=s["group_score"], renormalise=s["renorm"], scale=s["scale"])
            return gfr.route_gate(s["logits"], gate, s["topk"])
        if s["kind"] == "dense":
            return gfr.dense(s["x"], s["w"], bias=s["bias"], activation=s["act"], residual=s["residual"],
                             out_dtype=_out_dtype(s))
        if s["kind"] == "gated":
            return gfr.dense_gated(s["x"], s["w"], activation=s["act"], limit=s["limit"], out_dtype=_out_dtype(s))
        act = gfr.dense_gated(s["x"], s["w"], activation=s["act"], limit=s["limit"])
        return gfr.dense(act, s["down"], residual=s["residual"])
    if s["kind"] == "route":
        return _plain_route(s)
    if s["kind"] == "dense":
        y = s["x"].float() @ s["w"].float().t()
        y = _act(y if s["bias"] is None else y + s["bias"], s["act"])
        return (y if s["residual"] is None else y + s["residual"].float()).to(_out_dtype(s))
    a = _plain_gated(s)
    if s["kind"] == "gated":
        return a.to(_out_dtype(s))
    return (a @ s["down"].float().t() + s["residual"].float()).to(DTYPE[s["type"]])


def _act(v, act):
    if act == "relu":
        return v.clamp(min=0)
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh((2 / math.pi) ** 0.5 * (v + 0.044715 * v * v * v)))
    if act == "silu":
        return v / (1 + torch.exp(-v))
    return v


def _plain_gated(s):
    gu = s["x"].float() @ s["w"].float().t()
    g, u = gu[:, :s["n"]], gu[:, s["n"]:]
    if s["limit"]:
        g, u = g.clamp(max=s["limit"]), u.clamp(-s["limit"], s["limit"])
    return _act(g, s["act"]) * u


def _plain_route(s):
    """In 64 bits, so that neighbours in the order stay apart; sorts that keep the lower index first among equals."""
    l = s["logits"].double()
    rows, E = l.shape
    if s["score"] == "softmax":
        e = torch.exp(l - l.max(1, keepdim=True).values)
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-l))
    choice = l if s["bias"] is None else score + s["bias"].double()      # without a bias the logits have the scores' order
    if s["kept"] < s["groups"]:
        if s["group_score"] == "top2":
            per = (score if s["bias"] is None else choice).view(rows, s["groups"], -1)
            value = per.sort(dim=2, descending=True).values[:, :, :2].sum(2)
        else:
            value = choice.view(rows, s["groups"], -1).max(2).values
        kept = value.sort(dim=1, descending=True, stable=True).indices[:, :s["kept"]]
        keep = torch.zeros_like(value, dtype=torch.bool).scatter_(1, kept, True)
        choice = choice.masked_fill(~keep.repeat_interleave(E // s["groups"], 1), -math.inf)
    picks = choice.sort(dim=1, descending=True, stable=True).indices[:, :s["topk"]]
    w = score.gather(1, picks)
    if s["renorm"]:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    picks = torch.cat((picks, torch.full_like(picks[:, :1], E)), 1)
    w = torch.cat((w * s["scale"], torch.ones_like(w[:, :1])), 1)
    return picks.int(), w.float()


# ---- the work of a pass ---------------------------------------------------------------------------------------------
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    rows, e = case["rows"], size[case["type"]]
    if case["kind"] == "route":
        E = case["routed"]
        return {"bytes": rows * (E * e + 8 * (case["topk"] + 1)) + (4 * E if case["bias"] else 0),
                "flops": rows * E * 4}
    k, n = case["k"], case["n"]
    if case["kind"] == "mlp":
        return {"bytes": e * (3 * n * k + 3 * rows * k), "flops": 2 * rows * 3 * n * k}
    halves = 2 if case["kind"] == "gated" else 1
    out = rows * n * size[case["type"] if case["out"] == "same" else case["out"]]
    more = 0
    if case["kind"] == "dense":
        more += 4 * n if case["bias"] else 0
        more += {"none": 0, "same": e, "fp32": 4}[case["residual"]] * rows * n
    return {"bytes": e * (halves * n * k + rows * k) + out + more, "flops": 2 * rows * halves * n * k}


# ---- the same in 64 bits, from the definitions ------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "route":
        # an expert's place in the order: how many come before it (a larger value, or an equal one of a lower index)
        def place(v):
            i = torch.arange(v.shape[1], device="cuda")
            a, b = v.unsqueeze(2), v.unsqueeze(1)                         # a: the expert asked for, b: the others
            return ((b > a) | ((b == a) & (i < i.unsqueeze(1)))).sum(2)

        parts = []
        step = max(1, (1 << 27) // case["routed"] ** 2)
        for r in range(0, case["rows"], step):
            l = s["logits"][r:r + step].double()
            score = torch.softmax(l, 1) if case["score"] == "softmax" else torch.sigmoid(l)
            c = l if s["bias"] is None else score + s["bias"].double()
            if case["kept"] < case["groups"]:
                G, P = case["groups"], case["routed"] // case["groups"]
                if case["group_score"] == "top2":
                    v = (score if s["bias"] is None else c).reshape(-1, G, P)
                    first = place(v.reshape(-1, P)).view(v.shape)
                    v = torch.where(first < 2, v, torch.zeros_like(v)).sum(2)
                else:
                    v = c.reshape(-1, G, P).amax(2)
                c = torch.where((place(v) < case["kept"]).unsqueeze(2), c.reshape(-1, G, P), -math.inf).flatten(1)
            at = place(c)
            slot = torch.arange(case["topk"], device="cuda").view(1, -1, 1)
            w = ((at.unsqueeze(1) == slot).double() * score.unsqueeze(1)).sum(2)
            if case["renorm"]:
                w = w / (w.sum(1, keepdim=True) + 1e-20)
            parts.append(torch.cat((w * case["scale"], torch.ones_like(w[:, :1])), 1))
        return None, torch.cat(parts)

    def product(a, b):
        return torch.mm(a.double(), b.double().t())

    def activation(v, act):
        if act == "none":
            return v
        if act == "relu":
            return torch.where(v > 0, v, torch.zeros_like(v))
        if act == "gelu":
            return v * torch.special.ndtr(v)
        if act == "gelu_tanh":
            return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
        return v * torch.sigmoid(v)

    if case["kind"] == "dense":
        y = product(s["x"], s["w"])
        if s["bias"] is not None:
            y += s["bias"].double()
        y = activation(y, case["act"])
        return y if s["residual"] is None else y + s["residual"].double()
    g, u = product(s["x"], s["w"][:case["n"]]), product(s["x"], s["w"][case["n"]:])
    if case["limit"]:
        g, u = torch.clamp(g, max=case["limit"]), torch.clamp(u, -case["limit"], case["limit"])
    a = activation(g, case["act"]) * u
    return a if case["kind"] == "gated" else torch.mm(a, s["down"].double().t()) + s["residual"].double()
