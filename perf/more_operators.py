"""The operators between a layer's 16-bit products and experts and after them, as timed cases: the norms around a block
with its gate and residual, 16-bit routed experts for a few tokens, and the log probabilities of given tokens.

A case is a dict of plain values. kind:
  "norm"      gfr_moe.block_norm (gfr_moe.norm where it has no residual, gate and post norm): x [rows, n] ->
              h = residual_scale * residual + scale * gate * post(x), y = pre(h)
              norm ("rms", "layer" with biases), post (a norm before the gate), gate ("none", "column": [n], "row":
              [rows, 1], "full": [rows, n]), sigmoid (of the gate), stream (the type of residual and h, "none": neither
              is there), type (of x, the gate and y), weight (the type of the norms' weights), pad (columns between rows)
  "experts"   gfr_moe.experts16: x [rows, hidden], picks and weights [rows, slots] -> the weighted sum of the picked
              experts' gated MLPs, gu [experts, 2 inter, hidden], down [experts, hidden, inter]
              popular (experts that every row picks), shared (the last expert is every row's last slot), padded (rows at
              the end whose picks are all -1), residual
  "logprobs"  gfr_moe.token_logprobs: logits [rows, vocab], tokens [rows, tokens] -> log probabilities, entropy, the top
              alternatives; masked (share of the vocabulary at -inf)

`own` false: the plain form, in elementary torch operations; true: the framework's entry points.
"""
import math
import os
import sys

import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "none": 0}
EPS = 1e-5
NORM = dict(kind="norm", norm="rms", post=False, gate="none", sigmoid=False, scale=1.0, residual_scale=1.0, stream="bf16",
            x="same", type="bf16", weight="same", pad=0)
EXPERTS = dict(kind="experts", popular=0, shared=False, padded=0, act="silu", limit=0.0, residual=False, type="bf16")
LOGPROBS = dict(kind="logprobs", tokens=1, top=0, temperature=1.0, masked=0.0, pad=0, type="bf16")
# the largest listed cases': no drawn one has more
MOST_NORM, MOST_WEIGHTS, MOST_PAIRS, MOST_LOGITS = 16384 * 5120, 160 * 3 * 5120 * 1408, 64 * 8, 4096 * 160000


def listed():
    return [
        # one token's layer output (fp32, as the experts' layer gives it) into the stream, and the next block's rows
        dict(NORM, name="norm 1 row", rows=1, n=4096, x="fp32"),
        # a tail of odd sizes: a layer norm with biases, a gate a channel, a scaled branch
        dict(NORM, name="norm 77 rows odd", rows=77, n=1001, norm="layer", gate="column", scale=0.22, stream="fp16",
             type="fp16", weight="fp32"),
        # a prefill chunk's heads, each normed by itself, between the other columns of their projection
        dict(NORM, name="norm 65536 heads", rows=65536, n=128, stream="none", pad=64),
        # the largest: prefill chunks through both norms of a block and its gate, an fp32 stream
        dict(NORM, name="norm 16384 rows", rows=16384, n=5120, post=True, gate="full", sigmoid=True, residual_scale=0.9,
             stream="fp32"),
        # one token through the picked experts and the shared one
        dict(EXPERTS, name="experts 1 row", rows=1, hidden=4096, inter=512, experts=289, slots=9, shared=True),
        # a few rows of odd sizes off every alignment
        dict(EXPERTS, name="experts 5 rows odd", rows=5, hidden=1001, inter=333, experts=20, slots=3, act="gelu",
             type="fp16", residual=True),
        # a verify window padded to 12 rows, the limited SwiGLU
        dict(EXPERTS, name="experts 12 rows", rows=12, hidden=4096, inter=512, experts=288, slots=8, padded=2,
             limit=10.0),
        # the largest: the windows of several streams, one expert that all of them pick
        dict(EXPERTS, name="experts 64 rows", rows=64, hidden=5120, inter=1408, experts=160, slots=8, popular=1,
             residual=True),
        # one token's choice with its alternatives, from an fp32 head
        dict(LOGPROBS, name="logprobs 1 row", rows=1, vocab=160000, top=20, type="fp32"),
        # a verify window's drafted tokens
        dict(LOGPROBS, name="logprobs 16 rows", rows=16, vocab=131072, top=8),
        # candidates under a grammar's mask, an odd vocabulary, rows off alignment
        dict(LOGPROBS, name="logprobs 77 rows odd", rows=77, vocab=32003, tokens=3, top=5, temperature=0.7, masked=0.9,
             pad=6, type="fp16"),
        # the largest: a prompt's tokens scored
        dict(LOGPROBS, name="logprobs 4096 rows", rows=4096, vocab=160000, top=4),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    kind = rng.choice(["norm", "experts", "logprobs"])
    kinds = ["bf16", "bf16", "fp16"]
    step = rng.choice([128, 128, 8, 1])
    if kind == "norm":
        n = step * (spread(128, 16384) // step)
        case = dict(NORM, rows=spread(1, min(65536, MOST_NORM // n)), n=n, norm=rng.choice(["rms", "rms", "layer"]),
                    type=rng.choice(kinds), weight=rng.choice(["same", "fp32"]), pad=rng.choice([0, 0, 8, 3]))
        if rng.random() < 0.2:
            return dict(case, stream="none")
        gate = rng.choice(["none", "column", "row", "full"])
        return dict(case, post=rng.random() < 0.5, gate=gate, sigmoid=gate != "none" and rng.random() < 0.5,
                    scale=rng.choice([1.0, 0.22]), residual_scale=rng.choice([1.0, 0.9]),
                    stream=rng.choice([case["type"], case["type"], "fp32"]), x=rng.choice(["same", "fp32"]))
    if kind == "experts":
        hidden, inter = step * (spread(256, 7168) // step), step * (spread(128, 2048) // step)
        experts = rng.randint(8, max(8, min(320, MOST_WEIGHTS // (3 * hidden * inter))))
        slots = rng.randint(1, min(8, experts - 1))
        rows = spread(1, min(128, MOST_PAIRS // slots))
        return dict(EXPERTS, rows=rows, hidden=hidden, inter=inter, experts=experts, slots=slots,
                    popular=rng.choice([0, 0, 1]) if slots > 1 else 0, padded=rng.choice([0, 0, rows // 4]),
                    act=rng.choice(["silu", "silu", "gelu"]), limit=rng.choice([0.0, 10.0]),
                    residual=rng.random() < 0.5, type=rng.choice(kinds))
    vocab = step * (spread(1000, 160000) // step)
    return dict(LOGPROBS, rows=spread(1, min(8192, MOST_LOGITS // vocab)), vocab=vocab, tokens=rng.choice([1, 1, 4]),
                top=rng.choice([0, 1, 5, 20, 32]), temperature=rng.choice([1.0, 1.0, 0.7]),
                masked=rng.choice([0.0, 0.0, 0.5]), pad=rng.choice([0, 0, 8, 5]), type=rng.choice(kinds + ["fp32"]))


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _rows(g, rows, n, pad, dtype, size=1.0):
    """Rows of N(0, size^2) that are a slice of a wider buffer where pad is set."""
    return (_randn(g, rows, n + pad) * size).to(dtype)[:, :n]


def _stack(g, experts, n, k, dtype, size=1.0):
    """Every expert's [n, k] weights, whose products with rows of N(0, 1) are of the order of `size`."""
    w = torch.empty((experts, n, k), dtype=dtype, device="cuda")
    for e in range(experts):
        w[e] = _randn(g, n, k) * (size / k ** 0.5)
    return w


def _type(case, what):
    return DTYPE[case["type"] if case[what] == "same" else case[what]]


def prepare(case, seed):
    """Inputs from the seed alone: activations of order one with a few wide channels, weights that keep their size; picks
    of a row are distinct, weights a softmax over them; logits of a trained head's spread, tokens that it holds likely."""
    g, s = _gen(seed), dict(case)
    rows, dt = case["rows"], DTYPE[case["type"]]
    if case["kind"] == "norm":
        n = case["n"]
        wide = 1 + 8 * (torch.rand(n, generator=g, device="cuda") < 0.01).float()
        s["in"] = _rows(g, rows, n, case["pad"], _type(case, "x"))
        s["in"].mul_(wide)
        wt = _type(case, "weight")
        s["pre"] = (1 + 0.3 * _randn(g, n)).to(wt), (0.1 * _randn(g, n)).to(wt) if case["norm"] == "layer" else None
        s["after"] = None
        if case["post"]:
            s["after"] = (1 + 0.3 * _randn(g, n)).to(wt), (0.1 * _randn(g, n)).to(wt) if case["norm"] == "layer" else None
        shape = {"none": None, "column": (n,), "row": (rows, 1), "full": (rows, n)}[case["gate"]]
        s["by"] = None if shape is None else _randn(g, *shape).to(dt)
        s["residual"] = None if case["stream"] == "none" else (_randn(g, rows, n) * 2 * wide).to(DTYPE[case["stream"]])
        return s
    if case["kind"] == "experts":
        E, H, I, slots = case["experts"], case["hidden"], case["inter"], case["slots"]
        s["in"] = _randn(g, rows, H).to(dt)
        s["gu"], s["down"] = _stack(g, E, 2 * I, H, dt, 2.0), _stack(g, E, H, I, dt)
        routed = E - 1 if case["shared"] else E
        logits = _randn(g, rows, routed)
        logits[:, :case["popular"]] += 100
        top = logits.sort(dim=1, descending=True)
        picks = top.indices[:, :slots - 1 if case["shared"] else slots]
        weights = torch.softmax(_randn(g, *picks.shape), 1)
        if case["shared"]:
            picks = torch.cat((picks, torch.full_like(picks[:, :1], E - 1)), 1)
            weights = torch.cat((weights, torch.ones_like(weights[:, :1])), 1)
        picks = picks.int().contiguous()
        if case["padded"]:
            picks[rows - case["padded"]:] = -1
        s["picks"], s["weights"] = picks, weights.contiguous()
        s["residual"] = _randn(g, rows, H).to(dt) if case["residual"] else None
        return s
    V = case["vocab"]
    s["logits"] = _rows(g, rows, V, case["pad"], dt, 2.5)
    tokens = torch.randint(0, V, (rows, case["tokens"]), generator=g, device="cuda")
    best = s["logits"][:, :1000].float().argmax(1)                        # a likely one among the first thousand
    tokens[:, 0] = best
    if case["masked"]:
        s["logits"].masked_fill_(torch.rand((1, V), generator=g, device="cuda") < case["masked"], -math.inf)
        s["logits"][:, :1000][torch.arange(rows, device="cuda"), best] = 9.0
    s["tokens"] = tokens
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


def _own_norm(gfr, s):
    def made(w):
        return None if w is None else gfr.Norm(kind=s["norm"], weight=w[0], bias=w[1], eps=EPS)

    if s["stream"] == "none":
        return gfr.norm(s["in"], made(s["pre"]), out_dtype=DTYPE[s["type"]])
    return gfr.block_norm(s["in"], s["residual"], pre=made(s["pre"]), post=made(s["after"]), gate=s["by"],
                          gate_activation="sigmoid" if s["sigmoid"] else None, scale=s["scale"],
                          residual_scale=s["residual_scale"], out_dtype=DTYPE[s["type"]])


def run(state):
    s = state
    if own:
        gfr = _gfr()
        if s["kind"] == "norm":
            return _own_norm(gfr, s)
        if s["kind"] == "experts":
            return gfr.experts16(s["in"], gfr.Experts16(s["gu"], s["down"]), s["picks"], s["weights"],
                                 activation=s["act"], limit=s["limit"], residual=s["residual"])
        return tuple(t for t in gfr.token_logprobs(s["logits"], s["tokens"], top=s["top"], temperature=s["temperature"])
                     if t is not None)
    if s["kind"] == "norm":
        return _plain_norm(s)
    return _plain_experts(s) if s["kind"] == "experts" else _plain_logprobs(s)


def _normed(v, w, kind):
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(1, keepdim=True) + EPS) * w[0].float()
    return v if w[1] is None else v + w[1].float()


def _plain_norm(s):
    v = s["in"].float()
    if s["stream"] == "none":
        return _normed(v, s["pre"], s["norm"]).to(DTYPE[s["type"]])
    if s["after"] is not None:
        v = _normed(v, s["after"], s["norm"])
    if s["by"] is not None:
        b = s["by"].float()
        v = v * (1 / (1 + torch.exp(-b)) if s["sigmoid"] else b)
    h = s["residual_scale"] * s["residual"].float() + s["scale"] * v
    return h.to(DTYPE[s["stream"]]), _normed(h, s["pre"], s["norm"]).to(DTYPE[s["type"]])


def _act(v, act):
    return 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5)) if act == "gelu" else v / (1 + torch.exp(-v))


def _plain_experts(s):
    """Each pair's own copy of its expert's weights where the pairs are fewer than the experts, else every expert's
    product with every row, of which the picked ones are taken."""
    x, picks, I = s["in"].float(), s["picks"].long(), s["inter"]
    rows, slots = picks.shape
    there = picks >= 0
    ids = picks.clamp(min=0)

    def gated(gu):                                                        # [..., 2 inter]
        gate, up = gu[..., :I], gu[..., I:]
        if s["limit"]:
            gate, up = gate.clamp(max=s["limit"]), up.clamp(-s["limit"], s["limit"])
        return _act(gate, s["act"]) * up

    if rows * slots < s["experts"]:
        at = ids.flatten()
        each = x.repeat_interleave(slots, 0).unsqueeze(2)                 # [pairs, hidden, 1]
        a = gated(torch.bmm(s["gu"][at].float(), each).squeeze(2))
        y = torch.bmm(s["down"][at].float(), a.unsqueeze(2)).view(rows, slots, -1)
    else:
        E = s["experts"]
        a = gated(torch.bmm(s["gu"].float(), x.t().contiguous().expand(E, -1, -1)).transpose(1, 2))   # [E, rows, inter]
        y = torch.bmm(s["down"].float(), a.transpose(1, 2).contiguous())                              # [E, hidden, rows]
        y = y[ids, :, torch.arange(rows, device="cuda").unsqueeze(1)]
    y = (y * torch.where(there, s["weights"], torch.zeros_like(s["weights"])).unsqueeze(2)).sum(1)
    return (y if s["residual"] is None else y + s["residual"].float()).to(DTYPE[s["type"]])


def _plain_logprobs(s):
    l, T = s["logits"].float(), s["temperature"]
    d = (l - l.max(1, keepdim=True).values) / T
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log = torch.log(total)
    out = [d.gather(1, s["tokens"]) - log, (log - torch.where(e > 0, e * d, torch.zeros_like(d)).sum(1, keepdim=True)
                                            / total).squeeze(1)]
    if s["top"]:
        order = l.sort(dim=1, descending=True, stable=True).indices[:, :s["top"]]
        out += [order.int(), d.gather(1, order) - log]
    return tuple(out)


# ---- the work of a pass ---------------------------------------------------------------------------------------------
def work(case):
    rows, e = case["rows"], SIZE[case["type"]]
    if case["kind"] == "norm":
        n = case["n"]
        gate = {"none": 0, "column": n, "row": rows, "full": rows * n}[case["gate"]]
        weights = (1 + case["post"]) * (2 if case["norm"] == "layer" else 1) * n
        x = e if case["x"] == "same" else SIZE[case["x"]]
        return {"bytes": rows * n * (x + 2 * SIZE[case["stream"]] + e) + gate * e
                + weights * (e if case["weight"] == "same" else SIZE[case["weight"]]),
                "flops": rows * n * (6 + 4 * case["post"])}
    if case["kind"] == "experts":
        H, I, slots, real = case["hidden"], case["inter"], case["slots"], rows - case["padded"]
        # experts that at least one row picks: those that all do, and on average this many of the others
        always = case["popular"] + case["shared"]
        others = case["experts"] - always
        used = (always if real else 0) + others * (1 - (1 - (slots - always) / others) ** real)
        return {"bytes": e * (3 * used * H * I + rows * H * (2 + case["residual"])) + rows * slots * 8,
                "flops": 2 * real * slots * 3 * H * I}
    return {"bytes": rows * (case["vocab"] * e + case["tokens"] * 12 + 4 + case["top"] * 8),
            "flops": rows * case["vocab"] * 5}


# ---- the same in 64 bits, from the definitions ------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        def norm(z, w):
            if case["norm"] == "layer":
                var, mean = torch.var_mean(z, dim=1, correction=0, keepdim=True)
                z = (z - mean) * torch.rsqrt(var + EPS)
            else:
                z = z * torch.rsqrt(torch.linalg.vector_norm(z, dim=1, keepdim=True) ** 2 / z.shape[1] + EPS)
            return z * w[0].double() if w[1] is None else torch.addcmul(w[1].double(), z, w[0].double())

        z = s["in"].double()
        if case["stream"] == "none":
            return norm(z, s["pre"])
        if s["after"] is not None:
            z = norm(z, s["after"])
        if s["by"] is not None:
            z = z * (torch.sigmoid(s["by"].double()) if case["sigmoid"] else s["by"].double())
        h = s["residual"].double() * case["residual_scale"] + z * case["scale"]
        return h, norm(h, s["pre"])
    if case["kind"] == "experts":
        out = torch.zeros((case["rows"], case["hidden"]), dtype=torch.float64, device="cuda")
        if s["residual"] is not None:
            out += s["residual"].double()
        picks = s["picks"].tolist()
        members = {}
        for r, row in enumerate(picks):
            for slot, e in enumerate(row):
                if e >= 0:
                    members.setdefault(e, []).append((r, slot))
        for e, pairs in members.items():
            r = torch.tensor([p[0] for p in pairs], device="cuda")
            slot = torch.tensor([p[1] for p in pairs], device="cuda")
            both = torch.mm(s["in"][r].double(), s["gu"][e].double().t())
            gate, up = both.split(case["inter"], 1)
            if case["limit"]:
                gate, up = torch.clamp(gate, max=case["limit"]), torch.clamp(up, -case["limit"], case["limit"])
            gate = gate * (torch.special.ndtr(gate) if case["act"] == "gelu" else torch.sigmoid(gate))
            y = torch.mm(gate * up, s["down"][e].double().t())
            out.index_add_(0, r, y * s["weights"][r, slot].double().unsqueeze(1))
        return out
    parts = []
    for r in range(0, case["rows"], max(1, (1 << 27) // case["vocab"])):
        rows = slice(r, r + max(1, (1 << 27) // case["vocab"]))
        lp = torch.log_softmax(s["logits"][rows].double() / case["temperature"], 1)
        p = torch.exp(lp)
        part = [lp.gather(1, s["tokens"][rows]), -torch.special.xlogy(p, p).sum(1)]
        if case["top"]:
            part += [None, lp.topk(case["top"], 1).values]
        parts.append(part)
    return tuple(None if c[0] is None else torch.cat(c) for c in zip(*parts))
