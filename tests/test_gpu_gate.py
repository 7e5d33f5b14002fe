"""The general router gate (gfr_route_gate, Gate, Moe.set_gate) against its formulas in 64 bits, row by row in numpy.

Picks have to be equal. Weights: the kernel's scores are 32-bit sums and quotients: expf within 2 units (2^-22), at most
22 additions in a lane's and the lanes' part of the softmax's sum and 31 in the renormalisation's, one rounding (2^-24)
each, and a handful of roundings around them: under 64 * 2^-24 = 2^-18 relative. A 32-bit score below 2^-126 may be
flushed, which the renormalisation's 1e-20 turns into at most 2^-126 / 1e-20 = 1.2e-18 times the scale."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

REL, ABS = 2.0 ** -18, 1.2e-18


def reference(logits, topk, score, bias, groups, kept, group_score, renorm, scale, shared, undecided=None):
    """undecided: a list that gets the rows whose last kept and first dropped groups' values 64-bit arithmetic cannot
    tell apart."""
    l = np.asarray(logits, np.float64)
    rows, E = l.shape
    P = E // groups
    picks, weights = [], []
    for r in range(rows):
        row = l[r]
        live = ~np.isnan(row) & (row > -np.inf)
        s = np.zeros(E)
        if score == "softmax":
            if live.any():
                m = row[live].max()
                with np.errstate(invalid="ignore"):
                    e = np.where(row[live] == m, 1.0, np.exp(np.where(row[live] == m, 0, row[live] - m)))
                s[live] = e / e.sum()
        else:
            with np.errstate(over="ignore"):
                s[live] = 1 / (1 + np.exp(-row[live]))
        c = np.where(live, row if bias is None else s + np.asarray(bias, np.float64), -np.inf)
        live = live & ~np.isnan(c) & (c > -np.inf)
        c = np.where(live, c, -np.inf)
        keep = np.ones(E, bool)
        if kept < groups:
            value = np.full(groups, -np.inf)
            for g in range(groups):
                v = (s if group_score == "top2" and bias is None else c)[g * P:(g + 1) * P][live[g * P:(g + 1) * P]]
                v = np.sort(v)[::-1]
                if len(v):
                    value[g] = v[0] if group_score == "max" or len(v) == 1 else v[0] + v[1]
            order = sorted(range(groups), key=lambda g: (-value[g], g))
            keep[:] = False
            a, b = value[order[kept - 1]], value[order[kept]]
            if undecided is not None and group_score == "top2" and a - b <= 2.0 ** -50 * abs(a):
                undecided.append(r)
            for g in order[:kept]:
                keep[g * P:(g + 1) * P] = True
        first = sorted((e for e in range(E) if keep[e] and live[e]), key=lambda e: (-c[e], e))
        rest = [e for e in range(E) if keep[e] and not live[e]]
        pk = (first + rest)[:topk]
        w = np.array([s[e] if live[e] else 0.0 for e in pk])
        if renorm:
            w = w / (w.sum() + 1e-20)
        picks.append(pk + ([E] if shared else []))
        weights.append(list(w * scale) + ([1.0] if shared else []))
    return np.array(picks, np.int32), np.array(weights)


def run_both(gfr, logits, topk, score="sigmoid", bias=None, groups=1, kept=1, group_score="top2", renorm=True, scale=1.0,
             shared=True, what="", undecided=None):
    gate = gfr.Gate(score=score, bias=None if bias is None else torch.tensor(bias, dtype=torch.float32, device="cuda"),
                    groups=groups, kept_groups=kept, group_score=group_score, renormalise=renorm, scale=scale)
    p, w = gfr.route_gate(logits, gate, topk, shared=shared)
    torch.cuda.synchronize()
    wp, ww = reference(logits.float().cpu().numpy(), topk, score, bias, groups, kept, group_score, renorm,
                       np.float32(scale), shared, undecided)
    if undecided:
        p, w = p.clone(), w.clone()
        p[undecided], w[undecided] = torch.from_numpy(wp[undecided]).cuda(), torch.from_numpy(ww[undecided]).float().cuda()
    bad = np.nonzero((p.cpu().numpy() != wp).any(1))[0]
    assert not len(bad), f"{what} row {bad[0]}: picks {p[bad[0]].tolist()}, want {wp[bad[0]].tolist()}"
    got = w.cpu().numpy().astype(np.float64)
    err = np.abs(got - ww) - (REL * np.abs(ww) + ABS * scale)
    assert (err <= 0).all(), f"{what}: weight off by {np.abs(got - ww).max()}"
    return p, w


def bias_of(E, seed, size=0.02):
    return (np.random.default_rng(seed).standard_normal(E) * size).astype(np.float32)


def logits_of(rows, E, seed, dtype=torch.float32, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, E), generator=g) * spread).to(dtype).cuda()


SHAPES = [  # routed, groups, kept, topk
    (1, 1, 1, 1), (2, 2, 1, 1), (5, 1, 1, 5), (31, 1, 1, 31), (64, 1, 1, 4), (64, 64, 7, 7), (96, 3, 2, 6), (160, 8, 3, 6),
    (200, 5, 5, 8), (256, 8, 4, 8), (256, 1, 1, 12), (288, 8, 4, 8), (288, 9, 2, 31), (384, 2, 1, 10), (500, 4, 3, 16),
    (513, 1, 1, 8), (990, 33, 4, 20), (1023, 3, 1, 7), (1024, 1, 1, 31), (1024, 64, 9, 8),
]


@pytest.mark.parametrize("E,groups,kept,topk", SHAPES)
@pytest.mark.parametrize("score,bias", [("softmax", False), ("softmax", True), ("sigmoid", False), ("sigmoid", True)])
def test_gate_shapes(gfr, E, groups, kept, topk, score, bias):
    for i, (gs, renorm, dtype, rows) in enumerate([("top2", True, torch.float32, 37), ("max", False, torch.float32, 5),
                                                   ("top2", False, torch.bfloat16, 19), ("max", True, torch.float16, 70)]):
        l = logits_of(rows, E, 31 * E + i, dtype)
        run_both(gfr, l, topk, score, bias_of(E, E + i) if bias else None, groups, kept, gs, renorm, 2.5,
                 shared=i != 1, what=f"{gs} {dtype}")


@pytest.mark.parametrize("rows", [1, 2, 3, 63, 1023, 4097, 9001])
@pytest.mark.parametrize("E,groups,kept,topk", [(64, 1, 1, 4), (256, 8, 4, 8), (288, 8, 4, 8), (160, 8, 3, 6), (100, 1, 1, 15)])
def test_gate_rows(gfr, rows, E, groups, kept, topk):
    """Windows of every size, whatever form they run in; a row's bytes do not depend on the window."""
    l = logits_of(rows, E, rows + E)
    b = bias_of(E, 7)
    p, w = run_both(gfr, l[:997], topk, "sigmoid", b, groups, kept, scale=2.5)
    gate = gfr.Gate(bias=torch.from_numpy(b).cuda(), groups=groups, kept_groups=kept, scale=2.5)
    pa, wa = gfr.route_gate(l, gate, topk)
    assert torch.equal(pa[:997], p) and torch.equal(wa[:997], w)
    tail = l[-5:].contiguous()
    pt, wt = gfr.route_gate(tail, gate, topk)
    assert torch.equal(pa[-5:], pt) and torch.equal(wa[-5:], wt)


@pytest.mark.parametrize("E,groups,kept,topk", [(64, 1, 1, 4), (288, 8, 4, 8), (96, 3, 2, 6), (256, 8, 4, 8), (512, 4, 1, 20)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("gs", ["max", "top2"])
def test_gate_masks(gfr, E, groups, kept, topk, score, gs):
    """Masked experts: -inf and NaN logits, whole groups, rows with fewer live experts than picks and with none; the
    type's lowest value is a number; +inf logits; biases of -inf and NaN."""
    rng = np.random.default_rng(E + topk)
    l = (rng.standard_normal((40, E)) * 1.5).astype(np.float32)
    l[0] = -np.inf
    l[1] = np.nan
    l[2, :] = -np.inf
    l[2, E - 1] = 0.5                                   # one live expert
    l[3, rng.random(E) < 0.9] = -np.inf
    l[4, rng.random(E) < 0.9] = np.nan
    l[5] = np.finfo(np.float32).min
    l[6, rng.random(E) < 0.5] = np.finfo(np.float32).min
    l[7, : E // groups] = -np.inf                       # a group without live experts
    l[8, E // 3] = np.inf
    l[9, [0, E // 2, E - 1]] = np.inf
    l[10] = np.inf
    l[11, :] = -np.inf
    l[11, [1, E - 2]] = [-200.0, -201.0]                # live experts whose scores are all but nothing
    l[12] = np.finfo(np.float32).max
    for r in range(13, 40):
        l[r, rng.random(E) < rng.random()] = rng.choice([-np.inf, np.nan])
    b = bias_of(E, 3)
    odd = b.copy()
    odd[rng.random(E) < 0.3] = -np.inf
    odd[rng.random(E) < 0.1] = np.nan
    none = np.full(E, -np.inf, np.float32)
    for bias in (None, b, odd, none):
        for renorm in (True, False):
            run_both(gfr, torch.from_numpy(l).cuda(), topk, score, bias, groups, kept, gs, renorm, 1.5,
                     what=f"bias {None if bias is None else bias[:2]}")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("E,groups,kept,topk", [(64, 1, 1, 6), (256, 8, 4, 8), (288, 8, 3, 8), (40, 4, 2, 9)])
def test_gate_ties(gfr, score, with_bias, E, groups, kept, topk):
    """Equal logits: the lower id (and the lower group) first."""
    rng = np.random.default_rng(E)
    l = rng.integers(-3, 4, (300, E)).astype(np.float32)
    l[0] = 0.0
    l[1] = np.where(np.arange(E) % 2, 0.0, -0.0)
    l[2] = rng.choice([-0.0, 0.0], E)
    bias = rng.choice([0.0, 0.25], E).astype(np.float32) if with_bias else None
    for gs in ("max", "top2"):
        run_both(gfr, torch.from_numpy(l).cuda(), topk, score, bias, groups, kept, gs)


@pytest.mark.parametrize("E,groups,kept,topk", [(64, 1, 1, 6), (256, 8, 4, 8), (288, 8, 4, 8)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_gate_choices_closer_than_32_bits(gfr, E, groups, kept, topk, score):
    """Choices whose order 32-bit scores would lose: neighbouring logits, with a bias that makes the choice a sum.

    Sums of two scores of evenly spaced logits can be closer than 64 bits hold: for logits m - i d and m - j d they are
    exp(-i d) + exp(-j d) = 2 - (i + j) d + (i^2 + j^2) d^2 / 2 - .., so that pairs of equal i + j differ by d^2 / 2 times
    an integer: with the row of base 0.0197 (d = 1.86e-9) of the 256 experts, two group values are
    0.007812501695298235937.. and ..234693.. (computed with 40 digits), 1.5e-16 apart relative to their size, below
    2^-52. Either order is right there: rows whose border's two sums are within 2^-50 (two exponentials, a sum and a
    quotient of half to one unit 2^-52 each) are left out, at most a tenth of them."""
    rng = np.random.default_rng(E + topk)
    rows = 200
    l = np.empty((rows, E), np.float32)
    for r in range(rows):
        base = np.float32(rng.uniform(-1, 6))
        l[r] = base + rng.permutation(E).astype(np.float32) * np.spacing(base) * rng.integers(1, 4)
    assert (np.diff(np.sort(l, 1)) > 0).mean() > 0.8, "the logits have to differ"
    for bias in (np.zeros(E, np.float32), np.full(E, 0.75, np.float32)):
        for gs in ("max", "top2"):
            open_rows = []
            run_both(gfr, torch.from_numpy(l).cuda(), topk, score, bias, groups, kept, gs, undecided=open_rows)
            assert len(open_rows) <= rows // 10
    open_rows = []
    run_both(gfr, torch.from_numpy(l).cuda(), topk, score, None, groups, kept, "top2", undecided=open_rows)
    assert len(open_rows) <= rows // 10


def test_gate_strides_and_untouched_rows(gfr):
    """Rows of a wider buffer (odd strides, an odd start), and nothing written behind the rows' results."""
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for E, pad, start in ((64, 1, 1), (160, 3, 5), (256, 64, 4), (288, 7, 0)):
            buf = logits_of(23, E + pad + start, E, dtype)
            buf[:, :start] = float("nan")
            buf[:, start + E:] = float("inf")
            run_both(gfr, buf[:, start:start + E], 4, bias=bias_of(E, 1), what=f"{dtype} {E}")
    E, rows, topk = 64, 9, 4
    l = logits_of(rows, E, 3)
    picks = torch.full((rows + 2, topk + 1), -7, dtype=torch.int32, device="cuda")
    weights = torch.full((rows + 2, topk + 1), -7.0, device="cuda")
    L = gfr.lib()
    assert L.gfr_route_gate(gfr._stream(), l.data_ptr(), 2, E, rows, E, topk, gfr.Gate().pack(E), 1, picks.data_ptr(),
                            weights.data_ptr()) == 0
    torch.cuda.synchronize()
    assert (picks[:rows] >= 0).all() and (picks[rows:] == -7).all() and (weights[rows:] == -7).all()


def test_gate_offsets_past_32_bits(gfr):
    """Rows more than 2^32 bytes and 2^31 elements behind the first."""
    rows, E, stride = 1100, 64, 1 << 21
    buf = torch.empty(rows * stride, dtype=torch.bfloat16, device="cuda")
    view = buf.view(rows, stride)[:, :E]
    l = logits_of(rows, E, 5, torch.bfloat16)
    view.copy_(l)
    gate = gfr.Gate(score="softmax", renormalise=False)
    p, w = gfr.route_gate(view, gate, 4)
    p0, w0 = gfr.route_gate(l, gate, 4)
    assert torch.equal(p, p0) and torch.equal(w, w0)


def test_gate_streams_and_graph(gfr):
    """On another stream, and in a graph that is replayed with new logits between eager calls."""
    E, rows, topk = 256, 50, 8
    gate = gfr.Gate(bias=torch.from_numpy(bias_of(E, 2)).cuda(), groups=8, kept_groups=4, scale=2.5)
    l = logits_of(rows, E, 1)
    want = gfr.route_gate(l, gate, topk)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = gfr.route_gate(l, gate, topk, stream=s)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    static = l.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = gfr.route_gate(static, gate, topk)
    for seed in range(4):
        new = logits_of(rows, E, 10 + seed)
        static.copy_(new)
        graph.replay()
        eager = gfr.route_gate(new, gate, topk)
        torch.cuda.synchronize()
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])


def test_gate_against_the_two_gates(gfr):
    """Where they mean the same, the gates of gfr_route_topk and gfr_route_topk_biased: the same picks, weights within
    both sides' rounding (the bound above twice)."""
    E, rows, topk = 288, 200, 8
    l = logits_of(rows, E, 9)
    b = torch.from_numpy(bias_of(E, 4)).cuda()
    p, w = gfr.route_gate(l, gfr.Gate(score="softmax"), topk)
    p0, w0 = gfr.route(l, topk)
    assert torch.equal(p, p0) and ((w - w0).abs() <= 2 * REL * w0).all()
    p, w = gfr.route_gate(l, gfr.Gate(bias=b, scale=2.5), topk)
    p0, w0 = gfr.route_biased(l, b, topk, 2.5)
    assert torch.equal(p, p0) and ((w - w0).abs() <= 2 * REL * w0).all()


# ---- the layer with the gate ------------------------------------------------------------------------------------------
D, N, E, TOPK, BITS = 512, 256, 24, 4, 4
ROWS = [1, 2, 4, 5, 20, 40, 300]        # the decode engine, the split-K windows, the large grouping


@pytest.fixture(scope="module")
def layer_weights():
    import synth
    return synth.experts(E + 1, D, N, BITS, seed=5), synth.experts(E, D, N, BITS, seed=6)


@pytest.mark.parametrize("rows", ROWS)
def test_moe_with_the_gate(gfr, layer_weights, rows):
    """Groups in the layer: the same outputs as GLM's gate on logits whose other groups are out of reach (the same picks;
    weights and outputs within the two gates' rounding), and back to that gate afterwards, byte for byte."""
    import synth
    w = layer_weights[0]
    x, l = synth.activations(rows, D, rows), synth.logits(rows, E, 70 + rows)
    b = torch.from_numpy(bias_of(E, 8)).cuda()
    gate = gfr.Gate(bias=b, groups=6, kept_groups=3, group_score="top2", scale=2.5)
    m = gfr.Moe(D, N, E, TOPK, rows)
    m.set_router(b, 2.5)
    m.run(w, x, l, rows)
    before = m.output.clone(), m.picks.clone(), m.weights.clone()
    m.set_gate(gate)
    m.run(w, x, l, rows)
    p, wt = gfr.route_gate(l, gate, TOPK)
    torch.cuda.synchronize()
    assert torch.equal(m.picks, p) and torch.equal(m.weights, wt)
    got = m.output.clone()
    choice = torch.sigmoid(l.double()) + b.double()
    value = choice.view(rows, 6, -1).sort(dim=2, descending=True).values[:, :, :2].sum(2)
    kept = value.sort(dim=1, descending=True, stable=True).indices[:, :3]
    keep = torch.zeros(rows, 6, dtype=torch.bool, device="cuda").scatter_(1, kept, True).repeat_interleave(E // 6, 1)
    m.set_gate(None)
    m.run(w, x, torch.where(keep, l, torch.full_like(l, -60.0)), rows)
    torch.cuda.synchronize()
    assert torch.equal(m.picks, p)
    # a row is a weighted sum of TOPK + 1 outputs: weights 2 REL apart, one rounding a term
    scale = m.output.abs().amax(1, keepdim=True)
    assert ((got - m.output).abs() <= (2 * REL + 2.0 ** -20) * (TOPK + 1) * scale).all()
    m.run(w, x, l, rows)
    torch.cuda.synchronize()
    assert torch.equal(m.output, before[0]) and torch.equal(m.picks, before[1]) and torch.equal(m.weights, before[2])


@pytest.mark.parametrize("rows", [1, 3, 20, 300])
def test_moe_gate_fp8_shared(gfr, layer_weights, rows):
    """The FP8 shared expert next to the gate: byte-equal to the layer that is given its output."""
    import synth
    w = layer_weights[1]
    x, l = synth.activations(rows, D, rows), synth.logits(rows, E, rows)
    sw = synth.fp8_shared(D, N)
    m = gfr.Moe(D, N, E, TOPK, rows, shared_exl3=False)
    m.set_gate(gfr.Gate(score="softmax", groups=4, kept_groups=2, group_score="max", renormalise=False))
    m.run_fp8(w, x, l, sw, rows)
    torch.cuda.synchronize()
    got, shared = m.output.clone(), m.shared_output[:rows].clone()
    m.output.zero_()
    m.run(w, x, l, rows, shared=shared)
    torch.cuda.synchronize()
    assert torch.equal(m.output, got)


@pytest.mark.parametrize("rows", [1, 4, 30])
def test_moe_gate_graph(gfr, layer_weights, rows):
    """The whole set in one graph: router logits, the gate, the bf16 shared expert's products, the experts."""
    import synth
    w = layer_weights[1]
    g = torch.Generator().manual_seed(3)
    rw = (torch.randn((E, D), generator=g) / D ** 0.5).to(torch.bfloat16).cuda()
    sw = gfr.Bf16SharedWeights((torch.randn((2 * N, D), generator=g) / D ** 0.5).to(torch.bfloat16).cuda(),
                               (torch.randn((D, N), generator=g) / N ** 0.5).to(torch.bfloat16).cuda())
    m = gfr.Moe(D, N, E, TOPK, rows, shared_exl3=False)
    m.set_gate(gfr.Gate(bias=torch.from_numpy(bias_of(E, 8)).cuda(), groups=6, kept_groups=2, scale=2.5))
    x = synth.activations(rows, D, 1)
    m.run_router_bf16(w, x, rw, sw, rows)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(graph, stream=s):
            m.run_router_bf16(w, x, rw, sw, rows, stream=s)
    for seed in range(4):
        x.copy_(synth.activations(rows, D, 50 + seed))
        torch.cuda.synchronize()
        m.run_router_bf16(w, x, rw, sw, rows)
        torch.cuda.synchronize()
        eager = m.output.clone()
        m.output.zero_()
        with torch.cuda.stream(s):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(m.output, eager)


def test_moe_bf16_refuses(gfr, layer_weights):
    import synth
    w = layer_weights[1]
    x, l = synth.activations(4, D, 1), synth.logits(4, E, 1)
    sw = gfr.Bf16SharedWeights(torch.zeros(2 * N, D, dtype=torch.bfloat16, device="cuda"),
                               torch.zeros(D, N, dtype=torch.bfloat16, device="cuda"))
    m = gfr.Moe(D, N, E, TOPK, 4, shared_exl3=False)
    for args in ((x.half(), l, sw, 4), (x[:, :D - 8], l, sw, 4), (x, l.half(), sw, 4), (x, l[:3], sw, 4), (x, l, sw, 5)):
        with pytest.raises((ValueError, gfr.GfrError)):
            m.run_bf16(w, *args)
    wide = gfr.Bf16SharedWeights(torch.zeros(4 * N, D, dtype=torch.bfloat16, device="cuda"),
                                 torch.zeros(D, 2 * N, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(gfr.GfrError, match="inter up to"):
        m.run_bf16(w, x, l, wide, 4)
    with pytest.raises(gfr.GfrError, match="EXL3"):
        gfr.Moe(D, N, E, TOPK, 4).run_bf16(layer_weights[0], x, l, sw, 4)
    with pytest.raises(gfr.GfrError, match="topk"):
        m.set_gate(gfr.Gate(groups=12, kept_groups=1))


def test_moe_holds_the_gate_bias(gfr, layer_weights):
    """The layer's gate is the one it was given: its bias stays alive when the caller's object gets another, and when a
    later gate is refused; a later gate that is taken lets it go."""
    import weakref
    m = gfr.Moe(D, N, E, TOPK, 4)
    gate = gfr.Gate(bias=torch.from_numpy(bias_of(E, 9)).cuda())
    bias = weakref.ref(gate.bias)
    m.set_gate(gate)
    gate.bias = None
    assert bias() is not None
    with pytest.raises(gfr.GfrError, match="topk"):
        m.set_gate(gfr.Gate(groups=12, kept_groups=1))
    assert bias() is not None
    m.set_gate(gate)
    assert bias() is None


@pytest.mark.parametrize("rows", [1, 3, 20, 300])
@pytest.mark.parametrize("hidden", [512, 768])
def test_moe_bf16_shared(gfr, rows, hidden):
    """The layer with an unquantised shared expert: byte-equal to the layer that is given the two products' output."""
    import synth
    w = synth.experts(E, hidden, N, BITS, seed=6)
    x, l = synth.activations(rows, hidden, rows), synth.logits(rows, E, rows)
    g = torch.Generator().manual_seed(rows)
    inter = 192
    sw = gfr.Bf16SharedWeights((torch.randn((2 * inter, hidden), generator=g) * 3 / hidden ** 0.5).to(torch.bfloat16).cuda(),
                               (torch.randn((hidden, inter), generator=g) / inter ** 0.5).to(torch.bfloat16).cuda(), 2.0)
    m = gfr.Moe(hidden, N, E, TOPK, rows, shared_exl3=False)
    m.run_bf16(w, x, l, sw, rows)
    torch.cuda.synchronize()
    got = m.output.clone()
    act = gfr.dense_gated(x, sw.gu, limit=2.0)
    shared = gfr.dense(act, sw.down, out_dtype=torch.float32)
    m.output.zero_()
    m.run(w, x, l, rows, shared=shared)
    torch.cuda.synchronize()
    assert torch.equal(m.output, got)
