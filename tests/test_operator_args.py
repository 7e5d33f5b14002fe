"""What the general gate and the 16-bit products refuse: host checks before any launch (no GPU needed)."""
import pytest


def gate(gfr, **kw):
    g = dict(score=1, groups=1, kept_groups=1, group_score=0, renormalise=1, scale=1.0, bias=None)
    g.update(kw)
    return gfr._GATE.pack(*[g[n] or 0 for n in ("score", "groups", "kept_groups", "group_score", "renormalise", "scale", "bias")])


@pytest.mark.parametrize("kw,args,needle", [
    (dict(score=2), {}, "gate score 2"), (dict(score=-1), {}, "gate score"), (dict(groups=0), {}, "gate groups 0"),
    (dict(groups=65), {}, "gate groups 65"), (dict(groups=3), {}, "a divisor of routed 64"),
    (dict(groups=4, kept_groups=5), {}, "kept groups 5"), (dict(kept_groups=0), {}, "kept groups 0"),
    (dict(group_score=2), {}, "group score 2"), (dict(scale=0.0), {}, "scale"), (dict(scale=float("nan")), {}, "scale"),
    (dict(scale=float("inf")), {}, "scale"), (dict(bias=18), {}, "bias must be"),
    (dict(groups=8, kept_groups=1), dict(topk=9), "8 experts of the kept groups"), ({}, dict(topk=0), "topk 0"),
    ({}, dict(topk=32), "topk 32"), ({}, dict(rows=0), "rows 0"), ({}, dict(rows=-1), "rows -1"),
    ({}, dict(rows=(1 << 24) + 1), "outside 1..16777216"),
    ({}, dict(routed=0), "routed 0"), ({}, dict(routed=1025, stride=2000), "routed 1025"), ({}, dict(type=3), "logits type 3"),
    ({}, dict(stride=63), "stride 63"), ({}, dict(shared=2), "shared 2"), ({}, dict(logits=18), "aligned"),
    ({}, dict(logits=17, type=0), "aligned"), ({}, dict(picks=17), "aligned"), ({}, dict(logits=None), "null"),
    ({}, dict(weights=None), "null"),
])
def test_route_gate_refuses(kw, args, needle):
    import gfr_moe
    L = gfr_moe.lib()
    a = dict(logits=16, type=2, stride=64, rows=4, routed=64, topk=4, shared=1, picks=16, weights=16)   # never read
    a.update(args)
    st = gate(gfr_moe, **kw)
    rc = L.gfr_route_gate(None, a["logits"], a["type"], a["stride"], a["rows"], a["routed"], a["topk"], st,
                          a["shared"], a["picks"], a["weights"])
    assert rc == gfr_moe.GFR_EINVAL and needle in L.gfr_last_error().decode()


def test_null_gate_and_layer():
    import gfr_moe
    L = gfr_moe.lib()
    assert L.gfr_route_gate(None, 16, 2, 64, 4, 64, 4, None, 1, 16, 16) == gfr_moe.GFR_EINVAL
    st = gate(gfr_moe)
    assert L.gfr_moe_set_gate(None, st) == gfr_moe.GFR_EINVAL
    assert L.gfr_moe_run_bf16(None, None, None, None, None, None, 1) == gfr_moe.GFR_EINVAL
    assert L.gfr_moe_run_router_bf16(None, None, None, None, None, None, 1) == gfr_moe.GFR_EINVAL
    assert L.gfr_dense_run(None, None) == gfr_moe.GFR_EINVAL


@pytest.mark.parametrize("kw,needle", [
    (dict(x=None), "null"), (dict(w=None), "null"), (dict(out=None), "null"), (dict(rows=0), "rows 0"), (dict(n=0), "n 0"),
    (dict(k=0), "k 0"), (dict(rows=-4), "rows -4"), (dict(k=1 << 25, x_stride=1 << 25, w_stride=1 << 25), "outside"),
    (dict(type=2), "type 2"), (dict(type=-1), "type -1"), (dict(out_type=1), "x's type or fp32"),
    (dict(bias=16, bias_type=1), "x's type or fp32"), (dict(residual=16, residual_type=1), "x's type or fp32"),
    (dict(gated=2), "gated 2"), (dict(act=5), "activation 5"), (dict(act=-1), "activation"), (dict(limit=-1.0, gated=1), "limit"),
    (dict(limit=float("nan"), gated=1), "limit"), (dict(limit=1.0), "gated form's"), (dict(x_stride=31), "strides of x 31"),
    (dict(w_stride=0), "w 0"), (dict(out_stride=15), "out 15"), (dict(residual=16, residual_stride=15), "residual 15"),
    (dict(x_stride=(1 << 31) + 1), "2^31"), (dict(x=17), "aligned"), (dict(w=33), "aligned"), (dict(out=17), "aligned"),
    (dict(out=18, out_type=2), "aligned"), (dict(bias=18, bias_type=2), "aligned"), (dict(residual=18, residual_type=2), "aligned"),
    (dict(rows=1 << 24, n=1 << 24, out_stride=1 << 24), "too many tiles"),
])
def test_dense_refuses(kw, needle):
    import gfr_moe
    a = dict(rows=4, n=16, k=32, type=0, x=16, x_stride=32, w=16, w_stride=32, out=16, out_stride=16, residual_stride=16)
    a.update(kw)
    names = ("rows n k type x x_stride w w_stride gated act limit bias_type bias residual_type out_type residual "
             "residual_stride out out_stride").split()
    st = gfr_moe._DENSE.pack(*[a.get(n) or 0 for n in names])
    L = gfr_moe.lib()
    assert L.gfr_dense_run(None, st) == gfr_moe.GFR_EINVAL
    assert needle in L.gfr_last_error().decode()


def test_python_refusals():
    """The wrappers' own checks, on host tensors: shapes, types and columns that are not neighbours."""
    import torch
    import gfr_moe
    x, w = torch.zeros(4, 32, dtype=torch.bfloat16), torch.zeros(16, 32, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="same 16-bit type"):
        gfr_moe.dense(x, w.half())
    with pytest.raises(ValueError, match="same 16-bit type"):
        gfr_moe.dense(x, w[:, :16])
    with pytest.raises(ValueError, match="activation"):
        gfr_moe.dense(x, w, activation="tanh")
    with pytest.raises(ValueError, match="even number of rows"):
        gfr_moe.dense_gated(x, w[:15])
    with pytest.raises(ValueError, match="neighbours"):
        gfr_moe._row_stride(x.t())
    with pytest.raises(ValueError, match="gate logits"):
        gfr_moe.route_gate(torch.zeros(2, 8, dtype=torch.float64), gfr_moe.Gate(), 2)
    with pytest.raises(ValueError, match="gate: score"):
        gfr_moe.Gate(score="max").pack(8)
    with pytest.raises(ValueError, match="group score"):
        gfr_moe.Gate(group_score="sum").pack(8)
    with pytest.raises(ValueError, match="gate bias"):
        gfr_moe.Gate(bias=torch.zeros(7)).pack(8)
    with pytest.raises(ValueError, match="bf16"):
        gfr_moe.Bf16SharedWeights(w, w).struct()
