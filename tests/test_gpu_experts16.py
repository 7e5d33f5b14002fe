"""The 16-bit routed experts (gfr_experts16_run, experts16) against the formulas in 64 bits.

The tolerance of an element, counted before the first run: the products' sums as in test_gpu_dense.py, (k + 8) * 2^-23 *
sum |x||w| in any order; the activation's slope of at most 1.13 and its evaluation within 2^-20; the activations are the sum
of two 16-bit values, of which the second is off by half a step of what the first left: eps^2 / 4, and with fp16 by half of
its least value, 2^-25. Weights and the slots' sum: (slots + 2) * 2^-24. The residual adds one rounding, out's type half a
step."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

SLOPE, EVAL = 1.13, 2.0 ** -20
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def act64(v, act):
    if act == "relu":
        return v.clamp(min=0)
    if act == "gelu":
        return v * torch.special.ndtr(v)
    if act == "gelu_tanh":
        return v * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3))
    return v * torch.sigmoid(v) if act == "silu" else v


def reference(x, ex, picks, weights, act="silu", limit=None, residual=None):
    """(values, the bound of their error) in 64 bits."""
    E, H, I = ex.down.shape
    rows, slots = picks.shape
    y = torch.zeros((rows, H), dtype=torch.float64, device=x.device)
    size, e = torch.zeros_like(y), torch.zeros_like(y)
    half = torch.finfo(x.dtype).eps / 2
    for n in sorted(set(picks.flatten().tolist())):
        if n < 0 or n >= E:
            continue
        r, s = torch.where(picks == n)
        x64, w64, d64 = x[r].double(), ex.gu[n].double(), ex.down[n].double()
        gu, e_gu = x64 @ w64.t().contiguous(), (H + 8) * 2.0 ** -23 * (x64.abs() @ w64.abs().t().contiguous())
        g, u, eg, eu = gu[:, :I], gu[:, I:], e_gu[:, :I], e_gu[:, I:]
        if limit:
            g, u = g.clamp(max=limit), u.clamp(-limit, limit)
        a = act64(g, act)
        ea = SLOPE * eg + EVAL * g.abs()
        a, ea = a * u, ea * u.abs() + a.abs() * eu + ea * eu + 2.0 ** -23 * (a * u).abs()
        ea = ea + half * half * (a.abs() + ea) + (2.0 ** -25 if x.dtype is torch.float16 else 0.0)
        part = a @ d64.t().contiguous()
        mag = a.abs() @ d64.abs().t().contiguous()
        ep = ea @ d64.abs().t().contiguous() * (1 + 2.0 ** -10) + (2 * I + 16) * 2.0 ** -23 * mag   # (two products a weight)
        w = weights[r, s].double().unsqueeze(1)
        y.index_add_(0, r, part * w)
        e.index_add_(0, r, ep * w.abs())
        size.index_add_(0, r, (part * w).abs())
    e = e + (slots + 2) * 2.0 ** -24 * size
    if residual is not None:
        y = y + residual.double()
        e = e + 2.0 ** -23 * (y.abs() + residual.double().abs())
    return y, e


def check(out, want, what=""):
    y, e = want
    torch.cuda.synchronize()
    bound = e + torch.finfo(out.dtype).eps / 2 * (y.abs() + e) + torch.finfo(out.dtype).smallest_normal
    off = (out.double() - y).abs()
    assert torch.isfinite(out).all(), f"{what}: non-finite"
    at = (off - bound).flatten().argmax()
    assert (off <= bound).all(), f"{what}: off by {off.flatten()[at].item():.3g}, allowed {bound.flatten()[at].item():.3g}"


def randn(seed, *shape, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def stack(gfr, seed, E, H, I, dtype=torch.bfloat16):
    return gfr.Experts16(randn(seed, E, 2 * I, H, dtype=dtype, scale=2 * H ** -0.5), randn(seed + 1, E, H, I, dtype=dtype, scale=I ** -0.5))


def routing(seed, rows, slots, E, kind="any"):
    """"any": distinct picks where there are as many experts; "one": all the same expert; "holes": a third -1, some past the
    end; "repeats": the same expert twice in a row."""
    g = torch.Generator().manual_seed(seed)
    picks = torch.rand((rows, max(E, slots)), generator=g).argsort(1)[:, :slots] % E
    if kind == "one":
        picks[:] = E // 2
    if kind == "holes":
        hole = torch.rand((rows, slots), generator=g)
        picks[hole < 0.3] = -1
        picks[hole > 0.9] = E + 3
        picks[rows // 2:rows // 2 + 1] = -7
    if kind == "repeats":
        picks[:, slots // 2:] = picks[:, :1]
    weights = torch.rand((rows, slots), generator=g) - 0.2
    return picks.int().cuda(), weights.cuda()


SIZES = [(1, 1), (2, 3), (7, 8), (8, 16), (33, 17), (64, 64), (65, 63), (100, 31), (128, 96), (256, 128), (512, 260),
         (1000, 72), (1001, 333), (2048, 512), (600, 1032), (4104, 40)]


@pytest.mark.parametrize("hidden,inter", SIZES)
def test_experts16(gfr, hidden, inter):
    """Every size with several windows, numbers of experts, ways of routing, types and activations, drawn from it."""
    rng = random.Random(hidden * 10007 + inter)
    for rows in [1, 2, 5, 15, 16, 17, 33, 64, 65, 100, 150]:
        dtype = TYPES[rng.choice(list(TYPES))]
        E, slots = rng.choice([1, 2, 5, 12, 40]), rng.choice([1, 2, 3, 8, 9])
        kind = rng.choice(["any", "any", "one", "holes", "repeats"])
        x, ex = randn(rows, rows, hidden, dtype=dtype), stack(gfr, hidden + rows, E, hidden, inter, dtype)
        picks, weights = routing(rows, rows, slots, E, kind)
        act, limit = rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu", None]), rng.choice([None, 1.0])
        residual = rng.choice([None, randn(rows + 1, rows, hidden, dtype=rng.choice([dtype, torch.float32]))])
        out_dtype = rng.choice([None, torch.float32])
        y = gfr.experts16(x, ex, picks, weights, activation=act, limit=limit, residual=residual, out_dtype=out_dtype)
        assert y.dtype is (out_dtype or dtype) and y.shape == (rows, hidden)
        check(y, reference(x, ex, picks, weights, act, limit, residual), f"rows {rows} experts {E} slots {slots} {kind} {dtype} {act}")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows", [1, 3, 16, 17, 40, 130])
def test_rows_by_themselves(gfr, rows, dtype):
    """A row gives the same bits alone and in any window, whoever shares its experts; a row of NaN or with picks of an expert
    whose weights are NaN leaves the others as they are; rows without picks get their residual, or zeros."""
    H, I, E, slots, dt = 520, 200, 12, 4, TYPES[dtype]
    x, ex = randn(1, rows, H, dtype=dt), stack(gfr, 2, E, H, I, dt)
    ex.gu[E - 1], ex.down[E - 1] = torch.nan, torch.nan
    picks, weights = routing(3, rows, slots, E - 1)
    r = randn(4, rows, H, dtype=dt)
    y = gfr.experts16(x, ex, picks, weights, residual=r)
    for n in {0, rows // 2, rows - 1}:
        assert torch.equal(gfr.experts16(x[n:n + 1], ex, picks[n:n + 1], weights[n:n + 1], residual=r[n:n + 1])[0], y[n])
    if rows > 2:
        x2, p2 = x.clone(), picks.clone()
        x2[1] = torch.nan
        p2[2, 1] = E - 1
        p2[0] = -1
        y2 = gfr.experts16(x2, ex, p2, weights, residual=r)
        assert torch.equal(y2[3:], y[3:]) and torch.equal(y2[0], r[0])
        assert torch.isnan(y2[1]).all() and torch.isnan(y2[2]).all()
        assert not gfr.experts16(x2, ex, p2, weights)[0].any()
    assert torch.equal(gfr.experts16(x, ex, torch.full_like(picks, -1), weights, residual=r), r)


@pytest.mark.parametrize("hidden,inter", [(64, 64), (129, 33), (1000, 104)])
def test_slices_in_place(gfr, hidden, inter):
    """Weights, rows, residual and out that are slices, at odd addresses, of buffers full of NaN: the same bits, and what lies
    between stays as it was; in the residual's place."""
    for rows in (1, 20, 70):
        E, slots, dt = 9, 3, torch.bfloat16
        x, ex, (picks, weights) = randn(1, rows, hidden), stack(gfr, 2, E, hidden, inter), routing(3, rows, slots, E)
        r = randn(4, rows, hidden, dtype=torch.float32)
        y = gfr.experts16(x, ex, picks, weights, residual=r, out_dtype=torch.float32)

        def slice_of(t, off, pad):
            wide = torch.full((*t.shape[:-1], t.shape[-1] + off + pad), torch.nan, dtype=t.dtype, device="cuda")
            wide[..., off:off + t.shape[-1]] = t
            return wide, wide[..., off:off + t.shape[-1]]

        more = torch.full((E, 2 * inter + 3, hidden + 5), torch.nan, dtype=dt, device="cuda")
        gu = more[:, 1:1 + 2 * inter, 3:3 + hidden]
        gu.copy_(ex.gu)
        rw, rs = slice_of(r, 5, 3)
        got = gfr.experts16(slice_of(x, 1, 2)[1], gfr.Experts16(gu, slice_of(ex.down, 3, 1)[1]), picks, weights, residual=rs, out=rs)
        torch.cuda.synchronize()
        assert got is rs and torch.equal(rs, y)
        assert torch.isnan(rw[:, :5]).all() and torch.isnan(rw[:, hidden + 5:]).all()


def test_far_weights(gfr):
    """Experts and rows whose elements' offsets pass 2^31 and 2^32 bytes."""
    H, I, E = 136, 72, 4
    space = torch.empty(int(3.6e9), dtype=torch.bfloat16, device="cuda")
    ex = stack(gfr, 1, E, H, I)
    gu = space.as_strided((E, 2 * I, H), (1 << 30, 1 << 20, 1))
    down = space[1000:].as_strided((E, H, I), ((1 << 30) + 8, 1 << 21, 1))
    gu.copy_(ex.gu)
    down.copy_(ex.down)
    x, (picks, weights) = randn(3, 7, H), routing(4, 7, 2, E)
    want = gfr.experts16(x, ex, picks, weights)
    assert torch.equal(gfr.experts16(x, gfr.Experts16(gu, down), picks, weights), want)


def test_long_windows(gfr):
    """Hundreds of members an expert: many passes, the last of one."""
    for rows, slots, E in ((193, 2, 3), (1025, 1, 1), (4096, 8, 20)):
        H, I = 136, 80
        x, ex, (picks, weights) = randn(1, rows, H), stack(gfr, 2, E, H, I), routing(3, rows, slots, E)
        check(gfr.experts16(x, ex, picks, weights), reference(x, ex, picks, weights), f"rows {rows}")


def test_fp16_range(gfr):
    """Activations between fp16's range and twice it (90000 = 65504 + 24496, both fp16 numbers) and those of its subnormals keep
    their size; beyond that they are infinite (infinity times one, and times a weight of zero)."""
    H = I = 64
    ex = gfr.Experts16(torch.zeros((1, 2 * I, H), dtype=torch.float16, device="cuda"),
                       torch.zeros((1, H, I), dtype=torch.float16, device="cuda"))
    ex.gu[0, :I, 0] = 1
    ex.gu[0, I:, 1] = 1
    ex.down[0].fill_diagonal_(1)
    x = torch.zeros((3, H), dtype=torch.float16, device="cuda")
    x[0, :2], x[1, :2], x[2, :2] = torch.tensor([300.0, 300.0]), torch.tensor([200.0, 300.0]), torch.tensor([2.0 ** -10, 2.0 ** -8])
    picks, weights = torch.zeros((3, 1), dtype=torch.int32, device="cuda"), torch.ones((3, 1), device="cuda")
    y = gfr.experts16(x, ex, picks, weights, activation="relu", out_dtype=torch.float32)
    assert (y[0] == 90000).all() and (y[1] == 60000).all() and (y[2] == 2.0 ** -18).all()
    x[0, 0] = 600.0
    assert not torch.isfinite(gfr.experts16(x, ex, picks, weights, activation="relu", out_dtype=torch.float32)[0]).any()


def test_stream_graph_and_overlap(gfr):
    """On a stream of the caller's; two calls at once on two streams; captured, with replays that follow picks and inputs."""
    H, I, E, rows, slots = 512, 256, 16, 12, 4
    x, ex, (picks, weights) = randn(1, rows, H), stack(gfr, 2, E, H, I), routing(3, rows, slots, E)
    want = gfr.experts16(x, ex, picks, weights)
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
    x2, (p2, w2) = randn(5, 3 * rows, H), routing(6, 3 * rows, slots, E)
    want2 = gfr.experts16(x2, ex, p2, w2)
    torch.cuda.synchronize()
    got = [[gfr.experts16(*a, stream=s) for s, a in zip(sides, ((x, ex, picks, weights), (x2, ex, p2, w2)))] for _ in range(10)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) and torch.equal(b, want2) for a, b in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = gfr.experts16(x, ex, picks, weights)
    for seed in (7, 8, 9):
        x.copy_(randn(seed, rows, H))
        p, w = routing(seed, rows, slots, E, "holes" if seed == 8 else "any")
        picks.copy_(p)
        weights.copy_(w)
        graph.replay()
        assert torch.equal(y, gfr.experts16(x, ex, picks, weights))
        torch.cuda.synchronize()


def test_python_refusals(gfr):
    x, ex, (picks, weights) = randn(1, 4, 64), stack(gfr, 2, 5, 64, 32), routing(3, 4, 2, 5)
    good = dict(x=x, experts=ex, picks=picks, weights=weights)
    for bad in (dict(x=x.half()), dict(x=x[:, :32]), dict(experts=gfr.Experts16(ex.gu[:, :63], ex.down)),
                dict(experts=gfr.Experts16(ex.gu, ex.down[:4])), dict(picks=picks.long()), dict(picks=picks[:3]),
                dict(weights=weights[:, :1]), dict(weights=weights.double()), dict(activation="tanh"), dict(picks=picks.cpu()),
                dict(residual=x[:, :32]), dict(out=x[:, :32]), dict(out=x.clone(), out_dtype=torch.float32),
                dict(experts=gfr.Experts16(ex.gu.transpose(1, 2).contiguous().transpose(1, 2), ex.down)),
                dict(picks=picks.t().contiguous().t(), weights=weights.t().contiguous().t())):
        with pytest.raises(ValueError):
            gfr.experts16(**{**good, **bad})
    for bad, needle in ((dict(out=x), "overlaps x"), (dict(residual=x.float().half()), "residual"), (dict(limit=-1.0), "limit"),
                        (dict(x=x[:0], picks=picks[:0], weights=weights[:0]), "rows 0"),
                        (dict(picks=picks[:, :0], weights=weights[:, :0]), "slots 0"),
                        (dict(out_dtype=torch.float16), "x's type or fp32")):
        with pytest.raises(gfr.GfrError, match=needle):
            gfr.experts16(**{**good, **bad})


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("hidden,inter", [(600, 1032), (1001, 333), (4096, 512), (2047, 1025)])
def test_again(gfr, hidden, inter, dtype):
    """The same bits from the same call, with the weights in the caches after the first."""
    E, slots, dt = 40, 9, TYPES[dtype]
    ex = stack(gfr, 2, E, hidden, inter, dt)
    for rows in (1, 5, 40):
        x, (picks, weights) = randn(rows, rows, hidden, dtype=dt), routing(3, rows, slots, E)
        y = gfr.experts16(x, ex, picks, weights, out_dtype=torch.float32)
        check(y, reference(x, ex, picks, weights), f"rows {rows}")
        for _ in range(8):
            assert torch.equal(gfr.experts16(x, ex, picks, weights, out_dtype=torch.float32), y)
