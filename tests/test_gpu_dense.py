"""The 16-bit products with their epilogue (gfr_dense_run, dense, dense_gated) against the formulas in 64 bits.

The tolerance of an element, counted before the first run: products of 16-bit values are exact in 32 bits; a sum of k of
them in any order is off by at most (k + 8) * 2^-23 * sum |x||w| (a unit of the sum a step, rounded or cut); the bias adds
one rounding. An activation has a slope of at most 1.13 (GELU's and SiLU's largest) and is evaluated within 2^-20 of its
argument's size (expf, erff within 2^-21, a product and a quotient); the gated form multiplies two such values. The
residual adds one rounding, and out's type half a step (eps / 2)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SLOPE, EVAL = 1.13, 2.0 ** -20
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def act64(v, act):
    if act == "relu":
        return v.clamp(min=0)
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v / math.sqrt(2)))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    if act == "silu":
        return v / (1 + torch.exp(-v))
    return v


def reference(x, w, bias, act, gated, limit, residual, out_dtype):
    """(values, the bound of their error) in 64 bits."""
    x64, w64 = x.double(), w.double()
    k = x.shape[1]
    y = x64 @ w64.t().contiguous()
    e = (k + 8) * 2.0 ** -23 * (x64.abs() @ w64.abs().t().contiguous())
    if bias is not None:
        y = y + bias.double()
        e = e + 2.0 ** -24 * y.abs() + e * 2.0 ** -20
    if gated:
        n = w.shape[0] // 2
        g, u, eg, eu = y[:, :n], y[:, n:], e[:, :n], e[:, n:]
        if limit:
            g, u = g.clamp(max=limit), u.clamp(-limit, limit)
        a = act64(g, act)
        ea = SLOPE * eg + EVAL * g.abs()
        y, e = a * u, ea * u.abs() + a.abs() * eu + ea * eu + 2.0 ** -23 * (a * u).abs()
    else:
        y, e = act64(y, act), (SLOPE * e + EVAL * y.abs() if act not in (None, "none", "relu") else e)
    if residual is not None:
        y = y + residual.double()
        e = e + 2.0 ** -23 * (y.abs() + residual.double().abs())
    return y, e + torch.finfo(out_dtype).eps / 2 * (y.abs() + e) + torch.finfo(out_dtype).smallest_normal


def check(out, want, what=""):
    y, e = want
    torch.cuda.synchronize()
    over = (out.double() - y).abs() - e
    assert torch.isfinite(out).all(), f"{what}: non-finite"
    assert (over <= 0).all(), (f"{what}: off by {(out.double() - y).abs().max().item():.3g}, allowed there "
                               f"{e.flatten()[over.argmax()].item():.3g} at {divmod(over.argmax().item(), out.shape[1])}")


def randn(seed, *shape, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def one(gfr, rows, n, k, dtype=torch.bfloat16, gated=False, act=None, bias=None, residual=None, out_dtype=None, limit=None,
        seed=0, what=""):
    x, w = randn(seed + 1, rows, k, dtype=dtype), randn(seed + 2, (2 if gated else 1) * n, k, dtype=dtype, scale=k ** -0.5)
    b = None if bias is None else randn(seed + 3, w.shape[0], dtype=bias)
    r = None if residual is None else randn(seed + 4, rows, n, dtype=residual)
    out_dtype = out_dtype or dtype
    if gated:
        y = gfr.dense_gated(x, w, bias=b, activation=act, limit=limit, residual=r, out_dtype=out_dtype)
    else:
        y = gfr.dense(x, w, bias=b, activation=act, residual=r, out_dtype=out_dtype)
    assert y.dtype is out_dtype and y.shape == (rows, n)
    check(y, reference(x, w, b, act, gated, limit, r, out_dtype), f"rows {rows} n {n} k {k} {what}")


ROWS = [1, 2, 5, 15, 16, 17, 31, 33, 48, 64, 65, 100, 127, 128, 129, 200, 257, 400]
KN = [(1, 1), (2, 3), (7, 16), (8, 17), (31, 64), (32, 33), (63, 130), (64, 64), (65, 1), (96, 257), (128, 96), (129, 48),
      (256, 512), (512, 260), (1000, 72), (1024, 31), (2048, 160), (1001, 207), (4104, 100)]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("gated", [False, True])
def test_dense_sizes(gfr, rows, gated):
    for i, (k, n) in enumerate(KN):
        dtype = (torch.bfloat16, torch.float16)[(i + rows) % 2]
        one(gfr, rows, n, k, dtype, gated, act="silu" if gated else None, out_dtype=torch.float32 if i % 3 == 0 else dtype,
            seed=rows * 100 + i)


@pytest.mark.parametrize("rows,n,k", [(3, 40, 72), (40, 96, 128), (300, 130, 256), (700, 520, 512)])
@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("gated", [False, True])
def test_dense_epilogues(gfr, rows, n, k, name, gated):
    """Every activation with bias and residual in either type, out in either type."""
    dt = TYPES[name]
    case = 0
    for act in (None, "relu", "gelu", "gelu_tanh", "silu"):
        for bias in (None, dt, torch.float32):
            for residual in (None, dt, torch.float32):
                case += 1
                one(gfr, rows, n, k, dt, gated, act, bias, residual, (dt, torch.float32)[case % 2],
                    limit=(None, 0.5)[case % 3 == 0] if gated else None, seed=case, what=f"{act} {bias} {residual}")


@pytest.mark.parametrize("rows,n,k", [(1, 4096, 1024), (4, 1000, 5120), (16, 2048, 2048), (32, 512, 4096), (64, 1536, 768),
                                      (129, 4096, 512), (256, 1024, 4096), (512, 768, 1280), (1000, 2064, 264),
                                      (2048, 512, 1024), (4096, 1280, 256), (3001, 1111, 320), (520, 2304, 11008)])
@pytest.mark.parametrize("gated", [False, True])
def test_dense_larger(gfr, rows, n, k, gated):
    """Sizes of layers, on every form the sizes choose."""
    one(gfr, rows, n, k, torch.bfloat16, gated, "silu" if gated else None, None if gated else torch.float32,
        None if gated else torch.bfloat16, seed=rows, limit=1.0 if gated else None)
    one(gfr, rows, n, k, torch.float16, gated, "gelu" if gated else None, seed=rows + 1, out_dtype=torch.float32)


@pytest.mark.parametrize("rows,n,k", [(1000, 2047, 1001), (2100, 2055, 999), (4100, 1031, 333), (2100, 2056, 1000),
                                      (4099, 4104, 200), (700, 5000, 1032), (3000, 3001, 63), (2500, 2600, 72), (2600, 2700, 8)])
@pytest.mark.parametrize("gated", [False, True])
def test_dense_large_odd(gfr, rows, n, k, gated):
    """The tiles' own edges: rows, columns and k that end inside a tile, a step and a chunk, on and off alignment."""
    one(gfr, rows, n, k, torch.bfloat16, gated, "silu" if gated else None, torch.bfloat16, None, seed=rows)
    one(gfr, rows, n, k, torch.float16, gated, "gelu_tanh", None, torch.float32, torch.float32, seed=rows + 1)


@pytest.mark.parametrize("rows,n,k,gated", [(200, 4100, 520, False), (300, 4100, 1000, False), (1100, 1030, 200, False),
                                            (200, 5128, 72, False), (500, 2063, 1001, False), (300, 5131, 999, False),
                                            (500, 1030, 1000, True), (300, 2060, 200, True), (1100, 517, 1003, True),
                                            (200, 2061, 999, True), (384, 2560, 448, True)])
def test_dense_middle_odd(gfr, rows, n, k, gated):
    """Sizes between the thin forms' and the large tiles', on and off alignment."""
    one(gfr, rows, n, k, torch.bfloat16, gated, "silu" if gated else None, torch.bfloat16, torch.bfloat16, seed=rows)
    one(gfr, rows, n, k, torch.float16, gated, "gelu_tanh", None, None, torch.float32, seed=rows + 1)


@pytest.mark.parametrize("rows", [1, 9, 70, 300])
@pytest.mark.parametrize("gated", [False, True])
def test_dense_strides_alignment_and_padding(gfr, rows, gated):
    """Slices of wider buffers at every alignment; what lies beside the slices (NaN) is neither used nor written."""
    n, k = 70, 136
    for pad, start, opad, ostart in ((8, 8, 4, 4), (1, 0, 1, 1), (3, 1, 0, 0), (8, 4, 2, 2), (120, 0, 58, 0), (5, 2, 4, 3)):
        for odt in (torch.bfloat16, torch.float32):
            wn = 2 * n if gated else n
            xb = torch.full((rows + 1, k + pad + start), float("nan"), dtype=torch.bfloat16, device="cuda")
            wb = torch.full((wn + 1, k + pad + start), float("nan"), dtype=torch.bfloat16, device="cuda")
            ob = torch.full((rows + 1, n + opad + ostart), -7.0, dtype=odt, device="cuda")
            rb = torch.full((rows + 1, n + opad + ostart), float("nan"), dtype=odt, device="cuda")
            x, w = xb[:rows, start:start + k], wb[:wn, start:start + k]
            o, r = ob[:rows, ostart:ostart + n], rb[:rows, ostart:ostart + n]
            x.copy_(randn(1, rows, k))
            w.copy_(randn(2, wn, k, scale=k ** -0.5))
            r.copy_(randn(3, rows, n, dtype=odt))
            f = gfr.dense_gated if gated else gfr.dense
            y = f(x, w, residual=r, out=o, activation="silu")
            assert y is o
            check(o, reference(x, w, None, "silu", gated, None, r, odt), f"pad {pad} start {start}")
            assert (ob[rows] == -7).all() and (ob[:, :ostart] == -7).all() and (ob[:, ostart + n:] == -7).all()


@pytest.mark.parametrize("rows,n,k", [(1, 100, 64), (20, 256, 512), (300, 512, 512), (600, 1024, 1024)])
def test_dense_residual_in_place(gfr, rows, n, k):
    x, w = randn(1, rows, k), randn(2, n, k, scale=k ** -0.5)
    for dt in (torch.bfloat16, torch.float32):
        h = randn(3, rows, n, dtype=dt)
        want = gfr.dense(x, w, residual=h, out_dtype=dt)
        gfr.dense(x, w, residual=h, out=h)
        torch.cuda.synchronize()
        assert torch.equal(h, want)


def test_dense_refuses_on_the_gpu(gfr):
    x, w = randn(1, 8, 64), randn(2, 64, 64)
    for kw, needle in ((dict(out=x), "must not be x or w"), (dict(out=w[:8]), "must not be x or w"),
                       (dict(out=torch.empty(8, 63, dtype=torch.bfloat16, device="cuda")), "want \\(8, 64\\)"),
                       (dict(residual=randn(3, 7, 64)), "residual"), (dict(residual=randn(3, 8, 64).cpu()), "current device"),
                       (dict(bias=randn(3, 65)), "bias"), (dict(bias=randn(3, 64).cpu()), "current device"),
                       (dict(out=torch.empty(8, 64, dtype=torch.bfloat16)), "current device"),
                       (dict(out=torch.empty(64, 8, dtype=torch.bfloat16, device="cuda").t()), "neighbours")):
        with pytest.raises(ValueError, match=needle):
            gfr.dense(x, w, **kw)
    for bad in ((x[:0], w), (x[:1].expand(8, 64), w), (x.float(), w.float())):
        with pytest.raises((gfr.GfrError, ValueError)):
            gfr.dense(*bad)
    for kw in (dict(out_dtype=torch.float16), dict(residual=randn(3, 8, 64, dtype=torch.float16)),
               dict(bias=randn(3, 64, dtype=torch.float16))):
        with pytest.raises(gfr.GfrError, match="x's type or fp32"):
            gfr.dense(x, w, **kw)
    with pytest.raises(gfr.GfrError, match="limit"):
        gfr.dense_gated(x, w, limit=-1.0)


@pytest.mark.parametrize("rows", [2, 40, 300])
def test_dense_special_values(gfr, rows):
    """Infinities and NaN stay in the rows and columns that they meet; fp16 results past its range are infinite."""
    n, k = 96, 256
    for dtype in (torch.bfloat16, torch.float16):
        x, w = randn(1, rows, k, dtype=dtype), randn(2, n, k, dtype=dtype, scale=k ** -0.5)
        x[1, 5], w[7, 9] = float("inf"), float("nan")
        y = gfr.dense(x, w, out_dtype=torch.float32)
        torch.cuda.synchronize()
        finite = torch.ones(rows, n, dtype=torch.bool, device="cuda")
        finite[1], finite[:, 7] = False, False
        assert torch.isfinite(y[finite]).all() and torch.isnan(y[:, 7]).all()
        cols = [c for c in range(n) if c != 7]
        assert torch.equal(y[1, cols] > 0, w[cols, 5] > 0) and torch.isinf(y[1, cols]).all()
    # the limit bounds numbers and infinities, and keeps a NaN
    x, w = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda"), torch.zeros(2 * n, k, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = 1
    w[:n, 0], w[n:, 0] = float("inf"), float("-inf")
    w[3, 0], w[n + 4, 0] = float("nan"), float("nan")
    y = gfr.dense_gated(x, w, limit=2.0, out_dtype=torch.float32)
    torch.cuda.synchronize()
    want = -2.0 * 2.0 / (1 + math.exp(-2.0))
    assert torch.isnan(y[:, 3:5]).all()
    rest = torch.cat((y[:, :3], y[:, 5:]), 1).double()
    assert (rest - want).abs().max() <= 2.0 ** -18 * abs(want)
    big = torch.full((rows, k), 200.0, dtype=torch.float16, device="cuda")
    y = gfr.dense(big, torch.full((n, k), 8.0, dtype=torch.float16, device="cuda"))
    torch.cuda.synchronize()
    assert torch.isinf(y).all() and (y > 0).all()


def test_dense_offsets_past_32_bits(gfr):
    """Rows of x, w, residual and out more than 2^32 bytes behind the first."""
    rows, n, k, stride = 40, 130, 64, 1 << 26
    buf = torch.empty(n * stride, dtype=torch.bfloat16, device="cuda").view(n, stride)
    w, x, o, r = (buf[:n, :k], buf[:rows, 4096:4096 + k], buf[:rows, 8192:8192 + n], buf[:rows, 16384:16384 + n])
    w.copy_(randn(1, n, k, scale=k ** -0.5))
    x.copy_(randn(2, rows, k))
    r.copy_(randn(3, rows, n))
    gfr.dense(x, w, residual=r, out=o)
    check(o, reference(x.contiguous(), w.contiguous(), None, None, False, None, r.contiguous(), torch.bfloat16))


@pytest.mark.parametrize("rows,n,k", [(1, 512, 512), (24, 512, 1024), (300, 384, 512), (1100, 1024, 512)])
def test_dense_streams_graph_and_repeats(gfr, rows, n, k):
    """The same bytes on every call, on another stream, next to other calls and in a replayed graph."""
    x, w, d = randn(1, rows, k), randn(2, 2 * n, k, scale=2 * k ** -0.5), randn(3, k, n, scale=n ** -0.5)
    h = randn(4, rows, k)

    def mlp(x, h, stream=None):
        return gfr.dense(gfr.dense_gated(x, w, limit=10.0, stream=stream), d, residual=h, stream=stream)

    want = mlp(x, h)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [mlp(x, h, stream=s) for _ in range(2) for s in streams]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)
    xs, hs = x.clone(), h.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = mlp(xs, hs)
    for seed in range(4):
        xs.copy_(randn(20 + seed, rows, k))
        hs.copy_(randn(30 + seed, rows, k))
        eager = mlp(xs, hs)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
def test_mlp(gfr, name):
    """The two products together, as a dense layer's MLP: the activations' rounding to 16 bits (half a step, eps / 2)
    enters the second product next to the products' own bounds."""
    dt = TYPES[name]
    for rows, hidden, inter in ((1, 512, 1536), (7, 260, 100), (33, 512, 700), (300, 1024, 768), (1500, 512, 1024)):
        x, gu = randn(1, rows, hidden, dtype=dt), randn(2, 2 * inter, hidden, dtype=dt, scale=2 * hidden ** -0.5)
        down, h = randn(3, hidden, inter, dtype=dt, scale=inter ** -0.5), randn(4, rows, hidden, dtype=dt)
        y = gfr.dense(gfr.dense_gated(x, gu, limit=10.0), down, residual=h)
        a, ea = reference(x, gu, None, "silu", True, 10.0, None, dt)
        want, e = reference(a, down.double(), None, None, False, None, h, dt)
        e = e + ea @ down.double().abs().t().contiguous() * (1 + torch.finfo(dt).eps)
        check(y, (want, e), f"rows {rows}")
