"""The norms around a block (gfr_block_norm_run, block_norm, norm) against the formulas in 64 bits.

The tolerance of an element, counted before the first run. A sum over a row's columns is at most 32 values a lane, 6 sums
over a wave and 16 over the waves, in 32 bits: off by at most 64 * 2^-24 of the sum of the values' sizes, of squares by that
share of itself (and their root's reciprocal by half of it; the mean, eps, root and quotient add less than the other half):
REL. A mean that is off by em moves every difference from it by em. Errors e of a norm's inputs change the root of the mean
square by at most the root mean square of e. The logistic function is within 2^-20. Each product and sum adds half a unit of
32 bits, and an output's type half a step (eps / 2)."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

REL, HALF = 64 * 2.0 ** -24, 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def norm64(z, e, p):
    """(values, bound of the error) of a Norm of z, itself off by at most e."""
    if p.kind == "layer":
        mean = z.mean(1, keepdim=True)
        e = e + e.mean(1, keepdim=True) + REL * z.abs().mean(1, keepdim=True) + 2 * HALF * (z.abs() + mean.abs())
        z = z - mean
    root = torch.sqrt((z * z).mean(1, keepdim=True) + p.eps)
    rel = REL + torch.sqrt((e * e).mean(1, keepdim=True)) / root
    w = torch.ones_like(z[0]) if p.weight is None else p.weight.double() + p.offset
    y = z / root * w
    ey = (e + 1.01 * rel * (z.abs() + e)) / root * w.abs() + 4 * HALF * y.abs()
    if p.bias is not None:
        y = y + p.bias.double()
        ey = ey + HALF * y.abs()
    return y, ey


def reference(x, residual, pre, post, gate, sigmoid, scale, residual_scale):
    z = x.double()
    e = torch.zeros_like(z)
    if post is not None:
        z, e = norm64(z, e, post)
    if gate is not None:
        g = gate.double() if gate.dim() == 2 else gate.double().unsqueeze(0)
        eg = torch.zeros_like(g)
        if sigmoid:
            g = torch.sigmoid(g)
            eg = 2.0 ** -20 * g
        e = e * g.abs() + eg * z.abs() + HALF * (z * g).abs()
        z = z * g
    h = scale * z
    e = abs(scale) * e + 2 * HALF * h.abs()
    if residual is not None:
        h = h + residual_scale * residual.double()
        e = e + 2 * HALF * (residual.double().abs() * abs(residual_scale) + h.abs())
    return (h, e), None if pre is None else norm64(h, e, pre)


def check(out, want, what):
    y, e = want
    torch.cuda.synchronize()
    bound = e + torch.finfo(out.dtype).eps / 2 * (y.abs() + e) + torch.finfo(out.dtype).smallest_normal
    over = (out.double() - y).abs() - bound
    assert torch.isfinite(out).all(), f"{what}: not finite"
    assert (over <= 0).all(), f"{what}: off by {(out.double() - y).abs().flatten()[over.argmax()].item():.3g}, " \
                              f"allowed {bound.flatten()[over.argmax()].item():.3g}"


def randn(seed, *shape, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def made(gfr, seed, n, kind, weight, offset=0.0):
    return gfr.Norm(kind=kind, weight=None if weight is None else randn(seed, n, dtype=weight, scale=0.3) + 1 - offset,
                    bias=randn(seed + 1, n, dtype=weight, scale=0.2) if weight is not None and kind == "layer" else None,
                    eps=1e-5, offset=offset)


NS = [1, 2, 7, 8, 9, 31, 127, 128, 129, 255, 512, 513, 1000, 1001, 2048, 2049, 4096, 4100, 5120, 8191, 8192, 8193, 12288, 16384,
      16385, 32767, 32768]


@pytest.mark.parametrize("n", NS)
def test_block_norm(gfr, n):
    """Every width with several windows, types, kinds of norm and gates, drawn from the width."""
    rng = random.Random(n)
    for rows in [1, 2, 3, 15, 16, 17, 33, 130]:
        xt, rt, ot, wt = [rng.choice(TYPES) for _ in range(4)]
        x = randn(n + rows, rows, n, dtype=xt)
        residual = rng.choice([None, randn(n + rows + 1, rows, n, dtype=rt, scale=2.0)])
        gate = rng.choice([None, (n,), (rows, 1), (1, n), (rows, n), (1, 1)])
        gate = None if gate is None else randn(n + rows + 2, *gate, dtype=rng.choice(TYPES))
        sigmoid = gate is not None and rng.random() < 0.5
        pre = made(gfr, n + 3, n, rng.choice(["rms", "layer"]), rng.choice([wt, None]), rng.choice([0.0, 1.0]))
        post = rng.choice([None, made(gfr, n + 5, n, rng.choice(["rms", "layer"]), wt)])
        scale, residual_scale = rng.choice([1.0, 0.22]), rng.choice([1.0, 0.9])
        h, y = gfr.block_norm(x, residual, pre=pre, post=post, gate=gate, gate_activation="sigmoid" if sigmoid else None,
                              scale=scale, residual_scale=residual_scale, out_dtype=ot)
        want = reference(x, residual, pre, post, gate, sigmoid, scale, residual_scale)
        assert h.dtype is (x if residual is None else residual).dtype and y.dtype is ot and h.shape == y.shape == (rows, n)
        what = f"rows {rows} n {n} post {post is not None} gate {None if gate is None else tuple(gate.shape)}"
        check(h, want[0], what + " h")
        check(y, want[1], what + " y")


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [64, 128, 129, 576, 5120, 9000])
def test_norm_alone(gfr, n, dtype, kind):
    """The norm of heads and rows, without the stream; in place; and with h alone (no pre)."""
    x = randn(n, 300, n, dtype=dtype)
    p = made(gfr, n, n, kind, dtype)
    want = norm64(x.double(), torch.zeros_like(x, dtype=torch.float64), p)
    y = gfr.norm(x, p)
    assert y.dtype is dtype
    check(y, want, f"n {n}")
    h, none = gfr.block_norm(x, x, scale=0.5)
    assert none is None
    check(h, ((x.double() * 1.5), 4 * HALF * x.double().abs()), "h alone")
    assert gfr.norm(x, p, out=x) is x and torch.equal(x, y)


@pytest.mark.parametrize("n", [8, 129, 1001, 4096, 9000])
def test_slices_in_place(gfr, n):
    """Rows that are slices of wider buffers full of NaN, at odd addresses, with h in the residual's place: the same values
    as from tensors of their own, and what lies between the rows stays as it was."""
    for rows in (1, 5, 40):
        def slice_of(t, off, pad):
            wide = torch.full((rows, n + off + pad), float("nan"), dtype=t.dtype, device="cuda")
            wide[:, off:off + n] = t
            return wide, wide[:, off:off + n]

        x, r, g = randn(n, rows, n), randn(n + 1, rows, n, dtype=torch.float32), randn(n + 2, rows, n, dtype=torch.float16)
        pre, post = made(gfr, n, n, "rms", torch.float32), made(gfr, n + 2, n, "layer", torch.bfloat16)
        h, y = gfr.block_norm(x, r, pre=pre, post=post, gate=g, scale=0.3)
        (_, xs), (rw, rs), (_, gs) = slice_of(x, 1, 3), slice_of(r, 3, 2), slice_of(g, 5, 1)
        ow, os = slice_of(torch.zeros_like(x), 3, 7)
        h2, y2 = gfr.block_norm(xs, rs, pre=pre, post=post, gate=gs, scale=0.3, h=rs, out=os)
        torch.cuda.synchronize()
        assert h2 is rs and torch.equal(rs, h) and torch.equal(os, y)
        assert torch.isnan(rw[:, :3]).all() and torch.isnan(rw[:, n + 3:]).all()
        assert torch.isnan(ow[:, :3]).all() and torch.isnan(ow[:, n + 3:]).all()
        # both outputs in the inputs' places
        x3, r3 = x.clone(), r.clone()
        h3, y3 = gfr.block_norm(x3, r3, pre=pre, post=post, gate=g, scale=0.3, h=r3, out=x3)
        assert torch.equal(r3, h) and torch.equal(x3, y)


@pytest.mark.parametrize("n", [100, 500, 3000, 9000, 20000])
def test_rows_by_themselves(gfr, n):
    """A row gives the same bits alone and in any window, and rows with NaN or infinities leave the others as they are."""
    x, r = randn(n, 200, n), randn(n + 1, 200, n)
    p, post = made(gfr, n, n, "rms", torch.bfloat16), made(gfr, n + 1, n, "layer", torch.float32)
    h, y = gfr.block_norm(x, r, pre=p, post=post)
    for rows in (1, 2, 17):
        h1, y1 = gfr.block_norm(x[30:30 + rows], r[30:30 + rows], pre=p, post=post)
        assert torch.equal(h1, h[30:30 + rows]) and torch.equal(y1, y[30:30 + rows])
    x[7, 3 % n], x[19, n - 1] = float("nan"), float("inf")
    h2, y2 = gfr.block_norm(x, r, pre=p, post=post)
    keep = [i for i in range(200) if i not in (7, 19)]
    assert torch.equal(h2[keep], h[keep]) and torch.equal(y2[keep], y[keep])
    assert torch.isnan(h2[7]).all() and torch.isnan(y2[7]).all()


@pytest.mark.parametrize("n", [64, 300, 3000, 20000])
def test_rows_without_the_stream(gfr, n):
    """The C interface with h NULL: the same y, of the residual and the scales all the same."""
    rows = 5
    x, r, p = randn(1, rows, n), randn(2, rows, n), made(gfr, 3, n, "rms", torch.bfloat16)
    for residual, scale, residual_scale in ((r, 0.5, 0.9), (None, 0.5, 1.0), (r, 1.0, 1.0), (None, 1.0, 1.0)):
        want = gfr.block_norm(x, residual, pre=p, scale=scale, residual_scale=residual_scale)[1]
        y = torch.empty_like(x)
        call = gfr._BLOCK_NORM.pack(rows, n, 0, 0, 0, 0, 0, 0, 0, scale, residual_scale, x.data_ptr(), n,
                                    0 if residual is None else residual.data_ptr(), n, 0, 0, 0, 0, y.data_ptr(), n,
                                    *gfr._NO_NORM, *p.fields(n, torch.cuda.current_device()))
        gfr._check(gfr.lib().gfr_block_norm_run(gfr._stream(), call))
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_gates_of_one_row(gfr):
    """A gate that torch expands to all rows or columns is the row or column itself."""
    n, rows = 300, 7
    x, column, row = randn(1, rows, n), randn(2, n), randn(3, rows, 1)
    for gate, same in ((column.expand(rows, n), column), (column.view(1, n), column), (row[:1].expand(rows, 1), row[:1]),
                       (row[0, 0], row[:1]), (row, row.expand(rows, n).contiguous())):
        assert torch.equal(gfr.block_norm(x, gate=gate)[0], gfr.block_norm(x, gate=same)[0])


def test_rows_of_one_value(gfr):
    """No variance: the layer norm's bias alone; rows of zeros: zeros."""
    for n in (1, 5, 128, 1000, 9000):
        x = torch.full((3, n), 2.5, dtype=torch.bfloat16, device="cuda")
        b = randn(n, n)
        y = gfr.norm(x, gfr.Norm("layer", weight=randn(n + 1, n), bias=b))
        assert torch.equal(y, b.expand(3, n))
        assert not gfr.norm(torch.zeros_like(x), gfr.Norm("rms", weight=randn(n + 1, n))).any()


def test_far_rows(gfr):
    """Rows whose elements' offsets pass 2^31 and 2^32 bytes."""
    n, stride = 1000, 1 << 30
    wide = torch.empty(2 * stride + stride // 2, dtype=torch.bfloat16, device="cuda")
    x = wide.as_strided((3, n), (stride, 1))
    x.copy_(randn(1, 3, n))
    p = made(gfr, 2, n, "rms", torch.float32)
    want = gfr.norm(x.contiguous(), p)
    assert torch.equal(gfr.norm(x, p), want)
    gfr.norm(x, p, out=x)
    assert torch.equal(x, want)


def test_stream_and_graph(gfr):
    """On a stream of the caller's, and captured: replays follow the inputs' values."""
    n = 4096
    x, r, p = randn(1, 9, n, dtype=torch.float32), randn(2, 9, n), made(gfr, 3, n, "rms", torch.bfloat16)
    want = gfr.block_norm(x, r, pre=p, out_dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = gfr.block_norm(x, r, pre=p, out_dtype=torch.bfloat16, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, y = gfr.block_norm(x, r, pre=p, out_dtype=torch.bfloat16)
    for seed in (5, 6, 7):
        x.copy_(randn(seed, 9, n, dtype=torch.float32))
        graph.replay()
        want = gfr.block_norm(x, r, pre=p, out_dtype=torch.bfloat16)
        torch.cuda.synchronize()
        assert torch.equal(h, want[0]) and torch.equal(y, want[1])


def test_python_refusals(gfr):
    x = randn(1, 4, 64)
    p = gfr.Norm("rms", weight=randn(2, 64))
    for bad in (dict(residual=x[:, :32]), dict(residual=x.double()), dict(gate=x[:3]), dict(gate=x.double()),
                dict(gate=x, gate_activation="tanh"), dict(pre=gfr.Norm("l2")), dict(pre=gfr.Norm("rms", weight=x[0, :32])),
                dict(pre=p, out=x[:, :32]), dict(pre=p, out_dtype=torch.float64), dict(out=x.clone()),
                dict(gate=randn(4, 128)[::2]), dict(gate=randn(4, 1, 128)[:, ::2]),
                dict(residual=x.cpu()), dict(pre=p, out=torch.empty_like(x), out_dtype=torch.float32), dict(gate=x.t())):
        with pytest.raises(ValueError):
            gfr.block_norm(x, **bad)
    wide = randn(3, 4, 128)
    for bad in (dict(h=wide[:, 8:72]), dict(h=wide[:, :64], pre=p, out=wide[:, 32:96])):
        with pytest.raises(gfr.GfrError, match="overlaps"):
            gfr.block_norm(wide[:, :64] if "pre" not in bad else x, **bad)
    with pytest.raises(gfr.GfrError, match="rows 0"):
        gfr.block_norm(x[:0], pre=p)


def test_more_rows_than_a_launch_holds(gfr):
    """2^21 + 3 rows of a workgroup each: the rows on both sides of the second launch's start."""
    rows, n = (1 << 21) + 3, 520
    x = torch.randn((rows, n), dtype=torch.bfloat16, device="cuda")
    p = made(gfr, 1, n, "rms", torch.bfloat16)
    y = gfr.norm(x, p)
    for part in (slice(0, 5), slice(rows - 7, rows)):
        assert torch.equal(y[part], gfr.norm(x[part].contiguous(), p))


def test_more_rows_with_the_stream(gfr):
    """The same with a residual, whose rows are a launch's by themselves."""
    rows, n = (1 << 21) + 3, 520
    x, r = [torch.randn((rows, n), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    p = made(gfr, 1, n, "rms", torch.bfloat16)
    h, y = gfr.block_norm(x, r, pre=p)
    for part in (slice(0, 5), slice(rows - 7, rows)):
        h1, y1 = gfr.block_norm(x[part].contiguous(), r[part].contiguous(), pre=p)
        assert torch.equal(h[part], h1) and torch.equal(y[part], y1)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("n", [9, 120, 127, 128, 129, 500, 512, 513, 1001, 4100, 5120, 8191, 8192])
def test_many_rows(gfr, n, kind):
    """The norm of more rows than the card holds at once: the bits of windows of few, and the formula's values, from slices
    between NaN, in place, with and without a weight and a bias, and rows with NaN or infinities by themselves."""
    least = -(-8 * 256 * 2048 // n)
    for rows, dtype, weight, out in ((least, torch.bfloat16, torch.float32, torch.bfloat16),
                                     (least + 77, torch.float16, torch.float16, torch.float32),
                                     (3 * least + 1, torch.float32, torch.bfloat16, torch.bfloat16),
                                     (least, torch.float16, None, torch.float16)):
        p = made(gfr, n, n, kind, weight, 1.0)
        wide = torch.full((rows, n + 5), float("nan"), dtype=dtype, device="cuda")
        x = wide[:, 3:3 + n]
        x.copy_(torch.randn((rows, n), dtype=torch.float32, device="cuda"))
        x[least // 2, n // 2], x[least // 3, 0] = float("nan"), float("inf")
        y = gfr.norm(x, p, out_dtype=out)
        few = torch.cat([gfr.norm(part, p, out_dtype=out) for part in x.split(min(8 * 256 * 2048 // n, least // 3 + 1))])
        keep = torch.ones(rows, dtype=torch.bool, device="cuda")
        keep[[least // 2, least // 3]] = False
        assert torch.equal(y[keep], few[keep]) and torch.isnan(y[least // 2]).all() and not torch.isfinite(y[least // 3]).all()
        some = x[rows - 200:].double()
        check(y[rows - 200:], norm64(some, torch.zeros_like(some), p), f"rows {rows} n {n}")
        if out is dtype:
            assert gfr.norm(x, p, out=x) is x and torch.equal(x[keep], y[keep])
            assert torch.isnan(wide[:, :3]).all() and torch.isnan(wide[:, 3 + n:]).all()
