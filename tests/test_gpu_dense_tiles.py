"""The 16-bit products in every kernel that they have (dense_sizes.py), at addresses, strides and sizes where the kernels
differ. Formulas and tolerances: test_gpu_dense.py."""
import pytest
import torch

import dense_sizes
from test_gpu_dense import check, randn, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,n,k", [(384, 2560, 448), (500, 2064, 1000), (2048, 2064, 264), (4096, 4096, 136)])
@pytest.mark.parametrize("gated", [False, True])
def test_fp32_rows_at_16_bytes(gfr, rows, n, k, gated):
    """fp32 out and residual whose rows start 16 bytes past a multiple of 32 (every other one where the stride is odd in
    units of 16 bytes): eight columns are stored as two accesses of 16 bytes, aligned to no more."""
    x, w = randn(1, rows, k), randn(2, 2 * n if gated else n, k, scale=k ** -0.5)
    for start, pad in ((4, 4), (4, 0), (0, 4)):
        ob = torch.full((rows + 1, n + start + pad), -7.0, device="cuda")
        rb = torch.full((rows + 1, n + start + pad), float("nan"), device="cuda")
        o, r = ob[:rows, start:start + n], rb[:rows, start:start + n]
        r.copy_(randn(3, rows, n, dtype=torch.float32))
        f = gfr.dense_gated if gated else gfr.dense
        f(x, w, residual=r, out=o, activation="silu")
        check(o, reference(x, w, None, "silu", gated, None, r, torch.float32), f"start {start} pad {pad}")
        assert (ob[rows] == -7).all() and (ob[:, :start] == -7).all() and (ob[:, start + n:] == -7).all()


EVERY = [(f, g, *size) for (f, g), sizes in dense_sizes.SIZES.items() for size in sizes]


def beside(rows, columns, dtype, start, pad, fill):
    """A [rows, columns] slice of a wider buffer of `fill`, one row longer: (slice, buffer)."""
    buf = torch.full((rows + 1, start + columns + pad), fill, dtype=dtype, device="cuda")
    return buf[:rows, start:start + columns], buf


def operands(gfr, form, gated, rows, n, k, dtype):
    """x and w of that form, slices of buffers whose other values are NaN."""
    wide = -k % 8 + 16                                             # rows of 16-byte aligned addresses
    start, pad = (8, wide - 8) if form < 16 else (1, 2)
    x, _ = beside(rows, k, dtype, start, pad, float("nan"))
    w, _ = beside(2 * n if gated else n, k, dtype, start, pad, float("nan"))
    x.copy_(randn(1, rows, k, dtype=dtype))
    w.copy_(randn(2, w.shape[0], k, dtype=dtype, scale=k ** -0.5))
    taken = dense_sizes.form(gfr, rows, n, k, gated, x.data_ptr(), w.data_ptr(), x.stride(0), w.stride(0))
    assert taken == form, f"form {taken}"
    return x, w


@pytest.mark.parametrize("form,gated,rows,n,k", EVERY)
def test_slices_of_wider_buffers(gfr, form, gated, rows, n, k):
    """Both types, with and without each part of the epilogue, out of each type; NaN beside x and w enters no sum, and
    nothing is written beside out."""
    f = gfr.dense_gated if gated else gfr.dense
    for i, (dtype, act, bias, residual, f32, shift) in enumerate((
            (torch.bfloat16, "silu", None, torch.bfloat16, False, (8, 8)), (torch.float16, "gelu", torch.float16, None, True, (0, 8)),
            (torch.bfloat16, None, None, torch.float32, True, (4, 4)), (torch.float16, "relu", torch.float32, torch.float16, False, (1, 0)),
            (torch.bfloat16, None, None, None, False, (0, 0)), (torch.float16, "gelu_tanh", None, torch.float32, False, (8, 0)))):
        x, w = operands(gfr, form, gated, rows, n, k, dtype)
        odt = torch.float32 if f32 else dtype
        b = None if bias is None else randn(3, w.shape[0], dtype=bias)
        o, ob = beside(rows, n, odt, *shift, -7.0)
        r = None
        if residual is not None:
            r, _ = beside(rows, n, residual, *shift, float("nan"))
            r.copy_(randn(4, rows, n, dtype=residual))
        limit = 1.0 if gated and i % 2 else None
        f(x, w, bias=b, activation=act, residual=r, out=o, **({"limit": limit} if gated else {}))
        check(o, reference(x, w, b, act, gated, limit, r, odt), f"{dtype} {act}")
        start = shift[0]
        assert (ob[rows] == -7).all() and (ob[:, :start] == -7).all() and (ob[:, start + n:] == -7).all()


@pytest.mark.parametrize("form,gated,rows,n,k", EVERY)
def test_residual_in_place(gfr, form, gated, rows, n, k):
    """The residual that is out itself: the same bytes as into an out of its own."""
    x, w = operands(gfr, form, gated, rows, n, k, torch.bfloat16)
    f = gfr.dense_gated if gated else gfr.dense
    for dt in (torch.bfloat16, torch.float32):
        for act in (None, "silu"):
            h = randn(3, rows, n, dtype=dt)
            want = f(x, w, activation=act, residual=h, out_dtype=dt)
            f(x, w, activation=act, residual=h, out=h)
            torch.cuda.synchronize()
            assert torch.equal(h, want)


@pytest.mark.parametrize("far,rows,n,k", [("x", 407, 2730, 600), ("x", 386, 8384, 600), ("w", 1249, 816, 600), ("w", 4100, 816, 600)])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("off", [0, 1])
def test_far_apart_rows(gfr, far, rows, n, k, gated, off):
    """Row strides just below 2^22 elements (a tile's last row nearly 2^31 bytes behind its first: the tile kernels)
    and above (the thin kernels), of x and of w."""
    wrows = 2 * n if gated else n
    x, w = randn(1, rows, k), randn(2, wrows, k, scale=k ** -0.5)
    want = reference(x, w, None, "silu" if gated else None, gated, None, None, torch.float32)
    f = gfr.dense_gated if gated else gfr.dense
    for stride in ((1 << 22) - 8 + off, (1 << 22) + 8 + off):
        count = rows if far == "x" else wrows
        buf = torch.empty(count * stride + off, dtype=torch.bfloat16, device="cuda")
        view = torch.as_strided(buf, (count, k), (stride, 1), off)
        view.copy_(x if far == "x" else w)
        a, b = (view, w) if far == "x" else (x, view)
        taken = dense_sizes.form(gfr, rows, n, k, gated, a.data_ptr(), b.data_ptr(), a.stride(0), b.stride(0))
        assert (taken >= 16) == bool(off) and (taken % 16 < 5) == (stride > 1 << 22)
        check(f(a, b, out_dtype=torch.float32), want, f"{far} {stride} form {taken}")
        del buf, view, a, b


@pytest.mark.parametrize("rows", [1, 40, 300, 2000])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_activations_where_they_vanish(gfr, rows, gated, act):
    """Single products (exact in fp32) through each activation from -13 to 13, relative to the value itself, fp32 out.

    gelu = v / 2 erfc(t), t = -v / sqrt 2: erfc falls by the factor 1 - 2 t^2 e (t > 1) where t is off by a share e of it,
    here two roundings, 2^-23: v^2 2^-23; the rest within 2^-20. silu = v / (1 +
    exp(-v)): the exponential's argument is off by two roundings, |v| 2^-23; exp2, the sum, the quotient and a product (one
    unit each) within 2^-21. gelu_tanh the same with 2 z = 2 sqrt(2 / pi) (v + 0.044715 v^3) in the place of v, which takes
    seven roundings more: |2 z| 2^-21. Values below 2^-100 may be flushed."""
    v = torch.cat((torch.arange(-13 * 64, 13 * 64, device="cuda") / 64, torch.tensor([-0.001, 0.001, 0.0], device="cuda")))
    v = v.to(torch.float16)
    n, k = v.numel(), 64
    w = torch.zeros(2 * n if gated else n, k, dtype=torch.float16, device="cuda")
    x = torch.zeros(rows, k, dtype=torch.float16, device="cuda")
    x[:, 3] = 1
    w[:n, 3] = v
    if gated:
        w[n:, 3] = 1
    y = (gfr.dense_gated if gated else gfr.dense)(x, w, activation=act, out_dtype=torch.float32)
    torch.cuda.synchronize()
    d = v.double()
    if act == "gelu":
        want, rel = 0.5 * d * torch.special.erfc(-d / 2 ** 0.5), d * d * 2.0 ** -23 + 2.0 ** -20
    else:
        z = d if act == "silu" else 2 * (2 / torch.pi) ** 0.5 * (d + 0.044715 * d ** 3)
        want, rel = d / (1 + torch.exp(-z)), z.abs() * 2.0 ** (-23 if act == "silu" else -21) + 2.0 ** -21
    over = (y.double() - want).abs() - (rel * want.abs() + 2.0 ** -100)
    i = int(over.max(0).values.argmax())
    assert (over <= 0).all(), f"{act}({d[i].item()}): {y[0, i].item():.6g}, want {want[i].item():.6g}"
