"""The choice of the 16-bit products' kernels (gfr_dense_form; no GPU needed)."""
import pytest

import dense_sizes


def test_every_form_has_sizes():
    assert set(dense_sizes.SIZES) == {(f, g) for f in [*range(9), *range(16, 24)] for g in (False, True)}


@pytest.mark.parametrize("form,gated", list(dense_sizes.SIZES))
def test_sizes_take_their_form(form, gated):
    import gfr_moe
    for rows, n, k in dense_sizes.SIZES[form, gated]:
        x = (1 << 40) + (2 if form >= 16 else 0)
        assert dense_sizes.form(gfr_moe, rows, n, k, gated, x=x) == form, (rows, n, k)


def test_alignment_of_either_operand():
    import gfr_moe
    args = (gfr_moe, 500, 4096, 512, False)
    assert dense_sizes.form(*args) < 16
    for kw in (dict(x=2), dict(w=8), dict(x_stride=516), dict(w_stride=513)):
        assert dense_sizes.form(*args, **kw) >= 16, kw


@pytest.mark.parametrize("rows,n,k", [(500, 4096, 512), (2000, 8192, 1024), (400, 5000, 1001)])
def test_far_rows_take_the_thin_forms(rows, n, k):
    """The tiles address a tile's rows in 32 bits: row strides of 2^22 and more take the other kernels."""
    import gfr_moe
    for gated in (False, True):
        for which in ("x_stride", "w_stride"):
            assert dense_sizes.form(gfr_moe, rows, n, k, gated, **{which: (1 << 22) - 8}) % 16 >= 5
            assert dense_sizes.form(gfr_moe, rows, n, k, gated, **{which: 1 << 22}) % 16 < 5


def test_refusals_as_the_product():
    import gfr_moe
    L = gfr_moe.lib()
    assert L.gfr_dense_form(None) == gfr_moe.GFR_EINVAL
    assert dense_sizes.form(gfr_moe, 0, 16, 32, False) == gfr_moe.GFR_EINVAL and b"rows 0" in L.gfr_last_error()
    assert dense_sizes.form(gfr_moe, 4, 16, 32, False, x_stride=31) == gfr_moe.GFR_EINVAL


def shares_memory(a, b):
    """Whether two sets of rows ((address, bytes a row, pitch, rows) each) share a byte."""
    used = {r for i in range(a[3]) for r in range(a[0] + i * a[2], a[0] + i * a[2] + a[1])}
    return any(r in used for i in range(b[3]) for r in range(b[0] + i * b[2], b[0] + i * b[2] + b[1]))


def test_out_that_overlaps_an_operand_is_refused():
    """Rows of out, x, w, bias and residual at random addresses and strides in a small range, byte by byte: exactly those
    whose out shares a byte with an operand are refused, but for the residual that is out itself."""
    import random
    import gfr_moe
    L, rng = gfr_moe.lib(), random.Random(3)
    seen = {False: 0, True: 0}
    for _ in range(6000):
        rows, n, k, gated = rng.randint(1, 5), rng.randint(1, 6), rng.randint(1, 6), rng.randint(0, 1)
        otype, btype, rtype = (rng.choice([0, 2]) for _ in range(3))
        es, ws = {0: 2, 2: 4}, (1 + gated) * n
        at = lambda t: (1 << 20) + es[t] * rng.randint(0, 200)
        same = rng.random() < 0.4                                  # one row pitch, as slices of one buffer have
        pitch = 4 * rng.randint(12, 30)
        stride = lambda t, c: pitch // es[t] if same else c + rng.randint(0, 20)
        o = (at(otype), n * es[otype], stride(otype, n) * es[otype], rows)
        x = (at(0), k * 2, stride(0, k) * 2, rows)
        w = (at(0) + 2 * rng.choice([0, 1000]), k * 2, stride(0, k) * 2, ws)
        b = (at(btype), ws * es[btype], ws * es[btype], 1) if rng.random() < 0.3 else None
        r = (at(rtype), n * es[rtype], stride(rtype, n) * es[rtype], rows) if rng.random() < 0.6 else None
        if r and rng.random() < 0.3:
            r = o if rng.random() < 0.7 else (o[0], r[1], r[2], rows)
        in_place = bool(r) and r[0] == o[0] and rtype == otype and (rows == 1 or r[2] == o[2])
        if r and r[2] % es[rtype]:
            continue
        r_stride, r_at = (r[2] // es[rtype], r[0]) if r else (0, 0)
        if r and (r_stride < n or r_at % es[rtype]):
            continue
        if r:
            r = (r[0], n * es[rtype], r[2], rows)
        want = shares_memory(o, x) or shares_memory(o, w) or bool(b) and shares_memory(o, b) or (
            bool(r) and not in_place and shares_memory(o, r))
        st = gfr_moe._DENSE.pack(rows, n, k, 0, x[0], x[2] // 2, w[0], w[2] // 2, gated, 0, 0.0, btype, b[0] if b else 0, rtype,
                                 otype, r_at, r_stride, o[0], o[2] // es[otype])
        rc = L.gfr_dense_form(st)
        assert (rc < 0) == want, (o, x, w, b, r, rc, L.gfr_last_error())
        if want:
            assert b"out overlaps" in L.gfr_last_error()
        seen[want] += 1
    assert min(seen.values()) > 500, seen


@pytest.mark.parametrize("name,kw", [
    ("x", dict(out=(1 << 40) + 2)), ("x", dict(out=(1 << 40) + 31 * 64 + 62)), ("w", dict(out=(1 << 44) - 2)),
    ("bias", dict(bias=(1 << 50) + 30)), ("the residual", dict(residual=(1 << 50) + 2)),
    ("the residual", dict(residual=1 << 50, residual_stride=24)), ("the residual", dict(residual=1 << 50, residual_type=2)),
])
def test_run_refuses_overlaps(name, kw):
    """gfr_dense_run itself, on the host, before any launch."""
    import gfr_moe
    a = dict(rows=32, n=16, k=32, x=1 << 40, x_stride=32, w=1 << 44, w_stride=32, out=1 << 50, out_stride=16,
             residual_stride=16)
    a.update(kw)
    names = ("rows n k type x x_stride w w_stride gated act limit bias_type bias residual_type out_type residual "
             "residual_stride out out_stride").split()
    L = gfr_moe.lib()
    assert L.gfr_dense_run(None, gfr_moe._DENSE.pack(*[a.get(n) or 0 for n in names])) == gfr_moe.GFR_EINVAL
    assert f"out overlaps {name}" in L.gfr_last_error().decode()
