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
