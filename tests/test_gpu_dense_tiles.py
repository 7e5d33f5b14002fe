"""The 16-bit products' tile kernels at addresses, strides and sizes that the thin forms' tests do not reach them with.
Formulas and tolerances: test_gpu_dense.py."""
import pytest
import torch

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
