"""The general router gate with several rows in a wave (windows of some thousand rows): what test_gpu_gate.py asks of few
rows, in every lane deal. Formulas and tolerances as there."""
import numpy as np
import pytest
import torch

from test_gpu_gate import ABS, REL, bias_of, logits_of, reference

pytestmark = pytest.mark.gpu

# routed, groups, kept, topk. launch_gate gives a row 16 lanes from 4096 rows on where these hold its choices in 8
# registers each, from 8192 where in 16; the others 32 lanes, the last two 64.
SHAPES = [
    (1, 1, 1, 1), (2, 2, 1, 1), (5, 1, 1, 5), (16, 1, 1, 15), (64, 1, 1, 4), (96, 3, 2, 6), (128, 8, 3, 9), (100, 4, 3, 15),
    (160, 8, 3, 6), (256, 8, 4, 8), (256, 1, 1, 12), (200, 5, 5, 8),
    (64, 32, 9, 7), (288, 8, 4, 8), (288, 9, 2, 31), (384, 2, 1, 10), (512, 16, 3, 20), (500, 4, 3, 16), (40, 1, 1, 31),
    (513, 1, 1, 8), (990, 33, 4, 20),
]
ROWS = 8192 + 3


def check(gfr, l, order, topk, score, bias, groups, kept, gs, renorm, scale=2.5, shared=True, close=False, what=""):
    """l: rows of which row r is a copy of row order[r]; each is compared with the 64-bit result of the row that it copies.
    close: rows whose group sums 64 bits cannot tell apart are left out."""
    E = l.shape[1]
    gate = gfr.Gate(score=score, bias=None if bias is None else torch.tensor(bias, dtype=torch.float32, device="cuda"),
                    groups=groups, kept_groups=kept, group_score=gs, renormalise=renorm, scale=scale)
    p, w = gfr.route_gate(l, gate, topk, shared=shared)
    base = l[:int(order.max()) + 1].float().cpu().numpy()
    undecided = []
    wp, ww = reference(base, topk, score, bias, groups, kept, gs, renorm, np.float32(scale), shared,
                       undecided if close else None)
    ok = torch.ones(len(base), dtype=torch.bool)
    ok[undecided] = False
    assert len(undecided) <= len(base) // 10
    ok = ok.cuda()[order]
    wp, ww = torch.from_numpy(wp).cuda()[order], torch.from_numpy(ww).cuda()[order]
    torch.cuda.synchronize()
    bad = ((p != wp).any(1) & ok).nonzero().flatten()
    assert not len(bad), (f"{what}: {len(bad)} rows; row {bad[0].item()} (of {order[bad[0]].item()}): picks "
                          f"{p[bad[0]].tolist()}, want {wp[bad[0]].tolist()}")
    over = (w.double() - ww).abs() - (REL * ww.abs() + ABS * scale)
    assert (over[ok] <= 0).all(), f"{what}: weight off by {(w.double() - ww).abs()[ok].max().item()}"


def copies(base, rows, seed):
    """(rows of base in a random order, base itself first, the order)"""
    g = torch.Generator().manual_seed(seed)
    order = torch.cat((torch.arange(base.shape[0]), torch.randint(base.shape[0], (rows - base.shape[0],), generator=g))).cuda()
    return base[order].contiguous(), order


@pytest.mark.parametrize("E,groups,kept,topk", SHAPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_shapes(gfr, E, groups, kept, topk, score):
    """Every deal, with and without a bias, both group values, all three types; neighbouring rows differ."""
    case = 0
    for bias in (False, True):
        for gs in ("max", "top2"):
            for dtype in (torch.float32, torch.bfloat16, torch.float16):
                case += 1
                l, order = copies(logits_of(61, E, 17 * E + case, dtype), (4096 if case % 2 else ROWS) + 5, case)
                check(gfr, l, order, topk, score, bias_of(E, E + case) if bias else None, groups, kept, gs, case % 3 > 0,
                      shared=case % 4 > 0, what=f"bias {bias} {gs} {dtype}")


def masked_rows(E, groups, topk):
    rng = np.random.default_rng(E + topk)
    l = (rng.standard_normal((40, E)) * 1.5).astype(np.float32)
    low = np.finfo(np.float32).min
    l[0] = -np.inf
    l[1] = np.nan
    l[2, :E - 1] = -np.inf
    l[3, rng.random(E) < 0.9] = -np.inf
    l[4, rng.random(E) < 0.9] = np.nan
    l[5] = low
    l[6, rng.random(E) < 0.5] = low
    l[7, :E // groups] = -np.inf
    l[8, E // 3] = np.inf
    l[9, [0, E // 2, E - 1]] = np.inf
    l[10] = np.inf
    l[11] = -np.inf
    l[11, [min(1, E - 1), max(E - 2, 0)]] = [-200.0, -201.0]
    l[12] = np.finfo(np.float32).max
    l[13] = -1e-42                                          # subnormal
    l[14] = rng.integers(-40, 40, E) * np.float32(1e-45)
    for r in range(15, 40):
        l[r, rng.random(E) < rng.random()] = rng.choice([-np.inf, np.nan])
    return l


@pytest.mark.parametrize("E,groups,kept,topk", [(64, 1, 1, 4), (256, 8, 4, 8), (96, 3, 2, 6), (160, 8, 3, 6), (288, 8, 4, 8),
                                                (512, 4, 1, 20), (64, 32, 9, 7)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("gs", ["max", "top2"])
def test_masks(gfr, E, groups, kept, topk, score, gs):
    """Masked rows, whole and in part, beside live ones in a wave; +-inf, the types' lowest values, subnormals; biases of
    -inf and NaN."""
    base = masked_rows(E, groups, topk)
    b = bias_of(E, 3)
    rng = np.random.default_rng(E)
    odd = b.copy()
    odd[rng.random(E) < 0.3] = -np.inf
    odd[rng.random(E) < 0.1] = np.nan
    for i, dtype in enumerate((torch.float32, torch.bfloat16, torch.float16)):
        t = torch.from_numpy(base).to(dtype)
        if dtype is not torch.float32:
            t = torch.where(torch.from_numpy(base == np.finfo(np.float32).min), torch.finfo(dtype).min, t)
        l, order = copies(t.cuda(), ROWS, i)
        for j, bias in enumerate((None, b, odd, np.full(E, -np.inf, np.float32))):
            check(gfr, l, order, topk, score, bias, groups, kept, gs, (i + j) % 2 == 0, 1.5,
                  what=f"{dtype} bias {None if bias is None else bias[:2]}")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("E,groups,kept,topk", [(64, 1, 1, 6), (256, 8, 4, 8), (288, 8, 3, 8), (40, 4, 2, 9), (128, 1, 1, 15)])
def test_ties(gfr, score, with_bias, E, groups, kept, topk):
    """Equal logits within a row and across the rows of a wave: the lower id and the lower group first."""
    rng = np.random.default_rng(E)
    base = rng.integers(-3, 4, (200, E)).astype(np.float32)
    base[0] = 0.0
    base[1] = np.where(np.arange(E) % 2, 0.0, -0.0)
    base[2] = rng.choice([-0.0, 0.0], E)
    base[3:9] = base[9]                                     # the same row several times in a wave
    bias = rng.choice([0.0, 0.25], E).astype(np.float32) if with_bias else None
    for gs in ("max", "top2"):
        for dtype in (torch.float32, torch.float16):
            l, order = copies(torch.from_numpy(base).to(dtype).cuda(), ROWS, 5)
            check(gfr, l, order, topk, score, bias, groups, kept, gs, True, what=f"{gs} {dtype}")


@pytest.mark.parametrize("E,groups,kept,topk", [(64, 1, 1, 6), (256, 8, 4, 8), (288, 8, 4, 8), (100, 1, 1, 15)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_choices_closer_than_32_bits(gfr, E, groups, kept, topk, score):
    """Choices whose order 32-bit scores would lose, a fifth of the rows (a wave has rows in doubt beside certain ones);
    group sums closer than 64 bits hold are left out, as for few rows."""
    rng = np.random.default_rng(E + topk)
    base = (rng.standard_normal((150, E)) * 1.5).astype(np.float32)
    for r in range(0, 150, 5):
        at = np.float32(rng.uniform(-1, 6))
        base[r] = at + rng.permutation(E).astype(np.float32) * np.spacing(at) * rng.integers(1, 4)
    l, order = copies(torch.from_numpy(base).cuda(), ROWS, 2)
    for bias in (None, np.zeros(E, np.float32), np.full(E, 0.75, np.float32)):
        for gs in ("max", "top2"):
            check(gfr, l, order, topk, score, bias, groups, kept, gs, True, close=True, what=f"{gs} bias {bias is not None}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("E,groups,kept,topk", [(64, 1, 1, 4), (256, 8, 4, 8), (288, 8, 4, 8)])
def test_strides(gfr, dtype, E, groups, kept, topk):
    """Slices of wider buffers at odd strides and starts; values beside the slice are not used."""
    for pad, start in ((1, 1), (3, 5), (64, 4), (7, 0)):
        base = logits_of(50, E, E + pad, dtype)
        rows, order = copies(base, ROWS, pad)
        buf = torch.full((ROWS, E + pad + start), float("inf"), dtype=dtype, device="cuda")
        buf[:, :start] = float("nan")
        view = buf[:, start:start + E]
        view.copy_(rows)
        check(gfr, view, order, topk, "softmax", bias_of(E, 1), groups, kept, "top2", True, what=f"pad {pad} start {start}")


@pytest.mark.parametrize("E,groups,kept,topk", [(64, 1, 1, 4), (256, 8, 4, 8), (288, 8, 4, 8)])
def test_windows_of_a_softmax_gate(gfr, E, groups, kept, topk):
    """The picks of a row do not depend on its window; a softmax's weights may, in their last bits: its sum is taken in
    the order of the window's lane deal. (Both sides within the bound of the weights.)"""
    l = logits_of(ROWS, E, 3)
    for bias in (None, torch.from_numpy(bias_of(E, 2)).cuda()):
        gate = gfr.Gate(score="softmax", bias=bias, groups=groups, kept_groups=kept, renormalise=False)
        p, w = gfr.route_gate(l, gate, topk)
        for at in (0, 4000, ROWS - 77):
            pt, wt = gfr.route_gate(l[at:at + 77], gate, topk)
            assert torch.equal(p[at:at + 77], pt)
            assert ((w[at:at + 77] - wt).abs() <= 2 * REL * wt).all()
