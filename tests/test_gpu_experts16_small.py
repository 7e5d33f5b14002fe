"""The 16-bit experts' activations between their products, from ordinary sizes to far below one: kept to 22 bits with fp16
weights, or to 2^-35 where that is more, and to 16 bits with bf16 ones.

The tolerance, counted before the first run: an activation x of fp16 experts is held as 2 h + l / 1024 in two fp16 values. h is
off by 2^-12 |x|, or by half of its least step, 2^-25; l takes up what 2 h leaves, (at most 2^-11 |x| or 2^-24) times 1024, and
is off by 2^-11 of itself or by 2^-25: 2^-22 |x| or 2^-35. bf16: h + l, 2^-8 of 2^-8."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def held(a, dtype):
    return 2.0 ** -22 * a + 2.0 ** -35 if dtype is torch.float16 else 2.0 ** -16 * a


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,slots", [(1, 1), (10, 1), (12, 1), (20, 1), (40, 2), (70, 1)])
@pytest.mark.parametrize("inter", [64, 200])
def test_each_activation(gfr, rows, slots, inter, dtype):
    """One product of three factors a column, no activation, the unit matrix as the down product: the outputs are the
    activations, of 2^0 to 2^-40. Every form of the down product: few pairs, one pass, several."""
    dt = TYPES[dtype]
    g = torch.Generator().manual_seed(inter)

    def odd(*shape):                                                   # values of the type with all of their bits in use
        return (1 + torch.rand(shape, generator=g)).to(dt)

    H = inter
    gu, down = torch.zeros((1, 2 * inter, H), dtype=dt), torch.eye(inter, dtype=dt).unsqueeze(0)
    at = torch.arange(inter) % 14
    gu[0, :inter, 0] = odd(inter) * 2.0 ** -at
    gu[0, inter:, 1] = odd(inter) * 2.0 ** -at.flip(0)
    x = torch.zeros((rows, H), dtype=dt)
    x[:, 0] = odd(rows) * 2.0 ** -(torch.arange(rows) % 14)
    x[:, 1] = odd(rows) * 2.0 ** -(torch.arange(rows) % 9)
    experts = gfr.Experts16(gu.cuda(), down.cuda())
    picks = torch.zeros((rows, slots), dtype=torch.int32, device="cuda")
    weights = torch.zeros((rows, slots), device="cuda")
    weights[:, 0] = 1.0
    y = gfr.experts16(x.cuda(), experts, picks, weights, activation=None, out_dtype=torch.float32)
    want = (x[:, :1].double() * gu[0, :inter, 0].double()) * (x[:, 1:2].double() * gu[0, inter:, 1].double())
    off = (y.double().cpu() - want).abs()
    # the product of gate and up, the two parts' sum and two more sums: half a unit of 32 bits each
    bound = held(want, dt) + 4 * 2.0 ** -24 * want
    worst = (off / bound).max().item()
    assert worst <= 1, f"off by {worst:.3g} of what is allowed"


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("size", [1.0, 2.0 ** -4, 2.0 ** -8])
@pytest.mark.parametrize("rows,hidden,inter", [(1, 512, 260), (5, 1001, 333), (33, 256, 128)])
def test_small_windows(gfr, rows, hidden, inter, size, dtype):
    """Ordinary weights, inputs of several sizes (activations of size^2): the error of the products in 32 bits, and of the
    activations as they are held."""
    dt = TYPES[dtype]
    g = torch.Generator().manual_seed(rows)
    x = (size * torch.randn((rows, hidden), generator=g)).to(dt)
    gu = (hidden ** -0.5 * torch.randn((3, 2 * inter, hidden), generator=g)).to(dt)
    down = (inter ** -0.5 * torch.randn((3, hidden, inter), generator=g)).to(dt)
    picks, weights = torch.arange(2 * rows).view(rows, 2) % 3, torch.rand((rows, 2), generator=g)
    y = gfr.experts16(x.cuda(), gfr.Experts16(gu.cuda(), down.cuda()), picks.int().cuda(), weights.cuda(), activation=None,
                      out_dtype=torch.float32)
    want, bound = torch.zeros((rows, hidden), dtype=torch.float64), torch.zeros((rows, hidden), dtype=torch.float64)
    for r in range(rows):
        for s in range(2):
            e, w = picks[r, s], weights[r, s].double()
            v, m = gu[e].double() @ x[r].double(), (hidden + 8) * 2.0 ** -23 * (gu[e].double().abs() @ x[r].double().abs())
            a = v[:inter] * v[inter:]
            ea = v[:inter].abs() * m[inter:] + v[inter:].abs() * m[:inter] + m[:inter] * m[inter:] + 2.0 ** -24 * a.abs()
            ea = ea + held(a.abs() + ea, dt)
            d = down[e].double()
            want[r] += w * (d @ a)
            bound[r] += w * (d.abs() @ ea + (2 * inter + 16) * 2.0 ** -23 * (d.abs() @ a.abs()))
    bound += 4 * 2.0 ** -24 * (want.abs() + bound)
    worst = ((y.double().cpu() - want).abs() / bound).max().item()
    assert worst <= 1, f"off by {worst:.3g} of what is allowed"


def test_the_upper_end(gfr):
    """Activations of up to 131008 have their value, those above 131040 are infinite."""
    H = I = 64
    gu, down = torch.zeros((1, 2 * I, H), dtype=torch.float16), torch.eye(I, dtype=torch.float16).unsqueeze(0)
    gu[0, :I, 0] = 1
    gu[0, I:, 1] = 1
    pairs = [(256.0, 255.75), (511.75, 256.0), (-511.75, 256.0), (256.0, 511.5), (255.875, 256.0), (1.0, 65504.0), (512.0, 256.0)]
    for rows in (7, 28):
        x = torch.zeros((rows, H), dtype=torch.float16)
        x[:, :2] = torch.tensor(pairs).repeat(rows // 7, 1).half()
        picks, weights = torch.zeros((rows, 1), dtype=torch.int32, device="cuda"), torch.ones((rows, 1), device="cuda")
        y = gfr.experts16(x.cuda(), gfr.Experts16(gu.cuda(), down.cuda()), picks, weights, activation=None, out_dtype=torch.float32).cpu()
        want = x[:, :1] .float() * x[:, 1:2].float()
        last = torch.arange(rows) % 7 == 6
        assert torch.equal(y[~last], want[~last].expand(-1, H)) and not torch.isfinite(y[last]).any()
