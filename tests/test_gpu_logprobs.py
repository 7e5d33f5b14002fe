"""Log probabilities of tokens (gfr_logprobs_run, token_logprobs) against the definitions in 64 bits.

The tolerance, counted before the first run, with z = (l - max l) / T and U = 2^-24 (half a unit of 32 bits): z is a
difference and two products (1 / T is rounded): 3 U |z|. exp(z) by exp2: the argument is off by 3 U |z|, the function by
2 U, so that a term is off by (3 |z| + 2) U of itself, of which the chunk's shift takes as much again. Sums are at most 64
values a thread, 6 over a wave, 8 over the waves and 6 over the chunks: 90 U of themselves, rounded up to 128 U. log and
log1p are within 4 U of their values. The entropy's sum of -z exp(z) has the same terms times |z|, all of one sign."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def reference(logits, tokens, top, temperature):
    l = logits.double()
    l = torch.where(torch.isnan(l), torch.full_like(l, -torch.inf), l)
    rows, vocab = l.shape
    most = l.max(1, keepdim=True).values
    dead = torch.isneginf(most)
    z = torch.where(l == most, torch.zeros_like(l), (l - most) / temperature)
    z = torch.where(torch.isneginf(l), torch.full_like(l, -torch.inf), z)
    e = torch.exp(z)
    size = torch.where(e > 0, -z, torch.zeros_like(z))                 # |z| of what counts
    count = (l == most).double().sum(1, keepdim=True)
    rest = torch.where(l == most, torch.zeros_like(e), e).sum(1, keepdim=True)
    e_rest = (torch.where(l == most, torch.zeros_like(e), e) * (6 * size + 4) * U).sum(1, keepdim=True) + 128 * U * rest
    s = count + rest
    log = torch.log(count) + torch.log1p(rest / count)
    e_log = e_rest / s + 4 * U * log
    a = (e * size).sum(1, keepdim=True)
    e_a = (e * size * (6 * size + 4) * U).sum(1, keepdim=True) + 256 * U * a
    entropy = (log + a / s).squeeze(1)
    e_entropy = (e_log + e_a / s + a / s * e_rest / s + 4 * U * (log + a / s)).squeeze(1)

    def log_p(at):
        lp = torch.where(dead, torch.full_like(at, -torch.inf, dtype=torch.float64), z.gather(1, at) - log)
        err = 3 * U * z.gather(1, at).abs() + e_log + U * lp.abs()
        return lp, torch.where(torch.isfinite(lp), err, torch.zeros_like(lp))

    there = (tokens >= 0) & (tokens < vocab)
    lp, err = log_p(tokens.long().clamp(0, vocab - 1))
    lp = torch.where(there, lp, torch.full_like(lp, -torch.inf))
    out = [(lp, err), (torch.where(dead.squeeze(1), torch.zeros_like(entropy), entropy),
                       torch.where(dead.squeeze(1), torch.zeros_like(entropy), e_entropy))]
    if top:
        ids = l.sort(dim=1, descending=True, stable=True).indices[:, :top]
        out += [ids, log_p(ids)]
    return out


def near(out, want, what):
    y, e = want
    assert out.dtype is torch.float32 and out.shape == y.shape, what
    same = out == y.float()     # infinities, and what rounds to them: the lowest bf16 less the largest is -6.8e38, fp32's end 3.4e38
    off = torch.where(same, torch.zeros_like(y), (out.double() - y).abs())
    assert (off <= e).all(), f"{what}: off by {off.max().item():.3g}"


def check(gfr, logits, tokens, top=0, temperature=1.0, what=""):
    got = gfr.token_logprobs(logits, tokens, top=top, temperature=temperature)
    torch.cuda.synchronize()
    two = tokens if tokens.dim() == 2 else tokens.unsqueeze(1)
    want = reference(logits, two, top, temperature)
    assert got.logprobs.shape == tokens.shape, what
    near(got.logprobs.view(two.shape), want[0], what + " logprobs")
    near(got.entropy, want[1], what + " entropy")
    if top:
        assert got.top_ids.dtype is torch.int32 and torch.equal(got.top_ids.long(), want[2]), what + " top ids"
        near(got.top_logprobs, want[3], what + " top logprobs")
    else:
        assert got.top_ids is None and got.top_logprobs is None
    return got


def randn(seed, rows, vocab, dtype, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, vocab), generator=g) * scale).to(dtype).cuda()


VOCABS = [1, 2, 3, 7, 8, 9, 31, 32, 33, 63, 64, 65, 100, 1000, 1001, 4095, 4096, 4097, 8193, 16385, 32767, 32768, 32769, 65537,
          131072, 160001]


@pytest.mark.parametrize("vocab", VOCABS)
def test_logprobs(gfr, vocab):
    """Every vocabulary in several windows, with types, tokens, tops and temperatures drawn from it."""
    rng = random.Random(vocab)
    for rows in [1, 2, 3, 17] + ([70, 600] if vocab < 10000 else [70] if vocab < 40000 else []):
        dtype = TYPES[rng.choice(list(TYPES))]
        l = randn(vocab + rows, rows, vocab, dtype)
        count = rng.choice([None, 0, 1, 3, 70])
        g = torch.Generator().manual_seed(rows)
        tokens = torch.randint(-2, vocab + 2, (rows,) if count is None else (rows, count), generator=g)
        tokens = tokens.to(rng.choice([torch.int32, torch.int64])).cuda()
        top = rng.choice([t for t in (0, 1, 2, 5, 8, 9, 16, 17, 20, 32) if t <= vocab])
        check(gfr, l, tokens, top, rng.choice([1.0, 0.7, 1.3]), f"rows {rows} vocab {vocab} top {top} {dtype}")


@pytest.mark.parametrize("vocab", [5, 1000, 1024, 1025, 2048, 2049, 4095, 4096, 4097, 8191, 8192, 8193, 9000, 16384, 16385])
def test_many_rows(gfr, vocab):
    """Windows of more rows than CUs hold, in every form that they take."""
    for dtype in TYPES.values():
        l = randn(vocab, 1100, vocab, dtype)
        l[7] = -torch.inf
        l[9, 1:] = torch.nan
        l[11] = 2.0
        check(gfr, l, torch.randint(0, vocab, (1100, 2), device="cuda"), min(vocab, 32), 0.7, f"vocab {vocab} {dtype}")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,vocab", [(1, 5), (3, 40), (2, 5000), (300, 33000), (2, 100001)])
def test_orders(gfr, rows, vocab, dtype):
    """Rows that meet the threshold's worst cases: one value, ascending, descending, a few values, one block of lanes far
    below all others, two zeros of either sign; the lower token first among equal logits."""
    dt = TYPES[dtype]
    at = torch.arange(vocab, device="cuda")
    rest = randn(1, 1, vocab, dt)[0]
    low = torch.where(at % 4096 < 128, torch.full_like(rest, -1000.0), rest)
    zeros = torch.where(at % 3 == 0, torch.zeros_like(rest), -torch.zeros_like(rest))
    for name, row in dict(one=torch.full_like(rest, 1.5), up=(at * (10.0 / vocab)).to(dt), down=(-at * (10.0 / vocab)).to(dt),
                          few=(at % 5).to(dt), low=low, zeros=zeros).items():
        l = row.expand(rows, vocab).contiguous()
        tokens = torch.arange(rows, device="cuda") % vocab
        for top in (1, 5, min(32, vocab)):
            check(gfr, l, tokens, top, 1.0, f"{name} top {top}")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [3, 33, 64, 70, 4097, 100001])
def test_masked(gfr, vocab, dtype):
    """Rows with everything masked, with one, two, 20 or half of the logits left (by -inf, NaN and the type's lowest value),
    with +inf in one and in several places, next to a row without any."""
    dt = TYPES[dtype]
    l = randn(vocab, 9, vocab, dt)
    g = torch.Generator().manual_seed(vocab)
    for r, left in enumerate([0, 1, 2, 20, vocab // 2]):
        order = torch.randperm(vocab, generator=g).cuda()
        l[r, order[left:]] = -torch.inf
        l[r, order[left::3]] = torch.nan
    l[5, 1:] = torch.finfo(dt).min
    l[6, vocab // 2] = torch.inf
    l[7, :3] = torch.inf
    tokens = torch.arange(vocab, device="cuda")[:70].repeat(9, 1)
    for top in {0, 1, min(20, vocab), min(32, vocab)}:
        got = check(gfr, l, tokens, top, 1.0, f"top {top}")
        alone = gfr.token_logprobs(l[8:], tokens[8:], top=top)
        assert torch.allclose(alone.logprobs, got.logprobs[8:], rtol=1e-5, atol=1e-6)
    assert torch.isneginf(got.logprobs[0]).all() and got.entropy[0] == 0
    assert got.entropy[6] == 0 and got.logprobs[7, 0].item() == pytest.approx(-torch.log(torch.tensor(3.0)).item(), rel=1e-6)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,vocab", [(6, 4096), (1100, 3000), (1030, 8000), (1030, 16000), (6, 32768), (6, 70000)])
def test_magnitudes(gfr, rows, vocab, dtype):
    """Places where the logits' magnitudes lie far apart: whole columns of a few hundred at the lowest value or at -1e4, all
    of one value but some, values near the largest and the lowest finite one, and next to +inf."""
    dt = TYPES[dtype]
    l = randn(vocab, rows, vocab, dt)
    column = torch.arange(vocab, device="cuda")
    l[0, column // 8 % 64 >= 40] = torch.finfo(dt).min
    l[1, column // 8 % 64 >= 10] = -1e4
    l[2] = 1.0
    l[2, column % 701 == 3] = 2.0
    l[3] = torch.where(column % 2 == 0, torch.finfo(dt).max, torch.finfo(dt).min)
    l[4, column % 1009 == 5] = torch.inf
    l[5] = l[5] * 1e-3
    tokens = column[:40].repeat(rows, 1)
    for top in (1, 4, 9, 20, 32):
        check(gfr, l, tokens, top, 1.0, f"top {top}")


def test_near_certain(gfr):
    """A token with nearly all of the probability: its log p keeps its digits (1 + the others' sum would round them off)."""
    l = torch.zeros((4, 50000), device="cuda")
    for r, gap in enumerate([20.0, 30.0, 60.0, 87.0]):
        l[r, 777] = gap
    tokens = torch.full((4,), 777, device="cuda")
    got = gfr.token_logprobs(l, tokens).logprobs.double()
    want = -torch.log1p(49999 * torch.exp(-l[:, 777].double()))
    assert ((got - want).abs() <= 2.0 ** -17 * want.abs()).all(), (got, want)   # (the exponent: 3 * 87 U, the sum: 128 U)


def test_strides(gfr):
    """Logits and tokens that are slices, at odd addresses, of buffers full of NaN and of tokens out of range: the same
    bits as from tensors of their own."""
    for rows, vocab in ((1, 1000), (5, 32003), (40, 999)):
        for name, dt in TYPES.items():
            l = randn(vocab, rows, vocab, dt)
            tokens = torch.randint(0, vocab, (rows, 3), device="cuda")
            wide = torch.full((rows, vocab + 11), torch.nan, dtype=dt, device="cuda")
            wide[:, 3:3 + vocab] = l
            more = torch.full((rows, 9), vocab + 5, device="cuda")
            more[:, 2:5] = tokens
            a, b = gfr.token_logprobs(l, tokens, top=7), gfr.token_logprobs(wide[:, 3:3 + vocab], more[:, 2:5], top=7)
            assert all(torch.equal(x, y) for x, y in zip(a, b)), name


def test_far_rows(gfr):
    """Rows whose elements' offsets pass 2^31 and 2^32 bytes."""
    vocab, stride = 5000, 1 << 30
    wide = torch.empty(2 * stride + stride // 2, dtype=torch.bfloat16, device="cuda")
    l = wide.as_strided((3, vocab), (stride, 1))
    l.copy_(randn(1, 3, vocab, torch.bfloat16))
    check(gfr, l, torch.tensor([4, 5, 6], device="cuda"), 20)


def test_widest_vocabulary(gfr):
    check(gfr, randn(1, 2, 1 << 21, torch.bfloat16), torch.tensor([1, (1 << 21) - 1], device="cuda"), 32)
    check(gfr, randn(1, 1, (1 << 21) - 3, torch.float32), torch.tensor([7], device="cuda"), 3)


def test_stream_graph_and_repeats(gfr):
    """On a stream of the caller's; twice with the same bits; captured twice, replays in turn following the inputs."""
    l = randn(1, 9, 70000, torch.bfloat16)
    tokens = torch.randint(0, 70000, (9, 2), device="cuda")
    want = gfr.token_logprobs(l, tokens, top=20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = gfr.token_logprobs(l, tokens, top=20, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graphs, outs = [], []
    for t in (tokens, tokens.int()):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(gfr.token_logprobs(l, t, top=20))
    for seed in (5, 6, 7):
        l.copy_(randn(seed, 9, 70000, torch.bfloat16))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        want = gfr.token_logprobs(l, tokens, top=20)
        for out in outs:
            assert all(torch.equal(x, y) for x, y in zip(out, want))


def test_python_refusals(gfr):
    l = randn(1, 4, 100, torch.bfloat16)
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    for bad in ((l.double(), t), (l, t[:3]), (l, t.float()), (l, t.view(2, 2)), (l, t.cpu()), (l.t().contiguous().t(), t),
                (l, t.view(4, 1, 1))):
        with pytest.raises(ValueError):
            gfr.token_logprobs(*bad)
    for kw, needle in ((dict(top=33), "top 33"), (dict(top=-1), "top -1"), (dict(temperature=0.0), "temperature"),
                       (dict(temperature=float("nan")), "temperature")):
        with pytest.raises(gfr.GfrError, match=needle):
            gfr.token_logprobs(l, t, **kw)
    with pytest.raises(gfr.GfrError, match="rows 0"):
        gfr.token_logprobs(l[:0], t[:0])
    with pytest.raises(gfr.GfrError, match="below"):
        gfr.token_logprobs(l[:1].expand(4, 100), t)
