"""Log probabilities (gfr_logprobs_run, token_logprobs) where logits lie far from 0, lie close together at low temperatures, or
are masked by finite values, against the definitions in 64 bits.

The tolerance, counted before the first run, goes by the distance from the row's largest logit alone; U = 2^-24, half a unit
of 32 bits. z = (l - max l) / T is a difference, 1 / T rounded, and a product: 3 U |z|, by which a term exp(z) is off, and by
2 U for the exponential. Rows that are joined scale a chunk's sums: another exponential, a sum and a product, 6 U for all. A sum
of n terms that are not zero rounds n - 1 times at most in any order, and 80 times on any term's way (64 values a thread, 6
sums over a wave, 3 over the waves, 6 over chunks). Terms below 2^-126 may be taken for 0. The logarithms are within 4 U of
their sum, a quotient or product adds U. A token's own (l - max l) / T: 2 U of itself."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U, TINY = 2.0 ** -24, 2.0 ** -126
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def reference(logits, temperature):
    """Of each row: z and log p of every token with its error, the entropy with its error."""
    t = torch.tensor(temperature, dtype=torch.float32).double().item()
    l = logits.double()
    l = torch.where(torch.isnan(l), torch.full_like(l, -torch.inf), l)
    most = l.max(1, keepdim=True).values
    equal = l == most
    z = torch.where(equal, torch.zeros_like(l), (l - most) / t)
    e = torch.where(equal, torch.zeros_like(l), torch.exp(z))
    size = torch.where(e > 0, -z, torch.zeros_like(z))
    count, rest = equal.double().sum(1, keepdim=True), e.sum(1, keepdim=True)
    depth = ((e > TINY / 2).double().sum(1, keepdim=True) - 1).clamp(0, 80)
    term = 1.01 * U * (3 * size + 8)
    e_rest = (e * term).sum(1, keepdim=True) + depth * U * rest + l.shape[1] * TINY
    s = count + rest
    log = torch.log(count) + torch.log1p(rest / count)
    e_log = (e_rest + U * rest) / s + 4 * U * log
    a = (e * size).sum(1, keepdim=True)
    e_a = (e * size * (term + U)).sum(1, keepdim=True) + (depth + 7) * U * a + l.shape[1] * 128 * TINY
    entropy = log + a / s
    e_entropy = e_log + e_a / s + a / s * (e_rest / s + U) + U * entropy
    lp = z - log
    e_lp = 2 * U * size_of(z) + e_log + U * size_of(lp) + 2.0 ** -149
    return l, lp, e_lp, entropy.squeeze(1), e_entropy.squeeze(1)


def size_of(v):
    return torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v))


def near(out, y, e, what):
    same = out == y.float()                                            # infinities, and what rounds to them
    off = torch.where(same, torch.zeros_like(y), (out.double() - y).abs())
    bad = ~(off <= e)
    assert not bad.any(), f"{what}: row {bad.nonzero()[0].tolist()} is {out[bad][0].item():.9g} and not " \
        f"{y[bad][0].item():.9g}: off by {off[bad][0].item():.3g}, allowed {e[bad][0].item():.3g}"


def check(gfr, logits, tokens, top, temperature, what):
    got = gfr.token_logprobs(logits, tokens, top=top, temperature=temperature)
    torch.cuda.synchronize()
    l, lp, e, entropy, e_entropy = reference(logits, temperature)
    near(got.logprobs, lp.gather(1, tokens), e.gather(1, tokens), what + " logprobs")
    near(got.entropy, entropy, e_entropy, what + " entropy")
    ids = l.sort(dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(got.top_ids.long(), ids), what + " top ids"
    near(got.top_logprobs, lp.gather(1, ids), e.gather(1, ids), what + " top logprobs")


TEMPERATURES = [1e-6, 1e-3, 0.01, 0.1, 0.7, 1.0, 30.0, 1e6]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("temperature", TEMPERATURES)
def test_few_candidates(gfr, temperature, dtype):
    """Rows of a few logits near a value far from 0, a step of the type or 0.3 T apart, all others masked: few roundings, so
    that the bound is close. Every form: short rows, joined ones, many rows."""
    dt = TYPES[dtype]
    for rows, vocab in ((1, 40), (1, 5000), (1, 40000), (60, 700)):
        g = torch.Generator().manual_seed(vocab)
        lines, tokens = [], []
        for mean in (0.0, 39.125, 100.0, -300.0, 1000.0, 1e4, 6e4, 1e6, -3e7):
            if abs(mean) > torch.finfo(dt).max:
                continue
            step = max(0.3 * temperature, abs(mean) * torch.finfo(dt).eps)
            for left in (2, 5, 9):
                at = torch.randperm(vocab, generator=g)[:left]
                line = torch.full((vocab,), -torch.inf, dtype=dt)
                line[at] = (mean - step * torch.arange(left, dtype=torch.float64)).to(dt)
                lines.append(line)
                tokens.append(torch.stack((at[0], at[1], at[-1], at[0])))
        l, t = torch.stack(lines).repeat(rows, 1).cuda(), torch.stack(tokens).repeat(rows, 1).cuda()
        check(gfr, l, t, 9, temperature, f"{l.shape[0]} x {vocab}")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("temperature", TEMPERATURES)
def test_means(gfr, temperature, dtype):
    """Ordinary rows, N(mean, 2.5^2), in both forms."""
    dt = TYPES[dtype]
    means = torch.tensor([m for m in (0.0, 30.0, 100.0, -300.0, 1000.0, 1e4, 1e5) if m < torch.finfo(dt).max])
    for vocab in (4000, 40000):
        g = torch.Generator().manual_seed(vocab)
        l = (means.unsqueeze(1) + 2.5 * torch.randn((len(means), vocab), generator=g)).to(dt).cuda()
        check(gfr, l, torch.randint(0, vocab, (len(means), 3), generator=g).cuda(), 20, temperature, f"vocab {vocab}")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("temperature", [1e-6, 0.1, 0.7, 1.0])
def test_finite_far_values(gfr, temperature, dtype):
    """One logit of 1e4 to 1e38 over zeros; masks of -1e4 to -1e38 over all of a row, all but three tokens, a stretch that
    holds whole chunks of a joined row."""
    dt = TYPES[dtype]
    for vocab in (40, 5000, 32768, 70000):
        g = torch.Generator().manual_seed(vocab)
        ordinary = (3 * torch.randn(vocab, generator=g)).to(dt)
        lines = []
        for far in (1e4, 5e4, 1e6, 3e9, 1e10, 1e12, 1e15, 1e20, 1e25, 1e30, 1e38):
            if far > torch.finfo(dt).max:
                continue
            one, all_masked, three, stretch = torch.zeros(vocab, dtype=dt), torch.full((vocab,), -far, dtype=dt), ordinary.clone(), ordinary.clone()
            one[vocab // 3] = far
            three[torch.randperm(vocab, generator=g)[3:]] = -far
            stretch[vocab // 8:vocab // 2] = -far
            lines += [one, all_masked, three, stretch]
        l = torch.stack(lines).cuda()
        t = torch.tensor([[0, vocab // 3, vocab // 4, vocab - 1]]).repeat(len(lines), 1).cuda()
        check(gfr, l, t, 5, temperature, f"vocab {vocab}")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("temperature", [1.5, 4.0, 1e6])
def test_differences_beyond_32_bits(gfr, temperature, dtype):
    """Logits whose difference passes the range of 32 bits and whose difference over the temperature does not: no infinity."""
    dt = TYPES[dtype]
    big = torch.finfo(dt).max
    for vocab in (40, 5000, 70000):
        l = torch.zeros((3, vocab), dtype=dt)
        l[0, 3], l[0, 5] = big, -big
        l[1] = -big
        l[1, 3] = 0.75 * big
        l[2, 3], l[2, 4], l[2, 5] = big, -0.7 * big, -torch.inf
        t = torch.tensor([[3, 4, 5, 0]]).repeat(3, 1).cuda()
        check(gfr, l.cuda(), t, 5, temperature, f"vocab {vocab}")
        if temperature > 2:
            assert torch.isfinite(gfr.token_logprobs(l.cuda(), t, temperature=temperature).logprobs[:2]).all()
