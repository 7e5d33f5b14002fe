"""A decoder layer's second half and the head after it, as a caller puts them together: the norms around the block, the router's
logits and gate, the 16-bit routed experts, the next norm, the head's product, the tokens' log probabilities; eager, captured,
and with rows that are padding. Each step against its own definition is the other files' matter: here the whole against 64
bits, with the roundings of the 16-bit rows between the steps counted loosely as one relative error each."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HIDDEN, INTER, EXPERTS, TOPK, VOCAB = 1024, 256, 24, 4, 5000


def randn(seed, *shape, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


class Model:
    def __init__(self, gfr):
        self.gfr = gfr
        self.first = gfr.Norm("rms", weight=randn(1, HIDDEN, scale=0.2) + 1, eps=1e-5)
        self.post = gfr.Norm("rms", weight=randn(2, HIDDEN, scale=0.2) + 1, eps=1e-5)
        self.last = gfr.Norm("rms", weight=randn(3, HIDDEN, scale=0.2) + 1, eps=1e-5)
        self.router = randn(4, EXPERTS, HIDDEN, scale=3 * HIDDEN ** -0.5)
        self.gate = gfr.Gate(score="sigmoid", scale=1.5)
        # the shared expert is the last one, as the gate's picks have it
        self.experts = gfr.Experts16(randn(5, EXPERTS + 1, 2 * INTER, HIDDEN, scale=2 * HIDDEN ** -0.5),
                                     randn(6, EXPERTS + 1, HIDDEN, INTER, scale=INTER ** -0.5))
        self.head = randn(7, VOCAB, HIDDEN, scale=3 * HIDDEN ** -0.5)

    def run(self, stream, attention, tokens, real=None):
        """stream [rows, HIDDEN] and the block's output before it -> (stream after the layer, picks, log probabilities)."""
        gfr = self.gfr
        h, x = gfr.block_norm(attention, stream, pre=self.first)
        picks, weights = gfr.route_gate(gfr.dense(x, self.router, out_dtype=torch.float32), self.gate, TOPK)
        if real is not None:
            picks[real:] = -1
        y = gfr.experts16(x, self.experts, picks, weights, out_dtype=torch.float32)
        h, x = gfr.block_norm(y, h, post=self.post, pre=self.last, out_dtype=torch.bfloat16)
        return h, picks, gfr.token_logprobs(gfr.dense(x, self.head, out_dtype=torch.float32), tokens, top=5)

    def exact(self, stream, attention, tokens, picks):
        """The same in 64 bits, with these picks (near choices are the gate's own tests' matter)."""
        def rms(z, p):
            return z / torch.sqrt((z * z).mean(1, keepdim=True) + p.eps) * p.weight.double()

        def to(t):
            return t.double()

        h = to(stream) + to(attention)
        x = rms(h, self.first)
        scores = torch.sigmoid(x @ to(self.router).t().contiguous())
        out = torch.zeros_like(h)
        for r in range(h.shape[0]):
            ids = picks[r].tolist()
            if ids[0] < 0:
                continue
            w = scores[r, ids[:-1]]
            w = torch.cat((w / w.sum() * 1.5, torch.ones(1, dtype=torch.float64, device="cuda")))
            for e, weight in zip(ids, w):
                g, u = (to(self.experts.gu[e]) @ x[r]).split(INTER)
                out[r] += weight * (to(self.experts.down[e]) @ (g * torch.sigmoid(g) * u))
        h = h + torch.where(out.abs().sum(1, keepdim=True) > 0, rms(out, self.post), torch.zeros_like(out))
        return h, torch.log_softmax(rms(h, self.last) @ to(self.head).t().contiguous(), 1)


@pytest.mark.parametrize("rows", [1, 6, 40])
def test_layer_and_head(gfr, rows):
    m = Model(gfr)
    stream, attention = randn(8, rows, HIDDEN), randn(9, rows, HIDDEN)
    tokens = torch.randint(0, VOCAB, (rows, 2), device="cuda")
    h, picks, lp = m.run(stream, attention, tokens)
    h64, lp64 = m.exact(stream, attention, tokens, picks)
    # the stream is rounded twice (2^-8 each), x before the experts once, their weights' logits follow it: within 5 * 2^-8 of
    # the stream's size; the logits' errors are that of x times a row of the head of size 3
    assert torch.linalg.vector_norm(h.double() - h64) <= 5 * 2.0 ** -8 * torch.linalg.vector_norm(h64)
    got = lp.logprobs.double() - lp64.gather(1, tokens)
    assert got.abs().max() <= 3 * 4 * 5 * 2.0 ** -8, got.abs().max()      # (four times the size: the largest of some)
    assert (lp.top_logprobs[:, 0] >= lp.logprobs.max(1).values).all()


def test_padded_and_captured(gfr):
    """Rows behind the last sequence keep their stream; replays follow the inputs; a window in a graph equals the eager one."""
    m = Model(gfr)
    rows, real = 12, 9
    stream, attention = randn(8, rows, HIDDEN), randn(9, rows, HIDDEN)
    tokens = torch.randint(0, VOCAB, (rows, 2), device="cuda")
    h, picks, lp = m.run(stream, attention, tokens, real)
    assert torch.equal(h[real:], gfr.block_norm(attention, stream)[0][real:])
    alone = m.run(stream[:real], attention[:real], tokens[:real])
    assert torch.equal(alone[0], h[:real]) and torch.equal(alone[1], picks[:real])
    m.run(stream, attention, tokens, real)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.run(stream, attention, tokens, real)
    for seed in (11, 12, 13):
        stream.copy_(randn(seed, rows, HIDDEN))
        attention.copy_(randn(seed + 50, rows, HIDDEN))
        graph.replay()
        want = m.run(stream, attention, tokens, real)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        assert all(torch.equal(a, b) for a, b in zip(out[2], want[2]))
