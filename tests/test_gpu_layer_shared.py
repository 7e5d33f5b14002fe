"""The layer with a shared expert that is not EXL3: what its runs leave behind, refused ones among them."""
import pytest
import torch

pytestmark = pytest.mark.gpu

D, N, E, TOPK, BITS = 512, 256, 24, 4, 4


@pytest.fixture(scope="module")
def layer_weights():
    import synth
    return synth.experts(E + 1, D, N, BITS, seed=5), synth.experts(E, D, N, BITS, seed=6)


def bf16_shared(gfr, hidden, inter, seed=3, limit=2.0):
    g = torch.Generator().manual_seed(seed)
    return gfr.Bf16SharedWeights((torch.randn((2 * inter, hidden), generator=g) * 3 / hidden ** 0.5).to(torch.bfloat16).cuda(),
                                 (torch.randn((hidden, inter), generator=g) / inter ** 0.5).to(torch.bfloat16).cuda(), limit)


def router_weight(hidden, seed=4):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((E, hidden), generator=g) / hidden ** 0.5).to(torch.bfloat16).cuda()


@pytest.mark.parametrize("rows", [1, 3, 20, 300])
@pytest.mark.parametrize("kind", ["fp8", "bf16"])
@pytest.mark.parametrize("router", [False, True])
def test_refused_run_launches_nothing(gfr, layer_weights, rows, kind, router):
    """Weights of another number of experts: refused before the shared expert's launches, the outputs of the run before
    still in place."""
    import synth
    wrong, w = layer_weights
    x, l, rw = synth.activations(rows, D, rows), synth.logits(rows, E, rows), router_weight(D)
    sw = synth.fp8_shared(D, N) if kind == "fp8" else bf16_shared(gfr, D, N)
    m = gfr.Moe(D, N, E, TOPK, rows, shared_exl3=False)
    run = getattr(m, f"run_{'router_' if router else ''}{kind}")
    run(w, x, rw if router else l, sw, rows)
    torch.cuda.synchronize()
    before = [t.clone() for t in (m.output, m.shared_output, m.picks, m.weights)]
    x2 = synth.activations(rows, D, rows + 50)
    with pytest.raises(gfr.GfrError, match="weights hold 25 experts"):
        run(wrong, x2, rw if router else l, sw, rows)
    torch.cuda.synchronize()
    for a, b in zip(before, (m.output, m.shared_output, m.picks, m.weights)):
        assert torch.equal(a, b)
    m.output.zero_()
    run(w, x, rw if router else l, sw, rows)
    torch.cuda.synchronize()
    assert torch.equal(m.output, before[0])


def test_refused_down_matrix_launches_nothing(gfr, layer_weights):
    """The down matrix at an odd address (through the C interface): refused before the gate and up matrices' product."""
    import ctypes
    import synth
    w = layer_weights[1]
    rows = 3
    x, l, sw = synth.activations(rows, D, 1), synth.logits(rows, E, 1), bf16_shared(gfr, D, N)
    m = gfr.Moe(D, N, E, TOPK, rows, shared_exl3=False)
    m.run_bf16(w, x, l, sw, rows)
    torch.cuda.synchronize()
    before = m.output.clone(), m.shared_output.clone()
    ws, ss = w.struct(), sw.struct()
    ss.down += 1
    rc = gfr.lib().gfr_moe_run_bf16(m._h, gfr._stream(), ctypes.byref(ws), x.data_ptr(), l.data_ptr(), ctypes.byref(ss), rows)
    assert rc == gfr.GFR_EINVAL
    torch.cuda.synchronize()
    assert torch.equal(m.output, before[0]) and torch.equal(m.shared_output, before[1])


@pytest.mark.parametrize("hidden", [512, 768])
def test_shared_output_of_a_bf16_run(gfr, hidden):
    """gfr_moe_shared_output after gfr_moe_run_bf16: the two products' output, where the layer can have an FP8 shared
    expert (hidden a multiple of 512) and where it cannot."""
    import synth
    rows, inter = 20, 192
    w, sw = synth.experts(E, hidden, N, BITS, seed=6), bf16_shared(gfr, hidden, inter)
    x, l = synth.activations(rows, hidden, rows), synth.logits(rows, E, rows)
    m = gfr.Moe(hidden, N, E, TOPK, rows, shared_exl3=False)
    m.run_bf16(w, x, l, sw, rows)
    want = gfr.dense(gfr.dense_gated(x, sw.gu, limit=2.0), sw.down, out_dtype=torch.float32)
    torch.cuda.synchronize()
    assert torch.equal(m.shared_output[:rows], want)
    with pytest.raises(ValueError, match="EXL3"):
        gfr.Moe(hidden, N, E, TOPK, rows).shared_output


@pytest.mark.parametrize("hidden", [512, 768])
def test_bf16_buffers_are_allocated_when_asked_for(gfr, hidden):
    """A layer that never runs a bf16 shared expert holds no buffers for one; reserve_bf16 allocates them once, and a
    layer with the FP8 shared expert's buffers has them."""
    rows = 8192
    m = gfr.Moe(hidden, N, E, TOPK, rows, shared_exl3=False)
    torch.cuda.synchronize()
    free = [torch.cuda.mem_get_info()[0]]
    for _ in range(2):
        m.reserve_bf16()
        assert gfr.lib().gfr_moe_reserve_bf16(m._h) == 0
        free.append(torch.cuda.mem_get_info()[0])
    want = 0 if hidden % 512 == 0 else rows * (2 * N + 4 * hidden)
    assert free[1] == free[2] and want <= free[0] - free[1] <= want + (8 << 20)
    assert m.shared_output.shape == (rows, hidden)


def test_bf16_run_without_its_buffers(gfr):
    """Refused in C before reserve, and in Python inside a capture (where nothing may be allocated)."""
    import ctypes
    import synth
    hidden, rows = 768, 3
    w, sw = synth.experts(E, hidden, N, BITS, seed=6), bf16_shared(gfr, hidden, N)
    x, l = synth.activations(rows, hidden, rows), synth.logits(rows, E, rows)
    m = gfr.Moe(hidden, N, E, TOPK, rows, shared_exl3=False)
    with pytest.raises(ValueError, match="reserve_bf16"):
        m.shared_output
    ws, ss = w.struct(), sw.struct()
    L = gfr.lib()
    assert L.gfr_moe_run_bf16(m._h, gfr._stream(), ctypes.byref(ws), x.data_ptr(), l.data_ptr(), ctypes.byref(ss),
                              rows) == gfr.GFR_EINVAL and b"gfr_moe_reserve_bf16" in L.gfr_last_error()
    other = gfr.Moe(hidden, N, E, TOPK, rows, shared_exl3=False)
    other.run_bf16(w, x, l, sw, rows)                      # (its kernels are loaded before the capture)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError, match="capture"):
            m.run_bf16(w, x, l, sw, rows)
        other.run_bf16(w, x, l, sw, rows)
    m.run_bf16(w, x, l, sw, rows)
    torch.cuda.synchronize()
    want = m.output.clone()
    for _ in range(3):
        other.output.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(other.output, want)


def test_no_bf16_buffers_for_an_exl3_shared_expert(gfr):
    with pytest.raises(gfr.GfrError, match="EXL3"):
        gfr.Moe(D, N, E, TOPK, 4).reserve_bf16()


def test_bf16_run_on_another_device_is_refused(gfr, layer_weights, monkeypatch):
    """A launch goes to the current device's stream: the layer, the shared expert's weights and a given stream have to be
    on it."""
    import synth
    w, rows = layer_weights[1], 2
    x, l, rw, sw = synth.activations(rows, D, 1), synth.logits(rows, E, 1), router_weight(D), bf16_shared(gfr, D, N)
    m = gfr.Moe(D, N, E, TOPK, rows, shared_exl3=False)
    host = gfr.Bf16SharedWeights(sw.gu, sw.down.cpu())
    with pytest.raises(ValueError, match="shared expert on cpu"):
        m.run_bf16(w, x, l, host, rows)

    class Elsewhere:
        device_index, cuda_stream = 1, 0

    with pytest.raises(ValueError, match="stream of cuda:1"):
        m.run_bf16(w, x, l, sw, rows, stream=Elsewhere())
    monkeypatch.setattr(gfr, "_get_device", lambda: 1)
    for run, arg in ((m.run_bf16, l), (m.run_router_bf16, rw)):
        with pytest.raises(ValueError, match="current device is cuda:1"):
            run(w, x, arg, sw, rows)


@pytest.mark.parametrize("rows", [1, 3, 20, 40, 300])
def test_gate_with_the_shared_expert_on_a_branch(gfr, layer_weights, rows):
    """The bf16 shared expert's products on the branch stream (dense_gated and dense with its stream) beside the layer
    under the general gate: byte-equal to run_bf16, eagerly and in every replay of a graph."""
    import synth
    w, sw = layer_weights[1], bf16_shared(gfr, D, N)
    x, l = synth.activations(rows, D, rows), synth.logits(rows, E, rows)
    bias = torch.randn(E, generator=torch.Generator().manual_seed(5)).cuda() * 0.02
    m = gfr.Moe(D, N, E, TOPK, rows, shared_exl3=False)
    m.set_gate(gfr.Gate(bias=bias, groups=6, kept_groups=3, scale=2.5))
    m.run_bf16(w, x, l, sw, rows)
    torch.cuda.synchronize()
    want = m.output.clone()
    shared = torch.empty(rows, D, device="cuda")
    branch, main = gfr.SharedBranch(), torch.cuda.Stream()

    def layer():
        shared.fill_(float("nan"))

        def shared_fn(side):
            gfr.dense(gfr.dense_gated(x, sw.gu, limit=2.0, stream=side), sw.down, out=shared, stream=side)

        branch.run(main, shared_fn, lambda ready: m.run(w, x, l, rows, stream=main, shared=shared, shared_ready=ready))

    with torch.cuda.stream(main):
        m.output.zero_()
        layer()
    torch.cuda.synchronize()
    assert torch.equal(m.output, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(main):
        with torch.cuda.graph(graph, stream=main):
            layer()
    for _ in range(3):
        m.output.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(main):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(m.output, want)


@pytest.mark.parametrize("rows", [1, 4, 20, 300])
def test_router_logits_then_the_gate(gfr, layer_weights, rows):
    """run_router under the general gate: the picks and weights of route_gate on the router's logits."""
    import synth
    w, rw = layer_weights[0], router_weight(D)
    x = synth.activations(rows, D, rows)
    gate = gfr.Gate(score="softmax", groups=4, kept_groups=2, group_score="max", renormalise=False, scale=1.5)
    m = gfr.Moe(D, N, E, TOPK, rows)
    m.set_gate(gate)
    m.run_router(w, x, rw, rows)
    logits = gfr.router_logits(x, rw)
    p, wt = gfr.route_gate(logits, gate, TOPK)
    torch.cuda.synchronize()
    assert torch.equal(m.picks, p) and torch.equal(m.weights, wt)
    got = m.output.clone()
    m.run(w, x, logits, rows)
    torch.cuda.synchronize()
    assert torch.equal(m.output, got)


@pytest.mark.parametrize("rows", [1, 300])
def test_first_run_right_after_the_buffers(gfr, layer_weights, rows):
    """A layer made, its buffers reserved and run at once on a stream of the caller's: the buffers' clearing is over by
    then (the bytes of a run after a synchronization)."""
    import synth
    hidden = 768
    w, sw = synth.experts(E, hidden, N, BITS, seed=6), bf16_shared(gfr, hidden, N)
    x, l = synth.activations(rows, hidden, rows), synth.logits(rows, E, rows)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(3):
        m = gfr.Moe(hidden, N, E, TOPK, 8192, shared_exl3=False)
        m.run_bf16(w, x, l, sw, rows, stream=s)
        s.synchronize()
        first = m.output[:rows].clone(), m.shared_output[:rows].clone(), m.picks[:rows].clone(), m.weights[:rows].clone()
        torch.cuda.synchronize()
        m.run_bf16(w, x, l, sw, rows)
        torch.cuda.synchronize()
        for a, b in zip(first, (m.output, m.shared_output, m.picks, m.weights)):
            assert torch.equal(a, b[:rows])
