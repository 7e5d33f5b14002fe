"""What the norms, the 16-bit experts and the log probabilities refuse: host checks before any launch (no GPU needed)."""
import pytest


def refused(rc, needle):
    import gfr_moe
    said = gfr_moe.lib().gfr_last_error().decode()
    assert rc == gfr_moe.GFR_EINVAL and needle in said, said


NORM = ("rows n x_type residual_type gate_type h_type y_type gate_column sigmoid scale residual_scale x x_stride residual "
        "residual_stride gate gate_row h h_stride y y_stride").split()
PART = "kind weight_type bias_type eps offset weight bias".split()


@pytest.mark.parametrize("kw,needle", [
    (dict(x=0), "null"), (dict(h=0, y=0, pre=dict(kind=0)), "null"), (dict(rows=0), "rows 0"), (dict(rows=-3), "rows -3"),
    (dict(n=0), "n 0"), (dict(n=32769, x_stride=40000, h_stride=40000, y_stride=40000), "n 32769"),
    (dict(pre=dict(kind=3)), "pre kind 3"), (dict(post=dict(kind=-1)), "post kind -1"),
    (dict(post=dict(kind=0, weight=16)), "no kind"), (dict(pre=dict(eps=-1.0)), "eps"),
    (dict(pre=dict(eps=float("nan"))), "eps"), (dict(pre=dict(offset=float("inf"))), "offset"),
    (dict(pre=dict(weight=16, weight_type=3)), "types 3"), (dict(pre=dict(bias=18, bias_type=2)), "aligned"),
    (dict(y=0), "go together"), (dict(pre=dict(kind=0)), "go together"), (dict(gate_column=2), "gate column 2"),
    (dict(sigmoid=2), "sigmoid 2"), (dict(scale=float("inf")), "finite"), (dict(residual_scale=float("nan")), "finite"),
    (dict(x_type=3), "x type 3"), (dict(h_type=-1), "h type -1"), (dict(x_stride=31), "x stride 31"),
    (dict(y_stride=31), "y stride 31"), (dict(h_stride=(1 << 31) + 1), "h stride"),
    (dict(residual=1 << 33, residual_stride=16), "residual stride 16"), (dict(gate=1 << 33, gate_row=16, gate_column=1), "gate stride"),
    (dict(gate=1 << 33, gate_row=-1, gate_column=0), "gate stride"), (dict(x=17), "aligned"), (dict(h=(1 << 30) + 2, h_type=2), "aligned"),
    (dict(h=64, h_stride=32), "h overlaps x"), (dict(x=1 << 20, h=1 << 20, h_type=2), "h overlaps x"),
    (dict(x=1 << 20, y=1 << 20, y_stride=33), "y overlaps x"), (dict(y=1 << 30), "h overlaps y"),
    (dict(gate=1 << 31, gate_row=32, gate_column=1), "y overlaps gate"),
    (dict(pre=dict(weight=1 << 30)), "h overlaps pre weight"), (dict(post=dict(kind=2, bias=1 << 31)), "y overlaps post bias"),
])
def test_block_norm_refuses(kw, needle):
    import gfr_moe
    a = dict(rows=4, n=32, scale=1.0, residual_scale=1.0, x=16, x_stride=32, h=1 << 30, h_stride=32, y=1 << 31, y_stride=32)
    parts = dict(post=dict(kind=0, eps=0.0, offset=0.0), pre=dict(kind=1, eps=1e-5, offset=0.0))
    for k, v in kw.items():
        parts[k].update(v) if k in parts else a.update({k: v})
    st = gfr_moe._BLOCK_NORM.pack(*[a.get(n, 0) for n in NORM], *[parts[p].get(n, 0) for p in ("post", "pre") for n in PART])
    refused(gfr_moe.lib().gfr_block_norm_run(None, st), needle)
    refused(gfr_moe.lib().gfr_block_norm_run(None, None), "null")


LOGPROBS = ("rows vocab tokens top type wide_tokens temperature logits stride token tokens_stride logprobs entropy top_ids "
            "top_logprobs workspace workspace_bytes").split()


@pytest.mark.parametrize("kw,needle", [
    (dict(rows=0), "rows 0"), (dict(rows=-1), "rows -1"), (dict(vocab=0), "vocab 0"), (dict(vocab=(1 << 21) + 1), "vocab 2097153"),
    (dict(top=-1), "top -1"), (dict(top=33), "top 33"), (dict(vocab=4, top=5), "at most vocab"), (dict(rows=1 << 23), "too many"),
    (dict(tokens=-1), "tokens -1"), (dict(logits=0), "null"), (dict(entropy=0), "null"), (dict(workspace=0), "null"),
    (dict(token=0), "null"), (dict(logprobs=0), "null"), (dict(top_ids=0), "null"), (dict(top_logprobs=0), "null"),
    (dict(type=3), "type 3"), (dict(wide_tokens=2), "wide tokens 2"), (dict(temperature=0.0), "temperature"),
    (dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature"), (dict(stride=39999), "stride 39999"), (dict(tokens_stride=1), "tokens' 1"),
    (dict(stride=(1 << 31) + 1), "stride"), (dict(workspace_bytes=100), "workspace of 100 bytes"), (dict(logits=(1 << 40) + 1), "aligned"),
    (dict(token=(1 << 41) + 4), "aligned"), (dict(entropy=(1 << 43) + 2), "aligned"), (dict(workspace=(1 << 46) + 4), "aligned"),
    (dict(entropy=1 << 40), "overlaps"), (dict(workspace=1 << 41), "overlaps"), (dict(top_ids=(1 << 42) + 24), "overlaps"),
    (dict(top_logprobs=1 << 44), "overlaps"),
])
def test_logprobs_refuses(kw, needle):
    import gfr_moe
    a = dict(rows=4, vocab=40000, tokens=2, top=5, type=0, wide_tokens=1, temperature=1.0, logits=1 << 40, stride=40000,
             token=1 << 41, tokens_stride=2, logprobs=1 << 42, entropy=1 << 43, top_ids=1 << 44, top_logprobs=1 << 45,
             workspace=1 << 46, workspace_bytes=1 << 20)
    a.update(kw)
    L = gfr_moe.lib()
    refused(L.gfr_logprobs_run(None, gfr_moe._LOGPROBS.pack(*[a[n] for n in LOGPROBS])), needle)
    refused(L.gfr_logprobs_run(None, None), "null")


def test_logprobs_workspace():
    """Enough for every chunk's sums and places, and refused for what a run refuses."""
    import gfr_moe
    L = gfr_moe.lib()
    for rows, vocab, top in ((1, 1, 0), (5, 32768, 32), (70000, 1000, 5)):
        assert L.gfr_logprobs_workspace(rows, vocab, top) == 0          # a row is one chunk
    assert L.gfr_logprobs_workspace(1, 160000, 20) >= 40 * (16 + 20 * 8)
    for rows, vocab in ((1, 1 << 21), (3, 32769), (4096, 160000)):
        chunks = L.gfr_logprobs_workspace(rows, vocab, 0) // (16 * rows)
        assert 2 <= chunks <= 64 and chunks * 32768 >= vocab
        assert L.gfr_logprobs_workspace(rows, vocab, 32) == rows * chunks * (16 + 32 * 8)
    assert L.gfr_logprobs_workspace(0, 10, 0) < 0 and L.gfr_logprobs_workspace(1, 10, 11) < 0


EXPERTS = ("rows slots hidden inter experts type act limit residual_type out_type x x_stride gu gu_stride gu_expert down "
           "down_stride down_expert picks weights residual residual_stride out out_stride workspace workspace_bytes").split()


@pytest.mark.parametrize("kw,needle", [
    (dict(rows=0), "rows 0"), (dict(slots=0), "slots 0"), (dict(rows=8193, slots=8), "65536 pairs"), (dict(hidden=0), "hidden 0"),
    (dict(inter=-1), "inter -1"), (dict(hidden=(1 << 20) + 1), "outside"), (dict(experts=0), "experts 0"),
    (dict(experts=65537), "experts 65537"), (dict(x=0), "null"), (dict(gu=0), "null"), (dict(down=0), "null"), (dict(picks=0), "null"),
    (dict(weights=0), "null"), (dict(out=0), "null"), (dict(workspace=0), "null"), (dict(type=2), "type 2"),
    (dict(out_type=1), "x's type or fp32"), (dict(residual=1 << 50, residual_type=1), "x's type or fp32"), (dict(act=5), "activation 5"),
    (dict(limit=-1.0), "limit"), (dict(limit=float("nan")), "limit"), (dict(x_stride=63), "stride of x 63"),
    (dict(gu_stride=63), "gu 63"), (dict(down_stride=31), "down 31"), (dict(out_stride=63), "out 63"),
    (dict(residual=1 << 50, residual_stride=63), "residual 63"), (dict(x_stride=(1 << 31) + 1), "2^31"), (dict(gu_expert=-1), "between experts"),
    (dict(down_expert=(1 << 40) + 1), "between experts"), (dict(x=(1 << 40) + 1), "aligned"), (dict(picks=(1 << 43) + 2), "aligned"),
    (dict(out=(1 << 45) + 2, out_type=2), "aligned"), (dict(workspace=(1 << 46) + 8), "16-byte"), (dict(workspace_bytes=100), "workspace of 100"),
    (dict(rows=65536, slots=1, hidden=1 << 20, experts=65536, x_stride=1 << 20, gu_stride=1 << 20, out_stride=1 << 20,
          workspace_bytes=1 << 62), "too many"),
    (dict(out=1 << 40), "overlaps x"), (dict(out=(1 << 41) + 1000), "overlaps gu"), (dict(out=1 << 42), "overlaps down"),
    (dict(out=1 << 43), "overlaps picks"), (dict(out=1 << 44), "overlaps weights"), (dict(workspace=1 << 41), "workspace overlaps gu"),
    (dict(workspace=(1 << 45) + 16), "out overlaps the workspace"), (dict(residual=1 << 45, residual_stride=65), "not the residual itself"),
    (dict(residual=1 << 46), "workspace overlaps the residual"),
])
def test_experts16_refuses(kw, needle):
    import gfr_moe
    a = dict(rows=4, slots=2, hidden=64, inter=32, experts=5, type=0, act=4, limit=0.0, residual_type=0, out_type=0, x=1 << 40,
             x_stride=64, gu=1 << 41, gu_stride=64, gu_expert=64 * 64, down=1 << 42, down_stride=32, down_expert=64 * 32,
             picks=1 << 43, weights=1 << 44, residual=0, residual_stride=64, out=1 << 45, out_stride=64, workspace=1 << 46,
             workspace_bytes=1 << 20)
    a.update(kw)
    L = gfr_moe.lib()
    refused(L.gfr_experts16_run(None, gfr_moe._EXPERTS16.pack(*[a[n] for n in EXPERTS])), needle)
    refused(L.gfr_experts16_run(None, None), "null")


def test_experts16_workspace():
    """Room for the activations' two parts, padded to whole chunks, and the pairs' outputs."""
    import gfr_moe
    L = gfr_moe.lib()
    assert L.gfr_experts16_workspace(3, 2, 65, 65) >= 6 * (2 * 2 * 128 + 4 * 68)
    assert L.gfr_experts16_workspace(8192, 8, 4096, 512) > 0 and L.gfr_experts16_workspace(8193, 8, 4096, 512) < 0
