"""GPU: linear attention with a decay for each head, prompts and single tokens
(include/mamba_lm_ops.h), against the recurrence in float64.

Tolerances. Let A be the same recurrence over absolute values (|q|, |k|, |v|,
|h0|): the sum of the magnitudes an output adds up. A float32 evaluation
rounds each product and partial sum by at most 2^-24 of it, at most L + dk + 64
times along any path to an output, and the products of operands split in two
half-precision parts drop or round at most 3 * 2^-22 of themselves, twice (the
scores, then the values): 2^-19 A covers both products. So float32 results and
all states stay within (2^-19 + (L + dk + 64) 2^-24) A. With 16-bit inputs the
scores, or the state, are rounded once more to 11 bits on their way into an
output, 2^-12 A (2^-11 A with the rounding of elements far below their row's
largest), and the output itself by half a step, eps / 2 of its value.
"""
import pytest
import torch

from mamba_onnx import cuda

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def recurrence(q, k, v, g, h0, lengths, scale):
    """float64: outputs and final state."""
    q, k, v = q.double(), k.double(), v.double()
    B, L, G, dk = q.shape
    H, dv = v.shape[2:]
    a = torch.exp(g.double()).expand(B, L, H)
    S = torch.zeros(B, H, dk, dv, dtype=torch.float64, device=q.device) if h0 is None \
        else h0.double().clone()
    out = torch.zeros(B, L, H, dv, dtype=torch.float64, device=q.device)
    rep = H // G
    n = torch.full((B,), L, device=q.device) if lengths is None else lengths.clamp(0, L)
    for t in range(L):
        on = (t < n)[:, None, None, None]
        kt = k[:, t].repeat_interleave(rep, 1)[..., :, None]
        qt = q[:, t].repeat_interleave(rep, 1)
        new = a[:, t, :, None, None] * S + kt * v[:, t][..., None, :]
        S = torch.where(on, new, S)
        o = scale * torch.einsum("bhk,bhkv->bhv", qt, S)
        out[:, t] = torch.where(on[..., 0], o, torch.zeros_like(o))
    return out, S


def check(q, k, v, g, h0=None, lengths=None, scale=None, out=None, h_last=None):
    """Compares out and h_last with the recurrence of the same inputs."""
    B, L, G, dk = q.shape
    s = dk ** -0.5 if scale is None else scale
    ref, ref_s = recurrence(q, k, v, g, h0, lengths, s)
    mag, mag_s = recurrence(q.abs(), k.abs(), v.abs(), g, None if h0 is None else h0.abs(),
                            lengths, abs(s))
    tol32 = 2.0 ** -19 + (L + dk + 64) * 2.0 ** -24
    eps = torch.finfo(out.dtype).eps
    if out.dtype == torch.float32:
        bound = tol32 * mag
    else:
        # fp16's smallest step, 2^-24, rounds results below its normal range
        bound = eps / 2 * ref.abs() + (tol32 + 2.0 ** -11) * mag + 2.0 ** -25
    assert out.shape == ref.shape
    # a value past the type's largest by half a step or more rounds to infinity
    # (fp16: 65504 + 16), one within its bound of that border may
    border = torch.finfo(out.dtype).max * (1 + eps / 4)
    high = ref.abs() + bound >= border
    assert bool((torch.isinf(out) <= high).all())
    assert bool((torch.isinf(out) | (ref.abs() - bound < border)).all())
    assert bool((torch.signbit(out) == torch.signbit(ref))[high].all())
    err = (out.double() - ref).abs().masked_fill(torch.isinf(out), 0)
    assert bool((err <= bound + 1e-37).all()), \
        f"out off by {float((err / (bound + 1e-37)).max()):.3g} bounds"
    if h_last is not None:
        err = (h_last.double() - ref_s).abs()
        assert bool((err <= tol32 * mag_s + 1e-37).all()), \
            f"state off by {float((err / (tol32 * mag_s + 1e-37)).max()):.3g} bounds"


def inputs(B, L, H, G, dk, dv, dtype, seed=0, per_token=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    q, k, v = r(B, L, G, dk).to(dtype), r(B, L, G, dk).to(dtype), r(B, L, H, dv).to(dtype)
    g = -torch.rand(*((B, L, H) if per_token else (H,)), device="cuda", generator=gen).pow(4) * 3
    return q, k, v, g


def run(q, k, v, g, **kw):
    B, H, dk, dv = q.shape[0], v.shape[2], q.shape[3], v.shape[3]
    h_last = torch.full((B, H, dk, dv), float("nan"), device="cuda")
    out = cuda.linear_attention(q, k, v, g, h_last=h_last, **kw)
    return out, h_last


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L", [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 300])
def test_lengths_of_prompt(L, dtype):
    q, k, v, g = inputs(2, L, 4, 2, 64, 64, dtype, seed=L)
    out, h_last = run(q, k, v, g)
    check(q, k, v, g, out=out, h_last=h_last)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk,dv", [(1, 1), (3, 5), (8, 8), (16, 200), (17, 33), (32, 128),
                                   (48, 64), (64, 96), (72, 72), (100, 100), (128, 128),
                                   (128, 256), (129, 16), (200, 40), (256, 256)])
def test_head_sizes(dk, dv, dtype):
    q, k, v, g = inputs(2, 150, 3, 1, dk, dv, dtype, seed=dk * 300 + dv)
    h0 = torch.randn(2, 3, dk, dv, device="cuda")
    out, h_last = run(q, k, v, g, h0=h0)
    check(q, k, v, g, h0=h0, out=out, h_last=h_last)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,G", [(1, 1), (5, 5), (6, 2), (40, 8), (12, 1)])
def test_shared_heads_and_fixed_decays(H, G, dtype):
    q, k, v, g = inputs(1, 200, H, G, 64, 64, dtype, seed=H * 10 + G, per_token=False)
    out, h_last = run(q, k, v, g, scale=0.7)
    check(q, k, v, g, scale=0.7, out=out, h_last=h_last)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,L,H,dk,dv", [(1, 3000, 1, 128, 128), (1, 2049, 4, 64, 64),
                                         (2, 1111, 3, 96, 48), (1, 1300, 2, 100, 128)])
def test_few_heads_split_sequences(B, L, H, dk, dv, dtype):
    """Few (sequence, head) pairs over long sequences, with the states joined
    through the workspace, and the same in one piece."""
    q, k, v, g = inputs(B, L, H, H, dk, dv, dtype, seed=L)
    h0 = torch.randn(B, H, dk, dv, device="cuda")
    lengths = torch.tensor([L - 77] + [L] * (B - 1), dtype=torch.int32, device="cuda")
    for chunked in (True, False):
        out, h_last = run(q, k, v, g, h0=h0, lengths=lengths, chunked=chunked)
        check(q, k, v, g, h0=h0, lengths=lengths, out=out, h_last=h_last)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L", [40, 333])
def test_padded_rows_are_not_read(L, dtype):
    """Ragged lengths (0, 1, inside and at tile borders, out of range): NaN in
    every padded row of every input leaves no trace."""
    want = [0, 1, 16, 33, L - 1, L, L + 5, -3]
    B = len(want)
    q, k, v, g = inputs(B, L, 4, 2, 64, 80, dtype, seed=L)
    lengths = torch.tensor(want, dtype=torch.int32, device="cuda")
    pad = torch.arange(L, device="cuda")[None, :] >= lengths.clamp(0, L)[:, None]
    clean = [t.masked_fill(pad.view(B, L, *[1] * (t.dim() - 2)), 0) for t in (q, k, v, g)]
    dirty = [t.masked_fill(pad.view(B, L, *[1] * (t.dim() - 2)), float("nan"))
             for t in (q, k, v, g)]
    for h0 in (None, torch.randn(B, 4, 64, 80, device="cuda")):
        out, h_last = run(*dirty, h0=h0, lengths=lengths)
        check(*clean, h0=h0, lengths=lengths, out=out, h_last=h_last)
        assert bool((out[pad] == 0).all())
        assert torch.equal(h_last[0], torch.zeros_like(h_last[0]) if h0 is None else h0[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_resets_and_strong_decays(dtype):
    """log decays of -inf (the state is cleared), of the lowest value, of
    -1e30, of hundreds, and of 0 (nothing forgotten)."""
    q, k, v, g = inputs(2, 200, 4, 4, 64, 64, dtype, seed=3)
    g[:, 50] = float("-inf")
    g[:, 51] = torch.finfo(torch.float32).min
    g[:, 100:103] = float("-inf")
    g[0, 120:140] = -1e30
    g[1, 120:190] = -300.0
    g[:, 150:160, 0] = 0.0
    h0 = torch.randn(2, 4, 64, 64, device="cuda")
    out, h_last = run(q, k, v, g, h0=h0)
    check(q, k, v, g, h0=h0, out=out, h_last=h_last)


@pytest.mark.parametrize("dtype", DTYPES)
def test_uneven_magnitudes(dtype):
    """Rows of very different sizes (a few keys, values and queries hundreds of
    times the others, some of zeros) and long memories."""
    q, k, v, _ = inputs(1, 260, 2, 2, 128, 128, dtype, seed=9)
    g = torch.full((1, 260, 2), -1e-4, device="cuda")
    k[:, 10::50] *= 300
    v[:, 12::60] *= 200
    q[:, 15::40] *= 100
    k[:, 20:24] = 0
    v[:, 30:33] = 0
    q[:, 64:128] = 0
    out, h_last = run(q, k, v, g)
    check(q, k, v, g, out=out, h_last=h_last)


def test_tiny_and_large_float32_values():
    for exp in (-30, 12):
        q, k, v, g = inputs(1, 130, 2, 2, 64, 64, torch.float32, seed=1)
        k, v = k * 10.0 ** (exp / 2), v * 10.0 ** (exp / 2)
        h0 = torch.randn(1, 2, 64, 64, device="cuda") * 10.0 ** exp
        out, h_last = run(q, k, v, g, h0=h0)
        check(q, k, v, g, h0=h0, out=out, h_last=h_last)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["fused", "heads_first", "offset", "odd_stride", "expanded"])
def test_strides(layout, dtype):
    """Inputs that are views: slices of one projection's output, heads before
    rows, bases off 16 bytes, row strides off 16 bytes, broadcast batches."""
    B, L, H, G, dk, dv = 2, 140, 4, 2, 64, 48
    q, k, v, g = inputs(B, L, H, G, dk, dv, dtype, seed=5)
    if layout == "fused":
        buf = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], -1)
        q, k, v = buf.split([G * dk, G * dk, H * dv], -1)
        q, k, v = q.unflatten(-1, (G, dk)), k.unflatten(-1, (G, dk)), v.unflatten(-1, (H, dv))
        g = torch.stack([g, g + 1], -1)[..., 0]
    elif layout == "heads_first":
        q, k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))
        g = g.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    elif layout == "offset":
        def shift(t):
            buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
            buf[1:] = t.flatten()
            return buf[1:].view(t.shape)
        q, k, v, g = shift(q), shift(k), shift(v), shift(g)
    elif layout == "odd_stride":
        def widen(t):
            buf = torch.zeros(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device=t.device)
            buf[..., :t.shape[-1]] = t
            return buf[..., :t.shape[-1]]
        q, k, v = widen(q), widen(k), widen(v)
    else:
        q, k = q[:1].expand(B, L, G, dk), k[:, :1].expand(B, L, G, dk)
    out, h_last = run(q, k, v, g)
    check(q, k, v, g, out=out, h_last=h_last)


def test_offsets_past_32_bits():
    """Batch strides of more than 2^31 elements."""
    B, L, H, dk = 2, 70, 2, 64
    far = 2 ** 31 + 64
    buf = torch.empty(far + 3 * L * H * dk, dtype=torch.bfloat16, device="cuda")
    q0, k0, v0, g = inputs(B, L, H, H, dk, dk, torch.bfloat16, seed=2)
    views = []
    for i, t in enumerate((q0, k0, v0)):
        w = buf.as_strided((B, L, H, dk), (far, H * dk, dk, 1), i * L * H * dk)
        w.copy_(t)
        views.append(w)
    out, h_last = run(*views, g)
    check(q0, k0, v0, g, out=out, h_last=h_last)


@pytest.mark.parametrize("L", [0, 5])
@pytest.mark.parametrize("B", [0, 2])
def test_empty(B, L):
    q, k, v, g = inputs(B, L, 2, 1, 64, 64, torch.float32)
    h0 = torch.randn(B, 2, 64, 64, device="cuda")
    out, h_last = run(q, k, v, g, h0=h0)
    assert out.shape == (B, L, 2, 64)
    if L == 0:
        assert torch.equal(h_last, h0)
        out, h_last = run(q, k, v, g)
        assert torch.equal(h_last, torch.zeros_like(h0))


def test_repeated_calls_are_bit_identical():
    for B, L, H in ((4, 500, 20), (1, 4000, 2)):
        q, k, v, g = inputs(B, L, H, H, 128, 128, torch.bfloat16, seed=4)
        a, sa = run(q, k, v, g)
        b, sb = run(q, k, v, g)
        assert torch.equal(a, b) and torch.equal(sa, sb)


def test_other_stream_and_captured_graphs():
    """A side stream, and two captured graphs replayed in turn, each with its
    own workspace; both shapes split their sequences."""
    calls = []
    for seed, L in ((1, 1500), (2, 2300)):
        q, k, v, g = inputs(1, L, 2, 2, 64, 64, torch.float32, seed=seed)
        calls.append((q, k, v, g, *run(q, k, v, g)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for q, k, v, g, out, h_last in calls:
        got = cuda.linear_attention(q, k, v, g, stream=side)
        side.synchronize()
        assert torch.equal(got, out)
    graphs = []
    for q, k, v, g, out, h_last in calls:
        o, s = torch.zeros_like(out), torch.zeros_like(h_last)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cuda.linear_attention(q, k, v, g, out=o, h_last=s)
        graphs.append((graph, o, s))
    for _ in range(2):
        for graph, o, s in graphs:
            o.zero_()
            graph.replay()
        torch.cuda.synchronize()
        for (_, o, s), (*_, out, h_last) in zip(graphs, calls):
            assert torch.equal(o, out) and torch.equal(s, h_last)


# ------------------------------------------------------------- single tokens


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,G,dk,dv", [(1, 1, 1, 1, 1), (1, 24, 24, 64, 64), (3, 4, 2, 100, 36),
                                         (7, 12, 3, 80, 72), (2, 2, 1, 256, 256), (5, 3, 3, 33, 17),
                                         (64, 8, 8, 128, 128)])
@pytest.mark.parametrize("in_place", [True, False])
def test_step(B, H, G, dk, dv, dtype, in_place):
    q, k, v, g = inputs(B, 1, H, G, dk, dv, dtype, seed=B + dk)
    state = torch.randn(B, H, dk, dv, device="cuda")
    before = state.clone()
    new = state if in_place else torch.full_like(state, float("nan"))
    out = cuda.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], state,
                                     state_out=None if in_place else new)
    check(q, k, v, g, h0=before, out=out[:, None], h_last=new)
    if not in_place:
        assert torch.equal(state, before)


@pytest.mark.parametrize("dtype", DTYPES)
def test_step_strides_fixed_decays_and_unaligned_state(dtype):
    B, H, G, dk, dv = 3, 4, 2, 64, 64
    q, k, v, g = inputs(B, 1, H, G, dk, dv, dtype, seed=8, per_token=False)
    g[1] = float("-inf")
    g[2] = 0.0
    buf = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], -1)
    qs, ks, vs = buf.split([G * dk, G * dk, H * dv], -1)
    flat = torch.randn(B * H * dk * dv + 1, device="cuda")
    state = flat[1:].view(B, H, dk, dv)
    before = state.clone()
    out = cuda.linear_attention_step(qs.unflatten(-1, (G, dk)), ks.unflatten(-1, (G, dk)),
                                     vs.unflatten(-1, (H, dv)), g, state, scale=1.3)
    check(q, k, v, g, h0=before, scale=1.3, out=out[:, None], h_last=state)


def test_step_empty_batch_and_graph():
    q, k, v, g = inputs(0, 1, 2, 2, 16, 16, torch.float32)
    assert cuda.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0],
                                      torch.empty(0, 2, 16, 16, device="cuda")).shape == (0, 2, 16)
    q, k, v, g = inputs(2, 1, 4, 4, 64, 64, torch.bfloat16)
    state = torch.randn(2, 4, 64, 64, device="cuda")
    eager = state.clone()
    outs = [cuda.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], eager) for _ in range(3)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cuda.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], state)
    for want in outs:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert torch.equal(state, eager)


# ------------------------------------------------------------- refusals


def test_refusals():
    q, k, v, g = inputs(2, 8, 4, 2, 16, 16, torch.float32)
    ok = dict(q=q, k=k, v=v, log_decay=g)

    def refused(error, match, **change):
        with pytest.raises(error, match=match):
            cuda.linear_attention(**{**ok, **change})

    refused(ValueError, "k must have shape", k=k[:, :7])
    refused(TypeError, "v must be torch.float32", v=v.half())
    refused(TypeError, "float32, float16 or bfloat16", q=q.double())
    refused(TypeError, "q must be a CUDA tensor", q=q.cpu())
    refused(ValueError, "last dimension must be contiguous", v=torch.randn(2, 8, 16, 4, device="cuda")
            .transpose(2, 3))
    refused(ValueError, "log_decay must have shape", log_decay=g[:, :, :3])
    refused(TypeError, "log_decay must be torch.float32", log_decay=g.half())
    refused(TypeError, "lengths must be torch.int32", lengths=torch.ones(2, dtype=torch.int64,
                                                                         device="cuda"))
    refused(ValueError, "h0 must have shape", h0=torch.zeros(2, 4, 16, 17, device="cuda"))
    refused(ValueError, "out must be contiguous",
            out=torch.empty(2, 4, 8, 16, device="cuda").transpose(1, 2))
    refused(cuda.ScanError, "groups must divide heads",
            v=torch.randn(2, 8, 3, 16, device="cuda"), log_decay=g[:, :, :3])
    refused(cuda.ScanError, "dk and dv must be", v=torch.randn(2, 8, 4, 257, device="cuda"))
    refused(cuda.ScanError, "out overlaps an input", out=v)
    h = torch.zeros(2, 4, 16, 16, device="cuda")
    refused(cuda.ScanError, "h_last overlaps an input", h0=h, h_last=h)
    state = torch.zeros(2 * 4 * 16 * 16 + 4, device="cuda")
    with pytest.raises(cuda.ScanError, match="state_out must be state or not overlap"):
        cuda.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0],
                                   state[:-4].view(2, 4, 16, 16),
                                   state_out=state[4:].view(2, 4, 16, 16))
    assert cuda.check_device_error() == 0


def test_refuses_heads_without_elements():
    q, k, v, g = inputs(2, 8, 4, 2, 16, 16, torch.float32)
    none = q[..., :0]
    with pytest.raises(cuda.ScanError, match="dk and dv must be"):
        cuda.linear_attention(none, none, v, g)
    with pytest.raises(cuda.ScanError, match="dk and dv must be"):
        cuda.linear_attention_step(none[:, 0], none[:, 0], v[:, 0], g[:, 0],
                                   torch.zeros(2, 4, 0, 16, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,L,H,dk,dv", [(1, 33, 2, 129, 64), (2, 200, 3, 136, 128),
                                         (1, 1000, 2, 256, 256), (1, 129, 160, 192, 72),
                                         (3, 100, 40, 161, 130)])
def test_more_than_128_keys(B, L, H, dk, dv, dtype):
    """Heads whose keys are served in two halves: whole and split sequences, odd
    sizes, padded rows of NaN, states before and after, with and without
    workspace. The bounds of a sum over dk keys hold for any order of it."""
    q, k, v, g = inputs(B, L, H, H, dk, dv, dtype, seed=dk + L)
    h0 = torch.randn(B, H, dk, dv, device="cuda")
    lengths = torch.tensor([L - 21] + [L] * (B - 1), dtype=torch.int32, device="cuda")
    pad = torch.arange(L, device="cuda")[None, :] >= lengths[:, None]
    dirty = [t.masked_fill(pad.view(B, L, *[1] * (t.dim() - 2)), float("nan"))
             for t in (q, k, v, g)]
    clean = [t.masked_fill(pad.view(B, L, *[1] * (t.dim() - 2)), 0) for t in (q, k, v, g)]
    for chunked in (True, False):
        out, h_last = run(*dirty, h0=h0, lengths=lengths, chunked=chunked)
        check(*clean, h0=h0, lengths=lengths, out=out, h_last=h_last)
        assert bool((out[pad] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_more_than_128_keys_in_views_graphs_and_shared_groups(dtype):
    B, L, H, G, dk, dv = 2, 150, 4, 2, 200, 100
    buf = torch.randn(B, L, 2 * G * dk + H * dv + 1, device="cuda").to(dtype)
    q, k, v = buf[..., 1:].split([G * dk, G * dk, H * dv], -1)
    q, k, v = q.unflatten(-1, (G, dk)), k.unflatten(-1, (G, dk)), v.unflatten(-1, (H, dv))
    g = -torch.rand(H, device="cuda")
    out, h_last = run(q, k, v, g)
    check(q, k, v, g, out=out, h_last=h_last)
    # a graph replayed over other values gives what a call does, every time
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured, captured_last = run(q, k, v, g)
    for seed in (1, 2):
        buf.copy_(torch.randn(buf.shape, device="cuda",
                              generator=torch.Generator(device="cuda").manual_seed(seed)))
        graph.replay()
        again, last = run(q, k, v, g)
        torch.cuda.synchronize()
        assert torch.equal(captured, again) and torch.equal(captured_last, last)
