"""GPU: linear attention split into segments (few heads, long sequences) where
lengths, tiles and layouts meet the segments' borders; tolerances and the
float64 recurrence as in test_linear_attention_cuda.py.
"""
import pytest
import torch

from mamba_onnx import cuda
from test_linear_attention_cuda import DTYPES, check, inputs, run

pytestmark = pytest.mark.gpu


def split(B, L, H, G, dk, dv, dtype):
    return cuda.linear_attention_workspace_size(B, L, H, G, dk, dv, dtype) > 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 128), (72, 200)])
def test_lengths_end_in_every_kind_of_segment(dk, dv, dtype):
    """Lengths of 0, 1, one chunk, inside and at the borders of segments, all;
    NaN in the padded rows; with and without states to start from."""
    L, H = 1000, 2
    want = [0, 1, 64, 65, 127, 128, 192, 500, 640, 999, 1000]
    B = len(want)
    assert split(B, L, H, 1, dk, dv, dtype)
    q, k, v, g = inputs(B, L, H, 1, dk, dv, dtype, seed=dk + dv)
    lengths = torch.tensor(want, dtype=torch.int32, device="cuda")
    pad = torch.arange(L, device="cuda")[None, :] >= lengths[:, None]
    clean = [t.masked_fill(pad.view(B, L, *[1] * (t.dim() - 2)), 0) for t in (q, k, v, g)]
    dirty = [t.masked_fill(pad.view(B, L, *[1] * (t.dim() - 2)), float("nan"))
             for t in (q, k, v, g)]
    for h0 in (None, torch.randn(B, H, dk, dv, device="cuda")):
        out, h_last = run(*dirty, h0=h0, lengths=lengths)
        check(*clean, h0=h0, lengths=lengths, out=out, h_last=h_last)
        assert bool((out[pad] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["odd_stride", "fused"])
def test_split_sequences_in_views(layout, dtype):
    """Segments of inputs that TMA cannot take (rows off 8 or 16 bytes) and of
    slices of one projection."""
    B, L, H, G, dk, dv = 1, 900, 3, 1, 100, 60
    q, k, v, g = inputs(B, L, H, G, dk, dv, dtype, seed=11)
    if layout == "odd_stride":
        def widen(t):
            buf = torch.zeros(*t.shape[:-1], t.shape[-1] + 1, dtype=t.dtype, device=t.device)
            buf[..., 1:] = t
            return buf[..., 1:]
        q, k, v = widen(q), widen(k), widen(v)
    else:
        buf = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], -1)
        q, k, v = buf.split([G * dk, G * dk, H * dv], -1)
        q, k, v = q.unflatten(-1, (G, dk)), k.unflatten(-1, (G, dk)), v.unflatten(-1, (H, dv))
    assert split(B, L, H, G, dk, dv, dtype)
    h0 = torch.randn(B, H, dk, dv, device="cuda")
    out, h_last = run(q, k, v, g, h0=h0)
    check(q, k, v, g, h0=h0, out=out, h_last=h_last)


@pytest.mark.parametrize("dtype", DTYPES)
def test_whole_units_beside_a_split_tail(dtype):
    """More units than the GPU holds at once: most run in one piece, the last
    partial wave in segments."""
    B, L, H, dk = 3, 1300, 52, 128
    q, k, v, g = inputs(B, L, H, 4, dk, dk, dtype, seed=6)
    assert split(B, L, H, 4, dk, dk, dtype)
    lengths = torch.tensor([L, 77, L - 1], dtype=torch.int32, device="cuda")
    out, h_last = run(q, k, v, g, lengths=lengths)
    check(q, k, v, g, lengths=lengths, out=out, h_last=h_last)


@pytest.mark.parametrize("dtype", DTYPES)
def test_resets_inside_and_between_segments(dtype):
    q, k, v, g = inputs(1, 1300, 1, 1, 64, 64, dtype, seed=8)
    for t in (63, 64, 127, 128, 640, 1024, 1299):
        g[:, t] = float("-inf")
    g[:, 300:420] = -1e9
    h0 = torch.randn(1, 1, 64, 64, device="cuda")
    assert split(1, 1300, 1, 1, 64, 64, dtype)
    out, h_last = run(q, k, v, g, h0=h0)
    check(q, k, v, g, h0=h0, out=out, h_last=h_last)


@pytest.mark.parametrize("dtype", DTYPES)
def test_very_long_sequence_agrees_with_one_piece(dtype):
    """100 000 rows: split and in one piece are the same sums in other order.
    Decays of 0.4 a row on average forget all but some hundred rows, so each is
    within the derived bound of 300 rows of the exact value: 2 (2^-19 + 500 *
    2^-24) of the magnitudes, which the recurrence over absolute values gives."""
    L = 100_000
    q, k, v, g = inputs(1, L, 2, 1, 64, 64, dtype, seed=12)
    a, sa = run(q, k, v, g)
    b, sb = run(q, k, v, g, chunked=False)
    mag, smag = run(q.abs().float(), k.abs().float(), v.abs().float(), g)
    tol = 2 * (2.0 ** -19 + 500 * 2.0 ** -24) * 1.01
    if dtype == torch.float32:
        assert bool(((a - b).abs() <= tol * mag).all())
    else:
        eps = torch.finfo(dtype).eps
        bound = (tol + 2.0 ** -10) * mag + eps * a.float().abs() + 2.0 ** -24
        assert bool(((a.float() - b.float()).abs() <= bound).all())
    assert bool(((sa - sb).abs() <= tol * smag).all())


def test_growing_decays_stay_finite():
    """log decays above 0: the state grows by e^0.02 a row."""
    for dtype in DTYPES:
        q, k, v, g = inputs(1, 300, 2, 2, 64, 64, dtype, seed=13)
        g = torch.full_like(g, 0.02)
        out, h_last = run(q, k, v, g)
        check(q, k, v, g, out=out, h_last=h_last)


@pytest.mark.parametrize("rows,V", [(1, 50280), (5, 20001)])
def test_logprob_clusters_in_a_graph(rows, V):
    """Few rows over a long vocabulary run on clusters of CTAs, captured too."""
    x = torch.randn(rows, V, device="cuda", generator=torch.Generator("cuda").manual_seed(V))
    t = torch.randint(0, V, (rows,), device="cuda")
    graph = torch.cuda.CUDAGraph()
    cuda.token_logprobs(x, t, top=7)
    with torch.cuda.graph(graph):
        got = cuda.token_logprobs(x, t, top=7)
    x.copy_(torch.randn(rows, V, device="cuda"))
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, cuda.token_logprobs(x, t, top=7)))
