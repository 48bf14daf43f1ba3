"""GPU: the gated delta rule, prompts and single tokens (include/mamba_lm_ops.h),
against the recurrence in float64.

Tolerances. With keys of norm at most 1 (their rounding aside) and beta in 0..1
a token maps a state column c to a (I - beta k k^T) c, which does not lengthen
it, so local errors add up without growing. An error in a row's value, in what
the state holds under its key or in a score against an earlier row u_s of its
chunk enters like a change of the row's value, beta |k| times its size at most.
Sums of up to n terms in float32 carry at most n 2^-24 of their terms'
magnitudes, and by Cauchy's inequality those of k c are at most |k| |c|; a
product of operands split in two half-precision parts drops or rounds at most
3 * 2^-22 of itself, 8 * 2^-22 where the first part is cut off, not rounded (2^-20
for the low parts' product, 2^-21 for each low part's rounding), and 2 * 2^-22 of
those with one such operand and one exact. A row passes four of them: the scores
(3, or exact for 16-bit rows), the inverse's (3), T R (3, or 8) and K^T U (3, or
2), 12 or 13 * 2^-22, which 2^-18 covers. So with
  e = 2^-18 + (dk + 128) 2^-24
a column's error after token t, as a norm, is at most
  E_t = a_t E_{t-1} + e (2 |c_t'| + |v_t| + sum of |u_s| over the last 64 rows),
c' the decayed column, and an output's
  scale |q| (E_t + e (|c_t| + sum of |u_s|)) + half a step of its type.
"""
import pytest
import torch

from mamba_onnx import cuda

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def recurrence(q, k, v, g, beta, h0, lengths, scale):
    """float64: outputs, final state, and both errors' bounds."""
    q, k, v = q.double(), k.double(), v.double()
    B, L, G, dk = q.shape
    H, dv = v.shape[2:]
    kw = dict(dtype=torch.float64, device=q.device)
    a = torch.exp(g.double()).expand(B, L, H)
    beta = beta.double().expand(B, L, H)
    S = torch.zeros(B, H, dk, dv, **kw) if h0 is None else h0.double().clone()
    E = torch.zeros(B, H, dv, **kw)
    e = 2.0 ** -18 + (dk + 128) * 2.0 ** -24
    out, out_e = torch.zeros(B, L, H, dv, **kw), torch.zeros(B, L, H, dv, **kw)
    us = torch.zeros(B, max(L, 1), H, dv, **kw)
    rep = H // G
    n = torch.full((B,), L, device=q.device) if lengths is None else lengths.clamp(0, L)
    for t in range(L):
        on = (t < n)[:, None, None, None]
        kt = k[:, t].repeat_interleave(rep, 1)
        qt = q[:, t].repeat_interleave(rep, 1)
        D = torch.nan_to_num(a[:, t, :, None, None] * S)
        u = beta[:, t, :, None] * (v[:, t] - torch.einsum("bhk,bhkv->bhv", kt, D))
        us[:, t] = u.abs()
        near = us[:, max(0, t - 63):t + 1].sum(1)
        new = D + kt[..., :, None] * u[..., None, :]
        En = a[:, t, :, None] * E + e * (2 * D.norm(dim=2) + v[:, t].abs() + near)
        S, E = torch.where(on, new, S), torch.where(on[..., 0], En, E)
        o = scale * torch.einsum("bhk,bhkv->bhv", qt, S)
        oe = abs(scale) * qt.norm(dim=-1)[..., None] * (E + e * (S.norm(dim=2) + near))
        out[:, t] = torch.where(on[..., 0], o, torch.zeros_like(o))
        out_e[:, t] = torch.where(on[..., 0], oe, torch.zeros_like(o))
    return out, S, out_e, E


def check(q, k, v, g, beta, h0=None, lengths=None, scale=None, out=None, h_last=None):
    s = q.shape[-1] ** -0.5 if scale is None else scale
    ref, ref_s, bound, bound_s = recurrence(q, k, v, g, beta, h0, lengths, s)
    if out.dtype != torch.float32:  # (2^-25: fp16's smallest step)
        bound = bound + torch.finfo(out.dtype).eps / 2 * (ref.abs() + bound) + 2.0 ** -25
    assert out.shape == ref.shape
    err = (out.double() - ref).abs()
    assert bool((err <= bound + 1e-37).all()), \
        f"out off by {float((err / (bound + 1e-37)).max()):.3g} bounds"
    if h_last is not None:
        err = (h_last.double() - ref_s).abs()
        bound_s = bound_s[:, :, None]
        assert bool((err <= bound_s + 1e-37).all()), \
            f"state off by {float((err / (bound_s + 1e-37)).max()):.3g} bounds"


def inputs(B, L, H, G, dk, dv, dtype, seed=0, per_token=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kw = dict(device="cuda", generator=gen)
    q = torch.randn(B, L, G, dk, **kw).to(dtype)
    k = torch.randn(B, L, G, dk, **kw)
    k = (k / k.norm(dim=-1, keepdim=True).clamp(min=1e-30)).to(dtype)
    v = torch.randn(B, L, H, dv, **kw).to(dtype)
    lead = (B, L, H) if per_token else (H,)
    g = -torch.rand(*lead, **kw).pow(4) * 3
    return q, k, v, g, torch.rand(*lead, **kw)


def run(q, k, v, g, beta, **kw):
    B, H, dk, dv = q.shape[0], v.shape[2], q.shape[3], v.shape[3]
    h_last = torch.full((B, H, dk, dv), float("nan"), device="cuda")
    out = cuda.gated_delta_rule(q, k, v, g, beta, h_last=h_last, **kw)
    return out, h_last


def no_timeout():
    assert cuda.check_device_error() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L", [1, 2, 15, 16, 17, 48, 49, 63, 64, 65, 127, 129, 300])
def test_lengths_of_prompt(L, dtype):
    args = inputs(2, L, 4, 2, 64, 64, dtype, seed=L)
    out, h_last = run(*args)
    check(*args, out=out, h_last=h_last)
    no_timeout()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk,dv", [(1, 1), (3, 5), (8, 8), (16, 200), (17, 33), (32, 128),
                                   (48, 64), (64, 96), (72, 72), (100, 100), (128, 128),
                                   (128, 256), (129, 16), (200, 40), (256, 256)])
def test_head_sizes(dk, dv, dtype):
    args = inputs(2, 150, 3, 1, dk, dv, dtype, seed=dk * 300 + dv)
    h0 = torch.randn(2, 3, dk, dv, device="cuda")
    out, h_last = run(*args, h0=h0)
    check(*args, h0=h0, out=out, h_last=h_last)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (40, 24), (128, 40)])
def test_token_by_token_and_chunks(dk, dv, dtype):
    """Without a workspace the prompt runs token by token; both follow the rule."""
    args = inputs(1, 200, 4, 2, dk, dv, dtype, seed=dk)
    for chunked in (True, False):
        out, h_last = run(*args, chunked=chunked)
        check(*args, out=out, h_last=h_last)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,G", [(1, 1), (5, 5), (6, 2), (40, 8), (12, 1)])
def test_shared_heads_and_fixed_decays(H, G, dtype):
    args = inputs(1, 200, H, G, 64, 64, dtype, seed=H * 10 + G, per_token=False)
    out, h_last = run(*args, scale=0.7)
    check(*args, scale=0.7, out=out, h_last=h_last)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_heads(dtype):
    """More (sequence, head) pairs than SMs, both widths of a dv tile."""
    for dk, dv in ((128, 128), (128, 112), (64, 64)):
        args = inputs(4, 130, 64, 64, dk, dv, dtype, seed=dv)
        out, h_last = run(*args)
        check(*args, out=out, h_last=h_last)


@pytest.mark.parametrize("dtype", DTYPES)
def test_correlated_keys(dtype):
    """Keys that repeat or nearly do, beta 1 and no decay: the chunk's system is
    far from the identity, the updates cancel what earlier rows wrote."""
    q, k, v, g, beta = inputs(1, 260, 2, 2, 64, 64, dtype, seed=9)
    k[:, 1:] = torch.nn.functional.normalize(
        k[:, :1].float() + 0.05 * k[:, 1:].float(), dim=-1).to(dtype)
    k[:, 70:140] = k[:, 70:71]
    g, beta = torch.zeros_like(g), torch.ones_like(beta)
    out, h_last = run(q, k, v, g, beta)
    check(q, k, v, g, beta, out=out, h_last=h_last)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_prompt_in_several_launches(dtype):
    """So many chunks that the records of one launch do not hold them: the
    states go from launch to launch; with lengths that end in the first one."""
    B, L, H = 2, 4000, 80
    q, k, v, g, beta = inputs(B, L, H, 4, 32, 32, dtype, seed=5)
    h0 = torch.randn(B, H, 32, 32, device="cuda")
    lengths = torch.tensor([L, 100], dtype=torch.int32, device="cuda")
    size = cuda.gated_delta_rule_workspace_size
    assert size(B, 64 * L, H, 4, 32, 32, dtype) < 2 * size(B, 8 * L, H, 4, 32, 32, dtype)
    out, h_last = run(q, k, v, g, beta, h0=h0, lengths=lengths)
    check(q, k, v, g, beta, h0=h0, lengths=lengths, out=out, h_last=h_last)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,L", [(1, 3, 5000), (1, 2, 12400), (8, 80, 2000)])
def test_three_launches_and_more(B, H, L, dtype):
    """Records' buffers are used again from the third launch on; sequences end in
    any of them. Twice, in one workspace, where the second call finds the first one's
    records in every buffer, and captured."""
    q, k, v, g, beta = inputs(B, L, H, 1, 32, 32, dtype, seed=5)
    h0 = torch.randn(B, H, 32, 32, device="cuda")
    lengths = torch.randint(0, L + 1, (B,), dtype=torch.int32, device="cuda",
                            generator=torch.Generator(device="cuda").manual_seed(1))
    lengths[0] = L
    size = cuda.gated_delta_rule_workspace_size(B, L, H, 1, 32, 32, dtype)
    chunk = cuda.gated_delta_rule_workspace_size(B, 64, H, 1, 32, 32, dtype)
    assert 2 * (size - h0.numel() * 4) // (2 * chunk) < (L + 63) // 64  # (two launches' chunks)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    out, h_last = run(q, k, v, g, beta, h0=h0, lengths=lengths, workspace=ws)
    check(q, k, v, g, beta, h0=h0, lengths=lengths, out=out, h_last=h_last)
    again, s = run(q, k, v, g, beta, h0=h0, lengths=lengths, workspace=ws)
    assert torch.equal(again, out) and torch.equal(s, h_last)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cuda.gated_delta_rule(q, k, v, g, beta, h0=h0, lengths=lengths, out=again, h_last=s,
                              workspace=ws)
    again.zero_(), s.zero_()
    for _ in range(3):  # (back to back: the next one's first launch waits for this one)
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, out) and torch.equal(s, h_last)
    no_timeout()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,dk,dv,L", [(50, 4, 64, 64, 700), (5, 32, 40, 24, 1030),
                                         (10, 10, 128, 200, 515)])
def test_more_heads_than_sms(B, H, dk, dv, L, dtype):
    """More tiles of heads than SMs, many chunks, sequences that end early; twice
    in the same workspace, and captured."""
    q, k, v, g, beta = inputs(B, L, H, 2, dk, dv, dtype, seed=B)
    h0 = torch.randn(B, H, dk, dv, device="cuda")
    lengths = torch.randint(0, L + 1, (B,), dtype=torch.int32, device="cuda",
                            generator=torch.Generator(device="cuda").manual_seed(B))
    lengths[:4] = torch.tensor([0, 1, L, 256])
    ws = torch.full((cuda.gated_delta_rule_workspace_size(B, L, H, 2, dk, dv, dtype),), 255,
                    dtype=torch.uint8, device="cuda")
    out, h_last = run(q, k, v, g, beta, h0=h0, lengths=lengths, workspace=ws)
    check(q, k, v, g, beta, h0=h0, lengths=lengths, out=out, h_last=h_last)
    other, _ = run(q, k, v, g, beta, workspace=ws)  # another call's records
    again, s = run(q, k, v, g, beta, h0=h0, lengths=lengths, workspace=ws)
    assert torch.equal(again, out) and torch.equal(s, h_last)
    graph = torch.cuda.CUDAGraph()
    got = torch.zeros_like(out)
    with torch.cuda.graph(graph):
        cuda.gated_delta_rule(q, k, v, g, beta, out=got, workspace=ws)
    for _ in range(2):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, other)
    no_timeout()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L", [10, 40, 333])
def test_padded_rows_are_not_read(L, dtype):
    want = [0, 1, 16, 33, L - 1, L, L + 5, -3]
    B = len(want)
    args = inputs(B, L, 4, 2, 64, 80, dtype, seed=L)
    lengths = torch.tensor(want, dtype=torch.int32, device="cuda")
    pad = torch.arange(L, device="cuda")[None, :] >= lengths.clamp(0, L)[:, None]
    clean = [t.masked_fill(pad.view(B, L, *[1] * (t.dim() - 2)), 0) for t in args]
    dirty = [t.masked_fill(pad.view(B, L, *[1] * (t.dim() - 2)), float("nan")) for t in args]
    for h0 in (None, torch.randn(B, 4, 64, 80, device="cuda")):
        out, h_last = run(*dirty, h0=h0, lengths=lengths)
        check(*clean, h0=h0, lengths=lengths, out=out, h_last=h_last)
        assert bool((out[pad] == 0).all())
        assert torch.equal(h_last[0], torch.zeros_like(h_last[0]) if h0 is None else h0[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_resets_and_strong_decays(dtype):
    """log decays of -inf (the state is cleared), of the lowest value, of
    -1e30, of hundreds, and of 0; beta of 0 (nothing written) and 1."""
    q, k, v, g, beta = inputs(2, 200, 4, 4, 64, 64, dtype, seed=3)
    g[:, 50] = float("-inf")
    g[:, 51] = torch.finfo(torch.float32).min
    g[:, 100:103] = float("-inf")
    g[0, 120:140] = -1e30
    g[1, 120:190] = -300.0
    g[:, 150:160, 0] = 0.0
    beta[:, 20:30] = 0.0
    beta[:, 60:90] = 1.0
    beta[:, 130:200, 1] = 0.0
    h0 = torch.randn(2, 4, 64, 64, device="cuda")
    out, h_last = run(q, k, v, g, beta, h0=h0)
    check(q, k, v, g, beta, h0=h0, out=out, h_last=h_last)


@pytest.mark.parametrize("dtype", DTYPES)
def test_uneven_magnitudes(dtype):
    """Values and queries of very different sizes, keys of zero and of tiny norm."""
    q, k, v, g, beta = inputs(1, 260, 2, 2, 128, 128, dtype, seed=9)
    g = torch.full_like(g, -1e-4)
    v[:, 12::60] *= 200
    q[:, 15::40] *= 100
    k[:, 20:24] = 0
    k[:, 40:50] *= 2.0 ** -10
    v[:, 30:33] = 0
    q[:, 64:128] = 0
    out, h_last = run(q, k, v, g, beta)
    check(q, k, v, g, beta, out=out, h_last=h_last)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (64, 200), (24, 20)])
def test_large_values_forgotten_within_a_chunk(dk, dv, dtype):
    """One row's values 2^20 times the others', and a reset 20 rows on: the parts of
    the values and updates keep to 2^-39 of the largest, a value of 2^22 of the
    others' size, so 2^-17 of one value, twice (V and U); as norms, with what the
    operands leave otherwise (2^-18), the state and the later outputs are off by less
    than 2^-15, where an update scaled by less than its own largest element left
    2^-10."""
    q, k, v, g, beta = inputs(2, 64, 4, 2, dk, dv, dtype, seed=dk)
    v = v * 2.0 ** -7
    v[:, 10] *= 2.0 ** 20
    g[:, 30] = float("-inf")
    out, h_last = run(q, k, v, g, beta)
    ref, ref_s, _, _ = recurrence(*(x[:, 30:] for x in (q, k, v, g, beta)), None, None, dk ** -0.5)
    assert float((h_last.double() - ref_s).norm() / ref_s.norm()) < 2.0 ** -15
    eps = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps
    err = float((out[:, 30:].double() - ref).norm() / ref.norm())
    assert err < 2.0 ** -15 + eps / 2 / 3 ** 0.5


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rate", [0.05, 0.1, 0.2, 0.3])
def test_growing_states(rate, dtype):
    """Positive log decays, by which the state grows up to 2^14 within a chunk (parts
    to 2^-39 of a chunk's largest factor, so all of a factor's 22 bits stay up to
    2^17): errors grow with the state, as the bound has them."""
    q, k, v, g, beta = inputs(2, 130, 4, 2, 64, 64, dtype, seed=9)
    g = torch.rand_like(g) * rate
    out, h_last = run(q, k, v, g, beta, scale=2.0 ** -17)
    check(q, k, v, g, beta, scale=2.0 ** -17, out=out, h_last=h_last)


def test_tiny_and_large_float32_values():
    for exp in (-30, 12):
        q, k, v, g, beta = inputs(1, 130, 2, 2, 64, 64, torch.float32, seed=1)
        v = v * 10.0 ** exp
        h0 = torch.randn(1, 2, 64, 64, device="cuda") * 10.0 ** exp
        out, h_last = run(q, k, v, g, beta, h0=h0)
        check(q, k, v, g, beta, h0=h0, out=out, h_last=h_last)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["fused", "heads_first", "offset", "odd_stride", "expanded"])
def test_strides(layout, dtype):
    B, L, H, G, dk, dv = 2, 140, 4, 2, 64, 48
    q, k, v, g, beta = inputs(B, L, H, G, dk, dv, dtype, seed=5)
    if layout == "fused":
        buf = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], -1)
        q, k, v = buf.split([G * dk, G * dk, H * dv], -1)
        q, k, v = q.unflatten(-1, (G, dk)), k.unflatten(-1, (G, dk)), v.unflatten(-1, (H, dv))
        both = torch.stack([g, beta], -1)
        g, beta = both[..., 0], both[..., 1]
    elif layout == "heads_first":
        q, k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))
        g, beta = (t.permute(2, 0, 1).contiguous().permute(1, 2, 0) for t in (g, beta))
    elif layout == "offset":
        def shift(t):
            buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
            buf[1:] = t.flatten()
            return buf[1:].view(t.shape)
        q, k, v, g, beta = (shift(t) for t in (q, k, v, g, beta))
    elif layout == "odd_stride":
        def widen(t):
            buf = torch.zeros(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device=t.device)
            buf[..., :t.shape[-1]] = t
            return buf[..., :t.shape[-1]]
        q, k, v = widen(q), widen(k), widen(v)
    else:
        q, k = q[:1].expand(B, L, G, dk), k[:, :1].expand(B, L, G, dk)
        beta = beta[:1, :1].expand(B, L, H)
    out, h_last = run(q, k, v, g, beta)
    check(q, k, v, g, beta, out=out, h_last=h_last)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dv", [64, 200])
def test_output_at_any_address(dv, dtype):
    """Aligned inputs and an output that does not start at 16 bytes; what stands
    beside it is left as it was."""
    B, L, H = 2, 150, 4
    args = inputs(B, L, H, 2, 64, dv, dtype, seed=dv)
    lengths = torch.tensor([L, 70], dtype=torch.int32, device="cuda")
    buf = torch.full((B * L * H * dv + 2,), 7.0, dtype=dtype, device="cuda")
    out = buf[1:-1].view(B, L, H, dv)
    _, h_last = run(*args, lengths=lengths, out=out)
    check(*args, lengths=lengths, out=out, h_last=h_last)
    assert float(buf[0]) == 7.0 and float(buf[-1]) == 7.0


def test_offsets_past_32_bits():
    """Batch strides of more than 2^31 elements."""
    B, L, H, dk = 2, 70, 2, 64
    far = 2 ** 31 + 64
    buf = torch.empty(far + 3 * L * H * dk, dtype=torch.bfloat16, device="cuda")
    q0, k0, v0, g, beta = inputs(B, L, H, H, dk, dk, torch.bfloat16, seed=2)
    views = []
    for i, t in enumerate((q0, k0, v0)):
        w = buf.as_strided((B, L, H, dk), (far, H * dk, dk, 1), i * L * H * dk)
        w.copy_(t)
        views.append(w)
    out, h_last = run(*views, g, beta)
    check(q0, k0, v0, g, beta, out=out, h_last=h_last)


@pytest.mark.parametrize("L", [0, 5, 40])
@pytest.mark.parametrize("B", [0, 2])
def test_empty(B, L):
    args = inputs(B, L, 2, 1, 64, 64, torch.float32)
    h0 = torch.randn(B, 2, 64, 64, device="cuda")
    out, h_last = run(*args, h0=h0)
    assert out.shape == (B, L, 2, 64)
    if L == 0:
        assert torch.equal(h_last, h0)
        out, h_last = run(*args)
        assert torch.equal(h_last, torch.zeros_like(h0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_states_and_outputs_keep_their_bits(dtype):
    """Rounding errors of independent rows add up like a random walk: relative to
    the norm, 21-bit operands leave less than 2^-18 in the state, where one part
    of 11 bits would leave more than 2^-13; outputs no more than their rounding
    (uniform in half a step: eps / 2 / sqrt(3) of a value at the step's lower
    end) and that."""
    args = inputs(2, 500, 8, 8, 128, 128, dtype, seed=11)
    out, h_last = run(*args)
    ref, ref_s, _, _ = recurrence(*args, None, None, 128 ** -0.5)
    assert float((h_last.double() - ref_s).norm() / ref_s.norm()) < 2.0 ** -18
    eps = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps
    assert float((out.double() - ref).norm() / ref.norm()) < 2.0 ** -18 + eps / 2 / 3 ** 0.5


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L", [40, 500])
@pytest.mark.parametrize("d,limit", [(64, 4e-7), (128, 6e-7)])
def test_states_and_outputs_are_as_exact_as_float32(d, limit, L, dtype):
    """As norms: what a row's value passes through (weights, d / 16 additions of each
    product that are cut off, half a step of 2^-24 on average, the operands' 2^-22 and
    2^-21 of independent terms) are some 12 roundings of 2^-24, with twice the keys
    twice the additions, 2e-7 and 3e-7; limits of twice that. One accumulation for
    large and small products, or a factor's exponent in one float32 sum, leave more."""
    args = inputs(2, L, 8, 8, d, d, dtype, seed=11)
    out, h_last = run(*args)
    ref, ref_s, _, _ = recurrence(*args, None, None, d ** -0.5)
    assert float((h_last.double() - ref_s).norm() / ref_s.norm()) < limit
    if dtype == torch.float32:
        assert float((out.double() - ref).norm() / ref.norm()) < limit


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what", ["q", "k", "v", "beta", "h0", "g"])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("L", [12, 200])
def test_nonfinite_inputs_stay_in_their_sequence_and_head(what, bad, L, dtype):
    """Chunked and token by token: the others are bit for bit as without it, and so
    are its own chunks before it."""
    B, H, t = 2, 4, L // 2
    args = dict(zip(("q", "k", "v", "g", "beta"), inputs(B, L, H, H, 64, 64, dtype, seed=3)))
    args["h0"] = torch.randn(B, H, 64, 64, device="cuda")
    want, want_s = run(**args)
    x = args[what].clone()
    x[{"h0": (1, 2, 3, 4), "g": (1, t, 2), "beta": (1, t, 2)}.get(what, (1, t, 2, 5))] = bad
    out, h_last = run(**{**args, what: x})
    keep = torch.ones(B, H, dtype=torch.bool, device="cuda")
    keep[1, 2] = False
    assert torch.equal(out.transpose(1, 2)[keep], want.transpose(1, 2)[keep])
    assert torch.equal(h_last[keep], want_s[keep])
    if what != "h0":
        assert torch.equal(out[1, :t // 64 * 64, 2], want[1, :t // 64 * 64, 2])
    assert not bool(torch.isfinite(out[1, t:, 2]).all())
    no_timeout()


def test_repeated_calls_are_bit_identical():
    for B, L, H in ((4, 500, 40), (1, 2000, 2)):
        args = inputs(B, L, H, H, 128, 128, torch.bfloat16, seed=4)
        a, sa = run(*args)
        b, sb = run(*args)
        assert torch.equal(a, b) and torch.equal(sa, sb)


def test_other_stream_and_captured_graphs():
    """A side stream, and two captured graphs replayed in turn, each with its
    own workspace."""
    calls = []
    for seed, L in ((1, 900), (2, 1300)):
        args = inputs(1, L, 2, 2, 64, 64, torch.float32, seed=seed)
        calls.append((args, *run(*args)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for args, out, h_last in calls:
        got = cuda.gated_delta_rule(*args, stream=side)
        side.synchronize()
        assert torch.equal(got, out)
    graphs = []
    for args, out, h_last in calls:
        o, s = torch.zeros_like(out), torch.zeros_like(h_last)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cuda.gated_delta_rule(*args, out=o, h_last=s)
        graphs.append((graph, o, s))
    for _ in range(2):
        for graph, o, s in graphs:
            o.zero_()
            graph.replay()
        torch.cuda.synchronize()
        for (_, o, s), (_, out, h_last) in zip(graphs, calls):
            assert torch.equal(o, out) and torch.equal(s, h_last)


def test_callers_workspace():
    args = inputs(1, 300, 4, 4, 64, 64, torch.float16, seed=6)
    out, h_last = run(*args)
    size = cuda.gated_delta_rule_workspace_size(1, 300, 4, 4, 64, 64, torch.float16)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    got, s = run(*args, workspace=ws)
    assert torch.equal(got, out) and torch.equal(s, h_last)
    with pytest.raises(cuda.ScanError, match="workspace holds"):
        run(*args, workspace=ws[:-1])
    with pytest.raises(cuda.ScanError, match="16-byte"):
        run(*args, workspace=torch.empty(size + 8, dtype=torch.uint8, device="cuda")[8:])


# ------------------------------------------------------------- single tokens


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,G,dk,dv", [(1, 1, 1, 1, 1), (1, 24, 24, 64, 64), (3, 4, 2, 100, 36),
                                         (7, 12, 3, 80, 72), (2, 2, 1, 256, 256), (5, 3, 3, 33, 17),
                                         (2, 300, 3, 256, 64), (64, 8, 8, 128, 128),
                                         (64, 12, 4, 64, 128), (3, 2, 2, 200, 31)])
@pytest.mark.parametrize("in_place", [True, False])
def test_step(B, H, G, dk, dv, dtype, in_place):
    args = inputs(B, 1, H, G, dk, dv, dtype, seed=B + dk)
    state = torch.randn(B, H, dk, dv, device="cuda")
    before = state.clone()
    new = state if in_place else torch.full_like(state, float("nan"))
    out = cuda.gated_delta_rule_step(*(t[:, 0] for t in args), state,
                                     state_out=None if in_place else new)
    check(*args, h0=before, out=out[:, None], h_last=new)
    if not in_place:
        assert torch.equal(state, before)


@pytest.mark.parametrize("dtype", DTYPES)
def test_step_strides_fixed_decays_and_unaligned_state(dtype):
    B, H, G, dk, dv = 3, 4, 2, 64, 64
    q, k, v, g, beta = inputs(B, 1, H, G, dk, dv, dtype, seed=8, per_token=False)
    g[1] = float("-inf")
    g[2] = 0.0
    beta[0] = 0.0
    buf = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], -1)
    qs, ks, vs = buf.split([G * dk, G * dk, H * dv], -1)
    flat = torch.randn(B * H * dk * dv + 1, device="cuda")
    state = flat[1:].view(B, H, dk, dv)
    before = state.clone()
    out = cuda.gated_delta_rule_step(qs.unflatten(-1, (G, dk)), ks.unflatten(-1, (G, dk)),
                                     vs.unflatten(-1, (H, dv)), g, beta, state, scale=1.3)
    check(q, k, v, g, beta, h0=before, scale=1.3, out=out[:, None], h_last=state)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_then_steps(dtype):
    """A prompt's state decoded on token by token equals one longer prompt."""
    q, k, v, g, beta = inputs(2, 140, 4, 2, 64, 64, dtype, seed=21)
    cut = 130
    first = [t[:, :cut] for t in (q, k, v, g, beta)]
    out, state = run(*first)
    outs = [out]
    for t in range(cut, 140):
        outs.append(cuda.gated_delta_rule_step(*(x[:, t] for x in (q, k, v, g, beta)),
                                               state)[:, None])
    check(q, k, v, g, beta, out=torch.cat(outs, 1), h_last=state)


def test_step_empty_batch_and_graph():
    q, k, v, g, beta = inputs(0, 1, 2, 2, 16, 16, torch.float32)
    out = cuda.gated_delta_rule_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0],
                                     torch.empty(0, 2, 16, 16, device="cuda"))
    assert out.shape == (0, 2, 16)
    args = [t[:, 0] for t in inputs(2, 1, 4, 4, 64, 64, torch.bfloat16, seed=4)]
    state = torch.randn(2, 4, 64, 64, device="cuda")
    want_state = state.clone()
    want = cuda.gated_delta_rule_step(*args, want_state)
    kept = state.clone()
    got = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cuda.gated_delta_rule_step(*args, state, out=got)
    state.copy_(kept)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(state, want_state)


@pytest.mark.parametrize("change,error", [
    (dict(q=lambda t: t.cpu()), TypeError), (dict(q=lambda t: t[0]), ValueError),
    (dict(k=lambda t: t.half()), TypeError), (dict(k=lambda t: t[..., :32]), ValueError),
    (dict(v=lambda t: t.transpose(2, 3)), ValueError), (dict(g=lambda t: t.double()), TypeError),
    (dict(beta=lambda t: t[..., :1]), ValueError), (dict(beta=lambda t: t.half()), TypeError),
    (dict(beta=lambda t: t.cpu()), TypeError),
])
def test_wrapper_refusals(change, error):
    names = ["q", "k", "v", "g", "beta"]
    args = dict(zip(names, inputs(2, 20, 4, 2, 64, 48, torch.float32)))
    for name, f in change.items():
        args[name] = f(args[name])
    with pytest.raises(error):
        cuda.gated_delta_rule(*args.values())
