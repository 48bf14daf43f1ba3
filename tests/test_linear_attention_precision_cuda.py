"""GPU: how many bits of the scores and of the state reach a 16-bit output of
linear attention (include/mamba_lm_ops.h).

Inputs where an output is a single score or a single element of the state times
a factor, so that nothing averages a rounding away and nothing cancels. The
result before its own rounding may then be off, relative to itself, by
  2^-18  what is left of a score or state held as two bf16 parts (two fp16
         parts: 2^-22),
  2^-16  a sum of at most 256 positive products in float32, each addition
         rounding by 2^-24,
  2^-18  at most 64 more roundings of 2^-24 to 2^-22: decays, scale, chunks,
less than 2^-15 in all, and its rounding by half a step at its size. One part
alone (2^-12 and 2^-9 of a term) would leave these bounds.
"""
import pytest
import torch

from mamba_onnx import cuda

pytestmark = pytest.mark.gpu

REST = 2.0 ** -15
SIXTEEN = [pytest.param(torch.float16, id="fp16"), pytest.param(torch.bfloat16, id="bf16")]


def within(out, ref):
    ref = ref.double()
    eps = torch.finfo(out.dtype).eps
    most = ref.abs() * (1 + REST)
    step = torch.exp2(torch.floor(torch.log2(most))) * eps
    err = (out.double() - ref).abs() / (step / 2 + REST * ref.abs())
    assert float(err.max()) <= 1, f"off by {float(err.max()):.3g} bounds"


def uniform(gen, *shape):
    return torch.rand(*shape, device="cuda", generator=gen) + 0.5


def lay_out(t, layout):
    if layout == "packed":
        return t
    buf = torch.zeros(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device=t.device)
    buf[..., :t.shape[-1]] = t
    return buf[..., :t.shape[-1]]


@pytest.mark.parametrize("dtype", SIXTEEN)
@pytest.mark.parametrize("layout", ["packed", "odd_rows"])
@pytest.mark.parametrize("L,dk,dv", [(50, 64, 64), (50, 128, 128), (150, 64, 128), (300, 48, 96),
                                     (300, 128, 64), (300, 256, 64)])
def test_scores(L, dk, dv, layout, dtype):
    """Every row clears the state: an output is its own row's score times v."""
    gen = torch.Generator(device="cuda").manual_seed(L + dk)
    B, H, G = 2, 4, 2
    q, k = uniform(gen, B, L, G, dk).to(dtype), uniform(gen, B, L, G, dk).to(dtype)
    v = uniform(gen, B, L, H, dv).to(dtype)
    g = torch.full((B, L, H), float("-inf"), device="cuda")
    out = cuda.linear_attention(*(lay_out(t, layout) for t in (q, k, v)), g)
    score = (q.double() * k.double()).sum(-1).repeat_interleave(H // G, 2)
    within(out, dk ** -0.5 * score[..., None] * v.double())


@pytest.mark.parametrize("dtype", SIXTEEN)
@pytest.mark.parametrize("layout", ["packed", "odd_rows"])
@pytest.mark.parametrize("L,dk,dv", [(50, 64, 64), (50, 128, 128), (150, 64, 128), (300, 48, 96),
                                     (300, 128, 64), (300, 256, 64)])
def test_state(L, dk, dv, layout, dtype):
    """Keys of zero and queries of one element: an output is one element of h0,
    decayed, times that."""
    gen = torch.Generator(device="cuda").manual_seed(L * dk)
    B, H, G = 2, 4, 2
    at = torch.randint(0, dk, (B, L, G), device="cuda", generator=gen)
    value = uniform(gen, B, L, G).to(dtype)
    q = torch.zeros(B, L, G, dk, dtype=dtype, device="cuda")
    q.scatter_(3, at[..., None], value[..., None])
    k = torch.zeros_like(q)
    v = uniform(gen, B, L, H, dv).to(dtype)
    g = -torch.rand(B, L, H, device="cuda", generator=gen) / 100
    h0 = uniform(gen, B, H, dk, dv)
    out = cuda.linear_attention(*(lay_out(t, layout) for t in (q, k, v)), g, h0=h0)
    rep = H // G
    decay = torch.exp(torch.cumsum(g.double(), 1))
    rows = torch.arange(B, device="cuda")[:, None, None]
    heads = torch.arange(H, device="cuda")[None, None, :]
    element = h0.double()[rows, heads, at.repeat_interleave(rep, 2)]
    factor = dk ** -0.5 * decay * value.double().repeat_interleave(rep, 2)
    within(out, factor[..., None] * element)
