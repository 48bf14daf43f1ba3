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


@pytest.mark.parametrize("dtype", [pytest.param(torch.float32, id="fp32"), *SIXTEEN])
@pytest.mark.parametrize("layout", ["packed", "odd_rows"])
@pytest.mark.parametrize("L", [16, 150])
def test_elements_far_below_their_rows_largest(L, layout, dtype):
    """Channels of q and of k that are 256 times the others and meet zeros in
    the product, and such columns of v. Beside what any evaluation in float32
    may lose (2^-15 of the magnitudes added up covers 150 rows of 64 keys and
    two parts) the scaled kernel may be off by 2^-39 to 2^-38 of the largest
    that enters each product: two operands of the scores; scores, times 64 rows;
    values, times 64 rows and 3 chunks; the state, of at most 150 rows. With Q
    the largest of a row of q, and M the largest |k||v| of any two rows' largest
    elements, each is at most 2^-38 * 192 * dk Q M, all of them 2^-28 dk Q M.
    The recurrence of short prompts and the kernel for packed bf16 tensors have
    no such part."""
    gen = torch.Generator(device="cuda").manual_seed(L)
    B, H, dk, dv = 2, 2, 64, 64
    q, k = (torch.randn(B, L, H, dk, device="cuda", generator=gen) for _ in range(2))
    v = torch.randn(B, L, H, dv, device="cuda", generator=gen)
    q[..., :4] *= 256
    k[..., :4] = 0
    k[..., 4:8] *= 256
    q[..., 4:8] = 0
    v[..., 5:9] *= 256
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    g = -torch.rand(B, L, H, device="cuda", generator=gen) / 10
    out = cuda.linear_attention(*(lay_out(t, layout) for t in (q, k, v)), g, scale=1.0)

    def whole(q, k, v):
        G = torch.cumsum(g.double(), 1).transpose(1, 2)
        decay = torch.exp((G[..., :, None] - G[..., None, :])
                          .masked_fill(~torch.ones(L, L, device="cuda").tril().bool(), -torch.inf))
        scores = torch.einsum("bihd,bjhd->bhij", q.double(), k.double()) * decay
        return torch.einsum("bhij,bjhd->bihd", scores, v.double())

    ref, magnitude = whole(q, k, v), whole(q.abs(), k.abs(), v.abs())
    bound = REST * magnitude
    if dtype != torch.float32:
        bound = bound + torch.finfo(dtype).eps / 2 * ref.abs() + 2.0 ** -25
    if L > 16 and not (dtype == torch.bfloat16 and layout == "packed"):
        Q = q.double().abs().amax(-1, keepdim=True)
        M = k.double().abs().amax() * v.double().abs().amax()
        bound = bound + 2.0 ** -28 * dk * Q * M
    over = float(((out.double() - ref).abs() / bound).max())
    assert over <= 1, f"off by {over:.3g} bounds"
