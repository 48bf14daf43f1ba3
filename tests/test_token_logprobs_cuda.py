"""GPU: log probabilities of given tokens, entropies and alternatives
(include/mamba_lm_ops.h) against float64.

Tolerances. The logits are exact inputs; the sums are float32. A log
probability is (x - m) - log s: the difference rounds by 2^-24 |x - m|, s is a
sum of V positive terms, each within 4 * 2^-24 of e^(x - m) plus 2^-24 |x - m|
of its argument's rounding, added with at most 2^-24 per addition over fewer
than V / 32 + 64 additions along a path (threads, then lanes, then warps), and
the last subtraction rounds by 2^-24 of the result. Terms with |x - m| above 20
weigh e^-20, so 32 bounds the argument part. The entropy log s - t / s adds the
same for t, whose terms weigh |x - m| <= 32.
"""
import pytest
import torch

from mamba_onnx import cuda

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def reference(logits, targets, top):
    x = logits.double()
    V = x.shape[-1]
    # relative to the largest: log V is below float64's step at the types' lowest values
    m = x.amax(-1, keepdim=True)
    x = x - m
    lse = torch.logsumexp(x, -1)
    t = targets.clamp(0, V - 1)
    lp = torch.gather(x, -1, t[..., None])[..., 0] - lse
    lp = torch.where(targets < 0, torch.zeros_like(lp), lp)
    lp = torch.where(targets >= V, torch.full_like(lp, float("nan")), lp)
    p = torch.exp(x - lse[..., None])
    ent = -torch.xlogy(p, p).sum(-1)
    vals, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    return lp, ent, vals[..., :top] - lse[..., None], ids[..., :top]


def close(got, want, V, weight=1.0):
    tol = 2.0 ** -24 * (V / 32 + 64 + 4 + 32 + 4) * weight
    bound = tol + 2 * 2.0 ** -24 * want.abs()
    bad_nan = torch.isnan(got) != torch.isnan(want)
    same_inf = got.double() == want
    ok = same_inf | torch.isnan(want) | ((got.double() - want).abs() <= bound)
    assert not bool(bad_nan.any()) and bool(ok.all()), \
        f"off by {float((got.double() - want).abs().nan_to_num(0).max()):.3g}"


def check(logits, targets, top):
    got = cuda.token_logprobs(logits, targets, top=top)
    want = reference(logits, targets, top)
    V = logits.shape[-1]
    assert got[0].shape == targets.shape and got[1].shape == targets.shape
    close(got[0], want[0], V)
    close(got[1], want[1], V, weight=33.0)
    if top:
        assert torch.equal(got[3], want[3])
        close(got[2], want[2], V)
    else:
        assert len(got) == 2


def make(rows, V, dtype, seed=0, spread=3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, V, device="cuda", generator=gen) * spread).to(dtype)
    t = torch.randint(0, V, (rows,), device="cuda", generator=gen)
    return x, t


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,top", [
    (1, 1, 1), (1, 2, 2), (3, 5, 0), (2, 64, 64), (5, 100, 7), (1, 1000, 20), (4, 4099, 33),
    (1, 50280, 5), (300, 50280, 20), (33, 50277, 64), (2, 131072, 1), (1, 256001, 10),
    (700, 1003, 8), (1500, 40, 5)])
def test_rows_and_vocabularies(rows, V, top, dtype):
    x, t = make(rows, V, dtype, seed=V + rows)
    check(x, t, top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("V", [777, 50280])
def test_ties_go_to_the_lowest_id(V, rows, dtype):
    gen = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randint(-2, 3, (rows, V), device="cuda", generator=gen).to(dtype)
    t = torch.randint(0, V, (rows,), device="cuda", generator=gen)
    check(x, t, 50)
    check(torch.zeros_like(x), t, 64)               # one value
    check(-torch.zeros_like(x), t, 64)
    zeros = torch.zeros_like(x)
    zeros[:, ::2] = -0.0                            # -0 and 0 are equal
    check(zeros, t, 9)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 170])
def test_orders_that_crowd_the_largest(rows, dtype):
    """Rising, falling and clustered logits: the alternatives all in one place."""
    V = 9000
    ramp = torch.arange(V, device="cuda", dtype=torch.float32) / 256
    t = torch.zeros(rows, dtype=torch.int64, device="cuda")
    for base in (ramp, ramp.flip(0), (torch.arange(V, device="cuda") % 256 == 7).float() * 20 + ramp,
                 (torch.arange(V, device="cuda") % 1024 < 8).float() * 20 + ramp,
                 (torch.arange(V, device="cuda") // 64 == 3).float() * 20 - ramp):
        check(base.expand(rows, V).to(dtype).contiguous(), t, 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [2, 160])
def test_masked_vocabularies(rows, dtype):
    """-inf, or the type's lowest value, nearly everywhere; one or no token left."""
    V = 5003
    x, t = make(rows, V, dtype, seed=6)
    for fill in (float("-inf"), torch.finfo(dtype).min):
        y = x.clone()
        y[:, 3:] = fill
        check(y, t, 10)
        y = torch.full_like(x, fill)
        y[:, V - 1] = 1.0
        check(y, t, 5)
    empty = torch.full_like(x, float("-inf"))
    lp, ent, top_lp, top_id = cuda.token_logprobs(empty, t, top=4)
    assert bool(torch.isnan(lp).all() and torch.isnan(ent).all() and torch.isnan(top_lp).all())
    assert top_id[0].tolist() == [0, 1, 2, 3]
    low = torch.full_like(x, torch.finfo(dtype).min)
    check(low, t, 4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 150])
def test_nan_and_infinity_spoil_only_their_row(rows, dtype):
    x, t = make(rows + 2, 3001, dtype, seed=7)
    clean = cuda.token_logprobs(x[2:].contiguous(), t[2:].contiguous(), top=3)
    x[0, 1234] = float("nan")
    x[1, 77] = float("inf")
    lp, ent, top_lp, top_id = cuda.token_logprobs(x, t, top=3)
    assert bool(torch.isnan(lp[:2]).all() and torch.isnan(ent[:2]).all()
                and torch.isnan(top_lp[:2]).all())
    assert int(top_id[0, 0]) == 1234 and int(top_id[1, 0]) == 77
    for a, b in zip((lp, ent, top_lp, top_id), clean):
        assert torch.equal(a[2:], b)


def test_targets_outside_the_vocabulary():
    x, t = make(6, 500, torch.float32)
    t[0], t[1], t[2], t[3] = -1, -100, 500, 2 ** 40
    check(x, t, 2)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    x, _ = make(24, 1210, dtype, seed=8)
    t = torch.randint(0, 1001, (24,), device="cuda")
    check(x[:, :1001], t, 6)                              # rows in a wider buffer
    check(x[:, 3:1004], t, 6)                             # and off 16 bytes
    check(x[:1, :1001].expand(24, 1001), t, 6)            # one row for all
    check(x.view(4, 6, 1210)[..., :1001], t.view(4, 6), 6)
    check(x[0], t[0], 6)
    check(x.view(4, 6, 1210)[:, 2], t[:4], 6)
    with pytest.raises(ValueError, match="evenly spaced"):
        cuda.token_logprobs(x.view(4, 6, 1210)[:, :5], t[:20].view(4, 5).contiguous())


def test_rows_past_32_bits():
    V, stride = 4000, 2 ** 31 - 8
    buf = torch.empty(2 * stride + V, dtype=torch.float16, device="cuda")
    x = buf.as_strided((3, V), (stride, 1))
    y, t = make(3, V, torch.float16, seed=3)
    x.copy_(y)
    for a, b in zip(cuda.token_logprobs(x, t, top=5), cuda.token_logprobs(y, t, top=5)):
        assert torch.equal(a, b)


def test_large_spreads_and_offsets():
    for spread, offset in ((1e4, 0.0), (1e-3, 0.0), (1.0, 3e4), (1.0, -1e30)):
        x, t = make(3, 3000, torch.float32, spread=spread)
        x += offset
        check(x, t, 5)


def test_stream_graph_and_repeats():
    x, t = make(300, 20011, torch.bfloat16)
    want = cuda.token_logprobs(x, t, top=20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = cuda.token_logprobs(x, t, top=20, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = cuda.token_logprobs(x, t, top=20)
    x.copy_(make(300, 20011, torch.bfloat16, seed=5)[0])
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, cuda.token_logprobs(x, t, top=20)))


def test_empty_and_refusals():
    x, t = make(4, 50, torch.float32)
    lp, ent, tl, ti = cuda.token_logprobs(x[:0], t[:0], top=2)
    assert lp.shape == (0,) and ti.shape == (0, 2)
    with pytest.raises(cuda.ScanError, match="top must be"):
        cuda.token_logprobs(x, t, top=51)
    with pytest.raises(cuda.ScanError, match="top must be"):
        cuda.token_logprobs(make(1, 100, torch.float32)[0], t[:1], top=65)
    with pytest.raises(cuda.ScanError, match="vocab"):
        cuda.token_logprobs(x[:, :0], t)
    with pytest.raises(TypeError, match="targets must be torch.int64"):
        cuda.token_logprobs(x, t.int())
    with pytest.raises(ValueError, match="targets must have shape"):
        cuda.token_logprobs(x, t[:3])
    with pytest.raises(ValueError, match="last dimension"):
        cuda.token_logprobs(x.t(), t[:1].expand(50).contiguous())
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        cuda.token_logprobs(x.double(), t)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 450])
@pytest.mark.parametrize("V,top", [(1, 1), (5, 5), (64, 64), (5003, 7), (50280, 3)])
def test_nan_alternatives_go_by_rising_id(V, top, rows, dtype):
    """NaN stands above +inf, the lowest id first: at id 0, everywhere, beside
    +inf; every id returned is one of the vocabulary."""
    x, t = make(rows, V, dtype, seed=V)
    nan, inf = float("nan"), float("inf")
    first, everywhere, beside = x.clone(), torch.full_like(x, nan), x.clone()
    first[:, 0] = nan
    beside[:, 0], beside[:, V // 2], beside[:, -1] = inf, nan, nan
    for y in (first, everywhere, beside):
        lp, ent, top_lp, top_id = cuda.token_logprobs(y, t, top=top)
        assert bool(torch.isnan(lp).all() and torch.isnan(ent).all() and torch.isnan(top_lp).all())
        want = torch.sort(y.float(), dim=-1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(top_id, want)
