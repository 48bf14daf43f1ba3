"""GPU: the loss from hidden states and its gradients (include/mamba_lm_ops.h),
against float64.

Tolerances. A logit adds up `width` products in float32 on the tensor cores, at
most width 2^-24 of their magnitudes off, and parts of float32 operands drop 3 *
2^-22 of them: d = (2^-20 + width 2^-24) max_v sum |h| |w_v| for a row. m, a
partial sum's exponentials (2^-21 each, with their argument's rounding 2^-23
|z - m|, where terms matter at most 2^-18) and the logarithm add 2^-18 and 2^-22
of |m|: the loss is off by at most 2 d + 2^-18 + 2^-22 |m|. p is off by 2 d +
2^-17 relative. dz is rounded to its type: with b significant bits the values
next to x lie at least 2^(1-b) of it apart and the nearest is at most u = 2^-b
away, 2^-8 (bf16), 2^-11 (fp16), 2^-22 (two parts of fp16); the fp16 forms also by 2^-39 of
the largest |gradient|; so with E =
|g| p (2 d + 2^-17) + u |dz| + 2^-39 max |g|, a gradient is off by E times the
other operand's magnitudes, by (2^-20 + n 2^-24) of the n-term sums of |dz|
times them, and by half a step of its own type (fp16: at least 2^-25).
"""
import pytest
import torch

from mamba_onnx import cuda, model

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = {torch.float32: 2.0 ** -22, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def reference(hidden, weight, targets, grad):
    """float64: (loss, d_hidden, d_weight) and their bounds."""
    dtype = hidden.dtype
    h, w = hidden.double(), weight.double()
    counts = targets >= 0
    h = h.masked_fill(~counts[:, None], 0)
    rows, width = h.shape
    at = targets.clamp(min=0)[:, None]
    z = h @ w.t()
    m = z.amax(1)
    d = (2.0 ** -20 + width * 2.0 ** -24) * (h.abs() @ w.abs().t()).amax(1)
    loss = torch.logsumexp(z, 1) - torch.gather(z, 1, at)[:, 0]
    loss = loss.masked_fill(~counts, 0)
    loss_e = 2 * d + 2.0 ** -18 + 2.0 ** -22 * m.abs()
    g = grad.double().masked_fill(~counts, 0)
    p = torch.softmax(z, 1)
    dz = p.scatter_add(1, at, -torch.ones_like(at, dtype=torch.float64)) * g[:, None]
    E = g.abs()[:, None] * p * (2 * d + 2.0 ** -17)[:, None] + U[dtype] * dz.abs()
    E = E + 2.0 ** -39 * g.abs().max() * counts[:, None]
    out = [loss, dz @ w, dz.t() @ h]
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    bounds = [loss_e]
    for o, other, n, a, e in ((out[1], w.abs(), w.shape[0], dz.abs(), E),
                              (out[2], h.abs(), rows, dz.abs().t(), E.t())):
        b = e @ other + (2.0 ** -20 + n * 2.0 ** -24) * (a @ other)
        bounds.append(b + half * (o.abs() + b) + (2.0 ** -25 if half else 1e-37))
    return out, bounds


def inputs(rows, vocab, width, dtype, seed=0, lean=3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kw = dict(device="cuda", generator=gen)
    targets = torch.randint(0, vocab, (rows,), **kw)
    w = torch.randn(vocab, width, **kw) * width ** -0.5
    h = torch.randn(rows, width, **kw) + lean * torch.rand(rows, 1, **kw) * w[targets] * width ** 0.5
    grad = torch.rand(rows, **kw) + 0.1
    return h.to(dtype), w.to(dtype), targets, grad


def check(h, w, targets, grad, got):
    want, bounds = reference(h, w, targets, grad)
    for name, g, r, b in zip(("loss", "d_hidden", "d_weight"), got, want, bounds):
        if g is None:
            continue
        assert g.shape == r.shape
        err = (g.double() - r).abs()
        assert bool((err <= b).all()), f"{name} off by {float((err / b).max()):.3g} bounds"


def run(h, w, targets, grad, **kw):
    loss, stats = cuda.linear_cross_entropy(h, w, targets)
    return (loss, *cuda.linear_cross_entropy_grad(h, w, targets, stats, grad, **kw))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,width", [(1, 1, 1), (1, 2, 8), (5, 7, 3), (3, 300, 64),
                                              (33, 1000, 100), (128, 256, 64), (129, 257, 65),
                                              (256, 512, 128), (257, 513, 72), (300, 2000, 250),
                                              (700, 1500, 256), (64, 5000, 1000), (1000, 777, 520)])
def test_sizes(rows, vocab, width, dtype):
    h, w, t, g = inputs(rows, vocab, width, dtype, seed=rows + vocab)
    check(h, w, t, g, run(h, w, t, g))
    assert cuda.check_device_error() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 4, 5, 15, 16, 17])
@pytest.mark.parametrize("vocab,width", [(3, 4), (70, 130), (1003, 200), (5000, 129), (20011, 768),
                                         (600, 3300), (300, 13000)])
def test_few_rows(rows, vocab, width, dtype):
    """Rows that do not count among them, and the weights' and d_weight's rows at
    any address."""
    h, w, t, g = inputs(rows, vocab, width, dtype, seed=rows + width)
    if rows > 2:
        t[1] = -1
        h[1, 0] = float("nan")
    check(h, w, t, g, run(h, w, t, g))
    flat = torch.empty(w.numel() + 1, dtype=dtype, device="cuda")
    flat[1:] = w.flatten()
    shifted = flat[1:].view_as(w)
    check(h, shifted, t, g, run(h, shifted, t, g, need_hidden=False))
    check(h, w, t, g, run(h, w, t, g, need_weight=False))
    a, b = run(h, w, t, g), run(h, w, t, g)
    same = [torch.equal(x[t >= 0], y[t >= 0]) for x, y in zip(a[:2], b[:2])]
    assert all(same) and torch.equal(a[2], b[2])


@pytest.mark.parametrize("dtype", DTYPES)
def test_model_sized(dtype):
    """A 130m-sized head: many vocabulary tiles for each CTA pair, d_hidden's
    sums split."""
    h, w, t, g = inputs(300, 50277, 768, dtype, seed=1)
    check(h, w, t, g, run(h, w, t, g))


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows_in_pieces(dtype):
    """More rows than one pass of the loss takes, and dz in several pieces of
    the vocabulary, the last one narrower."""
    h, w, t, g = inputs(33000, 3400, 40, dtype, seed=2)
    t[::7] = -1
    check(h, w, t, g, run(h, w, t, g))


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_gradient_alone(dtype):
    h, w, t, g = inputs(200, 900, 96, dtype, seed=3)
    both = run(h, w, t, g)
    only_h, only_w = run(h, w, t, g, need_weight=False), run(h, w, t, g, need_hidden=False)
    assert only_h[2] is None and only_w[1] is None
    check(h, w, t, g, only_h)
    check(h, w, t, g, only_w)
    check(h, w, t, g, both)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_do_not_count(dtype):
    """Their hidden states (NaN, infinities) and gradients leave no trace."""
    h, w, t, g = inputs(300, 600, 128, dtype, seed=4)
    t[[0, 5, 17, 127, 128, 255, 256, 299]] = torch.tensor([-1, -100, -2 ** 40] + [-1] * 5,
                                                          device="cuda")
    clean = h.masked_fill((t < 0)[:, None], 0)
    dirty, bad = h.clone(), g.clone()
    dirty[t < 0] = float("nan")
    dirty[0, 3] = float("inf")
    bad[t < 0] = float("nan")
    got = run(dirty, w, t, bad)
    check(clean, w, t, g, got)
    assert bool((got[0][t < 0] == 0).all()) and bool((got[1][t < 0] == 0).all())
    t[:] = -1
    got = run(dirty, w, t, bad)
    assert all(bool((x == 0).all()) for x in got)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_of_different_sizes(dtype):
    """Zero, negative and very different upstream gradients; none at all."""
    h, w, t, g = inputs(260, 500, 64, dtype, seed=5)
    g[::3] = 0
    g[1::3] *= -1
    g[2::9] *= 1e-4
    g[4] = 1e4
    check(h, w, t, g, run(h, w, t, g))
    got = run(h, w, t, torch.zeros_like(g))
    assert bool((got[1] == 0).all()) and bool((got[2] == 0).all())
    g = g * 1e-30 if dtype == torch.float32 else g
    check(h, w, t, g, run(h, w, t, g))


@pytest.mark.parametrize("dtype", DTYPES)
def test_confident_and_hopeless_rows(dtype):
    """Logits far apart: targets of probability 1 up to rounding, and of 0."""
    h, w, t, g = inputs(256, 400, 64, dtype, seed=6)
    h = (h.float() * 12).to(dtype)
    check(h, w, t, g, run(h, w, t, g))


def test_float32_matrices_of_uneven_rows():
    """Rows thousands of times smaller than others, rows of zeros, elements far
    below their row's largest; tiny and huge matrices."""
    for scale in (1.0, 1e-20, 1e15):
        h, w, t, g = inputs(200, 700, 96, torch.float32, seed=7)
        w[::5] *= 2.0 ** -13
        w[3::50] = 0
        h[::4] *= 2.0 ** -12
        h[7] = 0
        w[:, ::10] *= 2.0 ** -8
        h, w = h * scale, w / scale
        check(h, w, t, g, run(h, w, t, g))


@pytest.mark.parametrize("dtype", DTYPES)
def test_nonfinite_rows_stay_apart(dtype):
    """A counted row with NaN or infinity has a NaN loss; the other rows' losses
    are those without it."""
    h, w, t, g = inputs(150, 300, 64, dtype, seed=8)
    want, _ = cuda.linear_cross_entropy(h, w, t)
    bad = h.clone()
    bad[3, 5], bad[70, 1] = float("nan"), float("inf")
    loss, _ = cuda.linear_cross_entropy(bad, w, t)
    keep = torch.ones(150, dtype=torch.bool, device="cuda")
    keep[[3, 70]] = False
    assert bool(torch.isnan(loss[~keep]).all())
    check(h[keep], w, t[keep], g[keep], (loss[keep],))
    check(h, w, t, g, (want,))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_nonfinite_upstream_gradients_stay_apart(bad, dtype):
    """They spoil their row of d_hidden (and d_weight, which adds it); the other
    rows' are those without them."""
    h, w, t, g = inputs(150, 300, 64, dtype, seed=8)
    g[3] = bad
    loss, dh, dw = run(h, w, t, g)
    keep = torch.arange(150, device="cuda") != 3
    check(h[keep], w, t[keep], g[keep], (loss[keep], dh[keep]))
    assert not bool(torch.isfinite(dh[3]).any()) and not bool(torch.isfinite(dw).all())
    t[3] = -1  # a row that does not count leaves no trace
    check(h, w, t, g.masked_fill(t < 0, 0), run(h, w, t, g))


@pytest.mark.parametrize("dtype", DTYPES)
def test_target_past_the_vocabulary(dtype):
    h, w, t, g = inputs(10, 20, 16, dtype, seed=9)
    t[4] = 20
    loss, dh, dw = run(h, w, t, g)
    keep = torch.arange(10, device="cuda") != 4
    assert bool(torch.isnan(loss[4])) and not bool(torch.isnan(loss[keep]).any())
    assert bool(torch.isnan(dh[4]).all()) and not bool(torch.isnan(dh[keep]).any())
    assert bool(torch.isnan(dw).any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["offset", "wide", "expanded_grad", "leading", "odd_width"])
def test_strides(layout, dtype):
    rows, vocab, width = 60, 333, 48
    if layout == "odd_width":
        width = 37
    h, w, t, g = inputs(rows, vocab, width, dtype, seed=10)
    if layout == "offset":
        def shift(x):
            buf = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)
            buf[1:] = x.flatten()
            return buf[1:].view(x.shape)
        h, w = shift(h), shift(w)
    elif layout == "wide":
        def widen(x, n):
            buf = torch.full((x.shape[0], x.shape[1] + n), float("nan"), dtype=x.dtype, device="cuda")
            buf[:, :x.shape[1]] = x
            return buf[:, :x.shape[1]]
        h, w = widen(h, 3), widen(w, 8)
    elif layout == "expanded_grad":
        g = torch.full((), 0.25, device="cuda").expand(rows)
    got = run(h, w, t, g)
    if layout == "leading":
        hh = h.view(3, 20, width).transpose(0, 1).contiguous().transpose(0, 1)
        with pytest.raises(ValueError, match="evenly"):
            cuda.linear_cross_entropy(hh, w, t.view(3, 20))
        loss, stats = cuda.linear_cross_entropy(h.view(3, 20, width), w, t.view(3, 20))
        assert loss.shape == (3, 20) and stats.shape == (3, 20, 2)
        assert torch.equal(loss.flatten(), got[0])
    check(h, w, t, g, got)


def test_stats_are_the_normaliser():
    h, w, t, g = inputs(70, 800, 64, torch.float32, seed=11)
    loss, stats = cuda.linear_cross_entropy(h, w, t)
    z = h.double() @ w.double().t()
    assert torch.allclose(stats[:, 0].double(), z.amax(1), rtol=1e-5, atol=1e-5)
    lse = stats[:, 0].double() + torch.log(stats[:, 1].double())
    assert torch.allclose(lse, torch.logsumexp(z, 1), rtol=0, atol=2e-5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_autograd(dtype):
    h, w, t, g = inputs(90, 500, 64, dtype, seed=12)
    want = run(h, w, t, g)
    h, w = h.requires_grad_(), w.requires_grad_()
    loss = model.linear_cross_entropy(h, w, t)
    assert torch.equal(loss, want[0])
    loss.backward(g)
    assert torch.equal(h.grad, want[1]) and torch.equal(w.grad, want[2])
    frozen = w.detach()
    (dh,) = torch.autograd.grad(model.linear_cross_entropy(h, frozen, t).sum(), h)
    check(h.detach(), frozen, t, torch.ones_like(g), (want[0], dh, None))


@pytest.mark.parametrize("rows", [(7, 5), (40, 50)])
def test_autograd_of_any_layout(rows):
    """Hidden states, targets and upstream gradients that are transposed views."""
    h, w, t, g = inputs(rows[0] * rows[1], 300, 64, torch.float32, seed=12)
    h = h.view(*rows, 64).transpose(0, 1).requires_grad_(True)
    w.requires_grad_(True)
    t, g = t.view(rows).t(), g.view(rows).t()
    loss = model.linear_cross_entropy(h, w, t)
    dh, dw = torch.autograd.grad((loss.t() * g.t()).sum(), (h, w))
    check(h.detach().reshape(-1, 64), w.detach(), t.reshape(-1), g.reshape(-1),
          (loss.detach().reshape(-1), dh.reshape(-1, 64), dw))
    dh, dw = torch.autograd.grad(model.linear_cross_entropy(h, w, t), (h, w), g)
    check(h.detach().reshape(-1, 64), w.detach(), t.reshape(-1), g.reshape(-1),
          (loss.detach().reshape(-1), dh.reshape(-1, 64), dw))
    dh, dw = torch.autograd.grad(model.linear_cross_entropy(h, w, t).sum(), (h, w))
    check(h.detach().reshape(-1, 64), w.detach(), t.reshape(-1), torch.ones_like(g).reshape(-1),
          (loss.detach().reshape(-1), dh.reshape(-1, 64), dw))


def test_gradients_against_differences():
    """float32, central differences along random directions: with steps of
    length s their own error is s^2 times the third derivative (at most
    |direction|^3-ish of order 1 here, s = 2^-6: 2^-12) and the loss's rounding
    over s (2^-16 |loss sum|)."""
    h, w, t, g = inputs(20, 60, 16, torch.float32, seed=13)
    _, dh, dw = run(h, w, t, g)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for _ in range(4):
        vh = torch.nn.functional.normalize(torch.randn(h.shape, device="cuda", generator=gen).flatten(),
                                           dim=0).view_as(h)
        vw = torch.nn.functional.normalize(torch.randn(w.shape, device="cuda", generator=gen).flatten(),
                                           dim=0).view_as(w)
        s = 2.0 ** -6
        ends = [float((cuda.linear_cross_entropy(h + e * s * vh, w + e * s * vw, t)[0].double()
                       * g.double()).sum()) for e in (1, -1)]
        slope = (ends[0] - ends[1]) / (2 * s)
        inner = float((dh.double() * vh).sum() + (dw.double() * vw).sum())
        assert abs(slope - inner) < 2.0 ** -10 * (1 + abs(inner))


def test_repeated_calls_streams_and_graphs():
    """Bit-identical results again, on a side stream, and from two captured
    graphs replayed in turn."""
    calls = []
    for seed, rows, dtype in ((1, 300, torch.bfloat16), (2, 140, torch.float32)):
        args = inputs(rows, 3000, 128, dtype, seed=seed)
        calls.append((args, run(*args)))
    for args, want in calls:
        assert all(torch.equal(a, b) for a, b in zip(run(*args), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for args, want in calls:
        loss, stats = cuda.linear_cross_entropy(*args[:3], stream=side)
        dh, dw = cuda.linear_cross_entropy_grad(*args[:3], stats, args[3], stream=side)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((loss, dh, dw), want))
    graphs = []
    for args, want in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run(*args)
        graphs.append((graph, outs, want))
    for _ in range(2):
        for graph, outs, want in graphs:
            for o in outs:
                o.zero_()
            graph.replay()
        torch.cuda.synchronize()
        for _, outs, want in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_callers_workspace_and_empty():
    h, w, t, g = inputs(50, 700, 64, torch.float32, seed=14)
    want, _ = cuda.linear_cross_entropy(h, w, t)
    size = cuda.linear_cross_entropy_workspace_size(h, w, t)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    got, _ = cuda.linear_cross_entropy(h, w, t, workspace=ws)
    assert torch.equal(got, want)
    with pytest.raises(cuda.ScanError, match="workspace holds"):
        cuda.linear_cross_entropy(h, w, t, workspace=ws[:-1])
    loss, stats = cuda.linear_cross_entropy(h[:0], w, t[:0])
    assert loss.shape == (0,) and stats.shape == (0, 2)
    dh, dw = cuda.linear_cross_entropy_grad(h[:0], w, t[:0], stats, g[:0])
    assert dh.shape == (0, 64) and bool((dw == 0).all())


@pytest.mark.parametrize("change,error", [
    (dict(h=lambda x: x.cpu()), TypeError), (dict(h=lambda x: x.double()), TypeError),
    (dict(w=lambda x: x.half()), TypeError), (dict(w=lambda x: x.t()), ValueError),
    (dict(w=lambda x: x[:, :8]), ValueError), (dict(t=lambda x: x.int()), TypeError),
    (dict(t=lambda x: x[:-1]), ValueError),
])
def test_refusals(change, error):
    args = dict(zip(("h", "w", "t"), inputs(20, 64, 16, torch.float32)[:3]))
    for name, f in change.items():
        args[name] = f(args[name])
    with pytest.raises(error):
        cuda.linear_cross_entropy(*args.values())


def test_model_loss_is_score_without_logits():
    """MambaLM.loss equals -score()[0]: both sum the same float32 logits (3 *
    2^-22 of their magnitudes apart, a few units at most here) in another
    order."""
    lm = model.MambaLM(model.MambaConfig(d_model=64, n_layer=2, vocab_size=1000)).init_random(3)
    lm = lm.cuda()
    ids = torch.randint(0, 1000, (2, 50), device="cuda")
    assert torch.allclose(lm.loss(ids), -lm.score(ids)[0], rtol=0, atol=2e-5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 3, 16, 40, 300])
@pytest.mark.parametrize("vocab", [1, 2, 129, 300])
def test_logits_far_below_zero(rows, vocab, dtype):
    """Logits of -2^109 each, exact in every form: the loss is log(vocab), p is
    1 / vocab to 2^-17 (no differences of logits to be off), bounds as above."""
    h = torch.full((rows, 4), -2.0 ** 53, dtype=dtype, device="cuda")
    w = torch.full((vocab, 4), 2.0 ** 54, dtype=dtype, device="cuda")
    t = torch.arange(rows, device="cuda") % vocab
    g = torch.linspace(0.5, 2.0, rows, device="cuda")
    loss, dh, dw = run(h, w, t, g)
    want = torch.log(torch.tensor(float(vocab), dtype=torch.float64))
    assert float((loss.double().cpu() - want).abs().max()) <= 2.0 ** -18 + 2.0 ** -23 * float(want)
    dz = (1.0 / vocab - torch.nn.functional.one_hot(t, vocab).double()) * g.double()[:, None]
    e = 2.0 ** -17 * g.double()[:, None] / vocab + U[dtype] * dz.abs() + 2.0 ** -39 * float(g.max())
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    for got, a, o, n in ((dh, dz, w, vocab), (dw, dz.t(), h, rows)):
        ref, o = a @ o.double(), o.double().abs()
        b = (e if got is dh else e.t()) @ o + (2.0 ** -20 + n * 2.0 ** -24) * (a.abs() @ o)
        assert bool(((got.double() - ref).abs() <= b + half * (ref.abs() + b)).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [2, 16])
def test_logits_of_minus_infinity(rows, dtype):
    """A column of -inf has probability 0: the other columns' losses are those
    without it (its own, as a target, is infinite)."""
    if dtype != torch.float32:
        rows *= 20
    h, w, t, g = inputs(rows, 200, 32, dtype, seed=15)
    h = h.abs() + 0.01
    t = t.clamp(min=1)
    w[0] = float("-inf")
    t[1] = 0
    loss, _ = cuda.linear_cross_entropy(h, w, t)
    keep = t > 0
    check(h[keep], w[1:], t[keep] - 1, g[keep], (loss[keep],))
    assert bool((loss[~keep] == float("inf")).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,width", [(33000, 256), (131072, 256), (100, 8192), (100, 32768)])
def test_long_sums_of_one_sign(rows, width, dtype):
    """Many rows (d_weight's sums) and wide ones (the logits' sums) of one sign do
    not lean to one side. 32 additions of a segment, cut off by half of 2^-23 of
    half the segment on average, leave 2^-20 of a sum; of a logit of 20 that is
    2^-15.7 of p: 2^-15 in the mean, and 2^-14 where a logit's comes to it. The
    reference is rounded to the type as well: a row's elements differ by 1/1000,
    less than bf16's steps, so their roundings do not average out (those of 299 rows,
    1.6e-3 each, leave 9e-5), while a lean shows as the share of elements that fall
    to the next value."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    kw = dict(device="cuda", generator=gen)
    lean, least = (1 / 64, 0.0) if width == 256 else (36 / width, 0.5)
    h = (0.5 + 0.5 * torch.rand(rows, width, **kw)).to(dtype)
    w = ((least + (1 - least) * torch.rand(300, width, **kw)) * lean).to(dtype)
    t = torch.zeros(rows, dtype=torch.int64, device="cuda")
    _, _, dw = run(h, w, t, torch.ones(rows, device="cuda"))
    p = torch.softmax(h.double() @ w.double().t(), 1)
    ref = p.t()[1:] @ h.double()
    off = float(((dw[1:].double() - ref.to(dtype).double()) / ref).mean())
    assert abs(off) < (2.0 ** -15 if width == 256 else 2.0 ** -14)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [3, 10, 40, 300])
def test_rows_that_do_not_count_and_nonfinite_weights(rows, dtype):
    """0 times an infinite weight is not in their d_hidden, nor in d_weight when no
    row counts."""
    h, w, t, g = inputs(rows, 300, 64, dtype, seed=4)
    w[7, 3], w[200, 1], w[299, 60] = float("inf"), float("nan"), float("-inf")
    t[::2] = -1
    loss, dh, _ = run(h, w, t, g)
    assert bool((loss[t < 0] == 0).all()) and bool((dh[t < 0] == 0).all())
    t[:] = -1
    assert all(bool((x == 0).all()) for x in run(h, w, t, g))


@pytest.mark.parametrize("which", [0, 1])
def test_forward_mode_derivatives_are_refused(which):
    """Not lost: a tangent of the hidden states or the weights that the loss would
    come back without."""
    args = list(inputs(20, 60, 16, torch.float32)[:3])
    with torch.autograd.forward_ad.dual_level():
        args[which] = torch.autograd.forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        for context in (torch.enable_grad, torch.no_grad):
            with context(), pytest.raises(RuntimeError):
                model.linear_cross_entropy(*args)


def test_loss_without_gradients_keeps_nothing():
    h, w, t, _ = inputs(40, 60, 16, torch.float32)
    h.requires_grad_(True)
    with torch.no_grad():
        assert model.linear_cross_entropy(h, w, t).grad_fn is None
    with torch.inference_mode():
        loss = model.linear_cross_entropy(h, w, t)
    assert model.linear_cross_entropy(h.detach(), w, t).grad_fn is None
    assert torch.equal(loss, model.linear_cross_entropy(h, w, t))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["transposed", "expanded", "wide", "every_second"])
def test_autograd_with_weights_of_any_layout(layout, dtype):
    h, w, t, g = inputs(40, 60, 16, dtype, seed=16)
    if layout == "transposed":
        w = w.t().contiguous().t()
    elif layout == "expanded":
        w = w[:1].expand(60, 16)
    elif layout == "wide":
        w = torch.cat([w, w], 1)[:, :16]
    else:
        w = w.repeat_interleave(2, 1)[:, ::2]
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    loss = model.linear_cross_entropy(h, w, t)
    grads = torch.autograd.grad(loss, (h, w), g)
    check(h.detach(), w.detach(), t, g, (loss.detach(), *grads))


@pytest.mark.parametrize("types", [(torch.bfloat16, torch.float32), (torch.float32, torch.float16),
                                   (torch.float16, torch.bfloat16)])
def test_autograd_of_two_types(types):
    """In float32, as on the CPU: float32's bounds, and half a step of a gradient's
    own type."""
    h, w, t, g = inputs(40, 60, 16, torch.float32, seed=16)
    h, w = h.to(types[0]).requires_grad_(), w.to(types[1]).requires_grad_()
    loss = model.linear_cross_entropy(h, w, t)
    grads = torch.autograd.grad(loss, (h, w), g)
    want, bounds = reference(h.detach().float(), w.detach().float(), t, g)
    assert bool(((loss.double() - want[0]).abs() <= bounds[0]).all())
    for got, x, r, b in zip(grads, (h, w), want[1:], bounds[1:]):
        assert got.dtype == x.dtype
        half = torch.finfo(x.dtype).eps / 2 if x.dtype != torch.float32 else 0.0
        assert bool(((got.double() - r).abs() <= b + half * (r.abs() + b) + 2.0 ** -25).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,width", [(3, 500, 64), (13, 700, 100), (60, 20000, 264),
                                              (300, 2000, 250), (16500, 3400, 40)])
@pytest.mark.parametrize("need", [(True, True), (True, False), (False, True)])
def test_callers_workspace_for_gradients(rows, vocab, width, need, dtype):
    """Few rows, d_hidden's sums split, columns that are padded, dz in pieces with a
    narrower last one: bit for bit what the default workspace gives, in one of
    0xFF and in one that another call has used; one byte less is refused."""
    h, w, t, g = inputs(rows, vocab, width, dtype, seed=17)
    t[1::5] = -1
    need = dict(zip(("need_hidden", "need_weight"), need))
    _, stats = cuda.linear_cross_entropy(h, w, t)

    def grads(a=(h, w, t, stats, g), **kw):
        return [x for x in cuda.linear_cross_entropy_grad(*a, **need, **kw) if x is not None]

    want = grads()
    size = cuda.linear_cross_entropy_grad_workspace_size(h, w, t, **need)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(grads(workspace=ws), want))
        grads((h * 2, w, t, stats, g * 3), workspace=ws)  # another call's contents
    with pytest.raises(cuda.ScanError, match="workspace holds"):
        grads(workspace=ws[:-1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,width", [(3, 500, 64), (300, 2000, 250), (33000, 700, 40)])
def test_callers_workspace_for_losses(rows, vocab, width, dtype):
    h, w, t, _ = inputs(rows, vocab, width, dtype, seed=18)
    want = cuda.linear_cross_entropy(h, w, t)
    ws = torch.full((cuda.linear_cross_entropy_workspace_size(h, w, t),), 255, dtype=torch.uint8,
                    device="cuda")
    for _ in range(2):
        got = cuda.linear_cross_entropy(h, w, t, workspace=ws)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        cuda.linear_cross_entropy(h * 2, w, t, workspace=ws)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,width", [(300, 20000, 768), (64, 5000, 1000), (12, 20000, 768),
                                              (2, 5000, 768)])
def test_losses_and_gradients_are_as_exact_as_float32(rows, vocab, width, dtype):
    """As norms. A logit's 8 additions of a segment are cut off, by half of 2^-23 of
    half the segment on average, and the segments' sums round: 2^-22 of it, 4e-7 with
    the operands' parts and the logarithm. In float32's gradients p's exponent, of up
    to 20, rounds as well: 20 ln 2 x 2^-25 / sqrt 3, 6e-7 with the rest. One
    accumulation over a row leaves 1.3e-6, of three products 4e-6. Where p of the
    target is 1 almost (both of 2 rows here), log s and p - 1 are what s = 1 + .. in
    float32 leaves of them, 2^-23 and 2^-22 of 1 each row."""
    h, w, t, g = inputs(rows, vocab, width, dtype, seed=1)
    got, (want, _) = run(h, w, t, g), reference(h, w, t, g)
    err = [float((a.double() - b).norm()) for a, b in zip(got, want)]
    assert err[0] < 4e-7 * float(want[0].norm()) + 2.0 ** -23 * rows ** 0.5
    if dtype == torch.float32:
        sizes = [float(g.norm()) * float(x.norm(dim=1).max()) for x in (w, h)]
        for e, b, size in zip(err[1:], want[1:], sizes):
            assert e < 6e-7 * float(b.norm()) + 2.0 ** -22 * size
