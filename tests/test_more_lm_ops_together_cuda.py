"""GPU: the gated delta rule, its single-token step and the loss from hidden
states in one small language model: a padded batch of prompts to states and
losses with their gradients, then tokens one at a time from a captured graph;
two such programs on two streams.

The float64 model takes the same float32 weights. Keys have norm 1 and beta lies
in 0..1, so a layer's outputs are within 2^-17 relative of the sizes that go into
them (test_gated_delta_cuda.py), and float32 sums of D = 96 products add 2^-24 a
term: two layers keep logits, which are sums of D products divided by D, within
1e-4, and losses and log probabilities within twice that.
"""
import pytest
import torch

from mamba_onnx import cuda, model

pytestmark = pytest.mark.gpu

D, H, G, DK, DV, V, LAYERS = 96, 6, 2, 32, 48, 301, 2


class Net:
    """Embedding -> LAYERS x (residual gated delta rule) -> tied head."""

    def __init__(self, dtype=torch.float32, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        self.dtype = dtype
        self.emb = r(V, D)
        self.w = [{"q": r(D, G * DK) / D ** 0.5, "k": r(D, G * DK) / D ** 0.5,
                   "v": r(D, H * DV) / D ** 0.5, "g": r(D, H) / D ** 0.5, "b": r(D, H) / D ** 0.5,
                   "o": r(H * DV, D) / (H * DV) ** 0.5} for _ in range(LAYERS)]

    def projections(self, h, w):
        lead, dtype = h.shape[:-1], h.dtype if h.dtype == torch.float64 else self.dtype
        k = (h @ w["k"]).view(*lead, G, DK)
        return ((h @ w["q"]).view(*lead, G, DK).to(dtype),
                torch.nn.functional.normalize(k, dim=-1).to(dtype),
                (h @ w["v"]).view(*lead, H, DV).to(dtype),
                -torch.nn.functional.softplus(h @ w["g"]), torch.sigmoid(h @ w["b"]))

    def prompt(self, ids, lengths, states):
        """Last hidden states; states after each sequence's length."""
        h = self.emb[ids]
        for w, s in zip(self.w, states):
            y = cuda.gated_delta_rule(*self.projections(h, w), lengths=lengths, h_last=s)
            h = h + y.flatten(-2).to(h.dtype) @ w["o"]
        return h

    def step(self, ids, states):
        h = self.emb[ids]
        for w, s in zip(self.w, states):
            y = cuda.gated_delta_rule_step(*self.projections(h, w), s)
            h = h + y.flatten(-2).to(h.dtype) @ w["o"]
        return h

    def states(self, B):
        return [torch.zeros(B, H, DK, DV, device="cuda") for _ in range(LAYERS)]

    def exact(self, ids):
        """float64 last hidden states of one sequence [L]."""
        h = self.emb.double()[ids]
        for w in self.w:
            q, k, v, g, beta = self.projections(h, {n: t.double() for n, t in w.items()})
            S = torch.zeros(H, DK, DV, dtype=torch.float64, device="cuda")
            out = []
            for t in range(ids.shape[0]):
                kt = k[t].repeat_interleave(H // G, 0)
                S = torch.exp(g[t])[:, None, None] * S
                u = beta[t][:, None] * (v[t] - torch.einsum("hk,hkv->hv", kt, S))
                S = S + kt[..., None] * u[:, None, :]
                out.append(torch.einsum("hk,hkv->hv", q[t].repeat_interleave(H // G, 0), S))
            h = h + DK ** -0.5 * torch.stack(out).flatten(-2) @ w["o"].double()
        return h


def ids_of(B, L, seed):
    return torch.randint(0, V, (B, L), device="cuda",
                         generator=torch.Generator(device="cuda").manual_seed(seed))


def test_prompts_losses_and_tokens():
    net, want = Net(), [150, 1, 64, 0, 97]
    B, L, extra = len(want), max(want), 9
    ids = ids_of(B, L + extra, 3)
    lengths = torch.tensor(want, dtype=torch.int32, device="cuda")
    states = net.states(B)
    exact = [net.exact(ids[b, :want[b] + extra] if want[b] else ids[b, L:L + extra])
             for b in range(B)]
    # (tokens that go on after a prompt stand behind its length; the batch's at L)
    for b in range(B):
        ids[b, L:] = ids[b, want[b]:want[b] + extra].clone() if want[b] else ids[b, L:]

    hidden = net.prompt(ids[:, :L], lengths, states).detach()
    targets = torch.full((B, L), -1, device="cuda")
    for b in range(B):
        if want[b] > 1:
            targets[b, :want[b] - 1] = ids[b, 1:want[b]]
    head = net.emb / D
    hidden.requires_grad_(True)
    head.requires_grad_(True)
    losses = model.linear_cross_entropy(hidden, head, targets)
    total = losses.sum() / (targets >= 0).sum()
    d_hidden, d_head = torch.autograd.grad(total, (hidden, head))
    assert bool((losses[targets < 0] == 0).all()) and bool((d_hidden[targets < 0] == 0).all())
    for b in range(B):
        n = want[b] - 1
        if n > 0:
            logp = torch.log_softmax(exact[b][:n] @ net.emb.double().t() / D, -1)
            ref = -torch.gather(logp, 1, targets[b, :n, None])[:, 0]
            assert float((losses[b, :n].detach().double() - ref).abs().max()) < 2e-4

    # the gradients of those hidden states: p is off by twice a logit's error, d,
    # and 2^-17, and sums of n terms by n 2^-24 and 2^-20 of their magnitudes
    h, w = hidden.detach().double()[targets >= 0], head.detach().double()
    z = h @ w.t()
    d = (2.0 ** -20 + D * 2.0 ** -24) * float((h.abs() @ w.abs().t()).max())
    p = torch.softmax(z, -1)
    dz = (p - torch.nn.functional.one_hot(targets[targets >= 0], V)) / h.shape[0]
    e = (2 * d + 2.0 ** -17) * p / h.shape[0] + 2.0 ** -19 * dz.abs()
    bound = e @ w.abs() + V * 2.0 ** -24 * (dz.abs() @ w.abs()) + 1e-12
    assert bool(((d_hidden[targets >= 0].double() - dz @ w).abs() <= bound).all())
    bound = e.t() @ h.abs() + h.shape[0] * 2.0 ** -24 * (dz.abs().t() @ h.abs()) + 1e-12
    assert bool(((d_head.double() - dz.t() @ h).abs() <= bound).all())

    # tokens from a captured graph, the states in place
    token = ids[:, L].clone()
    kept = [s.clone() for s in states]
    net.step(token, states)  # (what a first call loads is loaded)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = net.step(token, states)
    for s, k in zip(states, kept):
        s.copy_(k)
    for t in range(extra):
        token.copy_(ids[:, L + t])
        graph.replay()
        z = torch.log_softmax(got.double() @ net.emb.double().t() / D, -1)
        for b in range(B):
            ref = torch.log_softmax(exact[b][want[b] + t] @ net.emb.double().t() / D, -1)
            assert float((z[b] - ref).abs().max()) < 2e-4
    assert cuda.check_device_error() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_two_programs_on_two_streams(dtype):
    """Prompt, loss, gradients and a token each, captured once and replayed side by
    side: what each gives alone, bit for bit."""
    programs = []
    for seed, B, L in ((1, 3, 130), (2, 2, 300)):
        net = Net(dtype, seed)
        ids, states = ids_of(B, L + 1, seed), net.states(B)
        head = (net.emb / D).to(dtype)

        def run(net=net, ids=ids, states=states, head=head, L=L):
            hidden = net.prompt(ids[:, :L], None, states).to(dtype)
            targets = ids[:, 1:L + 1].contiguous()
            losses, stats = cuda.linear_cross_entropy(hidden, head, targets)
            grad = torch.ones_like(losses)
            grads = cuda.linear_cross_entropy_grad(hidden, head, targets, stats, grad)
            return [losses, *grads, net.step(ids[:, L], states), *(s.clone() for s in states)]

        want = run()
        assert all(bool(torch.isfinite(t).all()) for t in want)
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            got = run()
        programs.append((graph, stream, got, want, run))  # (run holds what the graph reads)
    for _ in range(3):
        for graph, stream, got, *_ in programs:
            with torch.cuda.stream(stream):
                for t in got:
                    t.zero_()
                graph.replay()
        torch.cuda.synchronize()
        for _, _, got, want, _ in programs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert cuda.check_device_error() == 0
