"""GPU: linear attention, its single-token step and the token log probabilities
in one small language model, as a serving program runs them: a padded batch of
prompts to states and scores, then tokens one at a time from a captured graph;
and MambaLM.score.

The float64 model takes the same float32 weights. Its logits are sums of d = 96
products of magnitude about 1 through two layers; a float32 evaluation keeps
them within 2^-19 relative of the layer outputs (test_linear_attention_cuda.py)
plus 2^-24 per addition, so 1e-4 absolute bounds the log probabilities.
"""
import pytest
import torch

from mamba_onnx import cuda
from mamba_onnx.model import MambaConfig, MambaLM

pytestmark = pytest.mark.gpu

D, H, G, DK, DV, V, LAYERS = 96, 6, 2, 32, 48, 301, 2


class Net:
    """Embedding -> LAYERS x (residual linear attention) -> tied head."""

    def __init__(self, dtype=torch.float32, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        self.emb = r(V, D)
        self.w = [{"q": r(D, G * DK) / D ** 0.5, "k": r(D, G * DK) / D ** 0.5,
                   "v": r(D, H * DV) / D ** 0.5, "g": r(D, H) / D ** 0.5,
                   "o": r(H * DV, D) / (H * DV) ** 0.5} for _ in range(LAYERS)]

    def projections(self, h, w, lead):
        q, k = (h @ w["q"]).view(*lead, G, DK), (h @ w["k"]).view(*lead, G, DK)
        return q, k, (h @ w["v"]).view(*lead, H, DV), -torch.nn.functional.softplus(h @ w["g"])

    def prompt(self, ids, lengths, states):
        h = self.emb[ids]
        for w, s in zip(self.w, states):
            q, k, v, g = self.projections(h, w, ids.shape)
            y = cuda.linear_attention(q, k, v, g, lengths=lengths, h_last=s)
            h = h + y.flatten(-2) @ w["o"]
        return h @ self.emb.t() / D

    def step(self, ids, states):
        h = self.emb[ids]
        for w, s in zip(self.w, states):
            q, k, v, g = self.projections(h, w, ids.shape)
            y = cuda.linear_attention_step(q, k, v, g, s)
            h = h + y.flatten(-2) @ w["o"]
        return h @ self.emb.t() / D

    def exact(self, ids):
        """float64 logits of one sequence [L]."""
        h = self.emb.double()[ids]
        L = ids.shape[0]
        for w in self.w:
            w = {n: t.double() for n, t in w.items()}
            q, k, v, g = self.projections(h, w, (L,))
            S = torch.zeros(H, DK, DV, dtype=torch.float64, device="cuda")
            y = []
            for t in range(L):
                kt, qt = k[t].repeat_interleave(H // G, 0), q[t].repeat_interleave(H // G, 0)
                S = torch.exp(g[t])[:, None, None] * S + kt[:, :, None] * v[t][:, None]
                y.append(DK ** -0.5 * torch.einsum("hk,hkv->hv", qt, S))
            h = h + torch.stack(y).flatten(-2) @ w["o"]
        return h @ self.emb.double().t() / D


def test_prompts_then_tokens_with_scores():
    torch.backends.cuda.matmul.allow_tf32 = False
    net = Net()
    lengths = [70, 1, 33, 128]
    B, L, new = len(lengths), max(lengths), 4
    g = torch.Generator(device="cuda").manual_seed(5)
    text = torch.randint(0, V, (B, L + new), device="cuda", generator=g)
    ids = text[:, :L].clone()
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    states = [torch.empty(B, H, DK, DV, device="cuda") for _ in range(LAYERS)]
    logits = net.prompt(ids, lens, states)
    targets = torch.full((B, L), -1, device="cuda")
    for b, n in enumerate(lengths):
        targets[b, :n - 1] = ids[b, 1:n]
    lp, ent, top_lp, top_id = cuda.token_logprobs(logits, targets, top=5)
    exact = [torch.log_softmax(net.exact(torch.cat([ids[b, :n], text[b, L:]])), -1)
             for b, n in enumerate(lengths)]
    for b, n in enumerate(lengths):
        ref = exact[b]
        want = torch.gather(ref[:n - 1], 1, ids[b, 1:n, None])[:, 0]
        assert bool(((lp[b, :n - 1].double() - want).abs() < 1e-4).all())
        assert bool((lp[b, n - 1:] == 0).all())
        p = ref[:n].exp()
        assert bool(((ent[b, :n].double() + (p * ref[:n]).sum(-1)).abs() < 1e-3).all())
        best = torch.gather(ref[:n], 1, top_id[b, :n])
        assert bool(((top_lp[b, :n].double() - best).abs() < 1e-4).all())
        assert bool((best[:, 0] >= ref[:n].amax(-1) - 2e-4).all())
    # tokens one at a time, from one graph of step and scores
    tok = torch.zeros(B, dtype=torch.int64, device="cuda")
    nxt = torch.zeros_like(tok)
    live = [s.clone() for s in states]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cuda.token_logprobs(net.step(tok, live), nxt, top=3)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = cuda.token_logprobs(net.step(tok, live), nxt, top=3)
    for a, b in zip(live, states):
        a.copy_(b)
    for i in range(new - 1):
        tok.copy_(text[:, L + i])
        nxt.copy_(text[:, L + i + 1])
        graph.replay()
        torch.cuda.synchronize()
        for b, n in enumerate(lengths):
            ref = exact[b][n + i]
            assert abs(float(got[0][b]) - float(ref[nxt[b]])) < 1e-4
            assert abs(float(got[2][b, 0]) - float(ref.max())) < 1e-4
    assert cuda.check_device_error() == 0


def test_mamba_score_matches_log_softmax_of_its_logits():
    cfg = MambaConfig(d_model=64, n_layer=2, vocab_size=203)
    m = MambaLM(cfg).init_random(seed=3).cuda()
    ids = torch.randint(0, 203, (3, 50), device="cuda",
                        generator=torch.Generator(device="cuda").manual_seed(1))
    lp, ent, top_lp, top_id = m.score(ids, top=4)
    ref = torch.log_softmax(m(ids).double(), -1)
    want = torch.gather(ref[:, :-1], 2, ids[:, 1:, None])[..., 0]
    # float32 sums of 203 terms, log probabilities near log 203
    tol = dict(rtol=0, atol=2.0 ** -24 * (203 / 32 + 104) * 4)
    torch.testing.assert_close(lp[:, :-1].double(), want, **tol)
    assert bool((lp[:, -1] == 0).all())
    torch.testing.assert_close(ent.double(), -(ref.exp() * ref).sum(-1), rtol=0,
                               atol=2.0 ** -24 * (203 / 32 + 104) * 40)
    assert torch.equal(top_id[..., 0], m(ids).argmax(-1))
    torch.testing.assert_close(top_lp.double(), torch.gather(ref, 2, top_id), **tol)
