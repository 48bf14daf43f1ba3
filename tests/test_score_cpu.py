"""CPU: the torch form of the log probabilities behind MambaLM.score, and the
targets that score lines up with the tokens."""
import pytest
import torch

from mamba_onnx import model as M


def test_token_logprobs_matches_float64():
    g = torch.Generator().manual_seed(0)
    logits = torch.randn(3, 5, 40, generator=g)
    logits[0, 0, 7:] = float("-inf")
    targets = torch.randint(0, 7, (3, 5), generator=g)
    targets[1, 2] = -1
    lp, ent, top_lp, top_id = M.token_logprobs(logits, targets, 6)
    ref = torch.log_softmax(logits.double(), -1)
    want = torch.gather(ref, -1, targets.clamp(min=0)[..., None])[..., 0]
    want[1, 2] = 0
    p = ref.exp()
    # float32 sums of 40 terms: 64 roundings of 2^-24, values up to about 10
    tol = dict(rtol=0, atol=64 * 2.0 ** -24 * 10)
    torch.testing.assert_close(lp.double(), want, **tol)
    torch.testing.assert_close(ent.double(), -torch.special.xlogy(p, p).sum(-1), **tol)
    order = torch.sort(logits, dim=-1, descending=True, stable=True)
    assert torch.equal(top_id, order.indices[..., :6])
    torch.testing.assert_close(top_lp.double(), torch.gather(ref, -1, order.indices[..., :6]), **tol)
    assert len(M.token_logprobs(logits, targets)) == 2


def test_score_pairs_each_position_with_the_next_token(monkeypatch):
    m = M.MambaLM(M.MambaConfig(d_model=8, n_layer=1, vocab_size=11))
    logits = torch.randn(2, 6, 11, generator=torch.Generator().manual_seed(1))
    monkeypatch.setattr(m, "forward", lambda ids, scan=None: logits)
    ids = torch.randint(0, 11, (2, 6), generator=torch.Generator().manual_seed(2))
    lp, ent, top_lp, top_id = m.score(ids, top=3)
    ref = torch.log_softmax(logits, -1)
    for b in range(2):
        for t in range(5):
            assert abs(float(lp[b, t] - ref[b, t, ids[b, t + 1]])) < 1e-6
    assert torch.equal(lp[:, 5], torch.zeros(2))
    assert torch.equal(top_id[..., 0], logits.argmax(-1)) and top_lp.shape == (2, 6, 3)
    lp32, _ = m.score(ids.int())
    assert torch.equal(lp32, lp)


def test_token_logprobs_outside_the_vocabulary_and_refusals():
    logits = torch.randn(4, 9, generator=torch.Generator().manual_seed(3))
    lp, _ = M.token_logprobs(logits, torch.tensor([0, 9, -1, 2 ** 40]))
    assert lp[1].isnan() and lp[3].isnan() and lp[2] == 0 and lp[0] < 0
    for top in (-1, 10):
        with pytest.raises(ValueError, match="top must be"):
            M.token_logprobs(logits, torch.zeros(4, dtype=torch.int64), top)
    with pytest.raises(ValueError, match="top must be"):
        M.token_logprobs(torch.zeros(1, 100), torch.zeros(1, dtype=torch.int64), 65)


def test_a_bad_top_is_a_value_error_wherever_the_logits_are(monkeypatch):
    class OnCuda:  # as far as the check of top looks
        is_cuda, shape = True, (4, 9)

    calls = []
    monkeypatch.setattr(M.cuda, "token_logprobs", lambda *a, top: calls.append(top))
    for top in (-1, 10, 65):
        with pytest.raises(ValueError, match="top must be"):
            M.token_logprobs(OnCuda(), None, top)
    M.token_logprobs(OnCuda(), None, 9)
    assert calls == [9]
