"""The language-model operators beside the selective scan, as they are measured.

Three operators: ``linear_attention`` (a prompt through attention without a
softmax whose state decays by a factor for each head), ``linear_attention_step``
(one token of it per sequence) and ``token_logprobs`` (log probabilities of
given tokens, the entropy and the most likely alternatives). ``run`` computes
them in plain torch operations, or, where ``own`` is true, by this package's
entry points.
"""
import math
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
# a drawn prompt has at most this many (token, head) pairs: the largest listed case's
MAX_TOKEN_HEADS = 8 * 2048 * 40
MAX_LOGITS = 4096 * 50280


def _prompt(name, batch, length, heads, groups, dk, dv, dtype, decay="token", ragged=False,
            h0=False):
    return {"name": name, "op": "linear_attention", "batch": batch, "length": length,
            "heads": heads, "groups": groups, "dk": dk, "dv": dv, "dtype": dtype,
            "decay": decay, "ragged": ragged, "h0": h0}


def _step(name, batch, heads, groups, dk, dv, dtype, decay="token"):
    return {"name": name, "op": "linear_attention_step", "batch": batch, "heads": heads,
            "groups": groups, "dk": dk, "dv": dv, "dtype": dtype, "decay": decay}


def _logprobs(name, rows, vocab, dtype, top, masked=False, padded=False):
    return {"name": name, "op": "token_logprobs", "rows": rows, "vocab": vocab, "dtype": dtype,
            "top": top, "masked": masked, "padded": padded}


def listed():
    return [
        # a 1024-token prompt of a 130m-sized model: 24 heads of 64 make d_inner 1536
        _prompt("prompt_1024_f32", 1, 1024, 24, 24, 64, 64, "f32"),
        # a long document, one sequence: few heads, so the sequence itself has to be split
        _prompt("prompt_16384_bf16", 1, 16384, 16, 16, 128, 128, "bf16"),
        # a full prefill batch at d_inner 5120 (40 heads of 128)
        _prompt("prompt_8x2048_bf16", 8, 2048, 40, 40, 128, 128, "bf16"),
        # the same width in fp32, continuing from the states of an earlier part
        _prompt("prompt_4x2048_f32", 4, 2048, 40, 40, 128, 128, "f32", h0=True),
        # a padded batch of odd lengths; all heads share the keys and queries, fixed decays
        _prompt("prompt_ragged_5x777_f16", 5, 777, 20, 1, 64, 96, "f16", decay="head",
                ragged=True),
        # one sequence decoding
        _step("step_1_f32", 1, 24, 24, 64, 64, "f32"),
        # a serving batch decoding at d_inner 5120
        _step("step_64_bf16", 64, 40, 40, 128, 128, "bf16"),
        # an odd batch with shared keys, odd head sizes and fixed decays
        _step("step_7_f16", 7, 12, 3, 80, 72, "f16", decay="head"),
        # the sampled token of one decoding sequence, with five alternatives
        _logprobs("logprobs_1_f32", 1, 50280, "f32", 5),
        # scoring a 1024-token document
        _logprobs("logprobs_1024_f32", 1024, 50280, "f32", 0),
        # scoring a batch of documents with twenty alternatives for each token
        _logprobs("logprobs_4096_bf16", 4096, 50280, "bf16", 20),
        # decoding under a constraint: most of an odd vocabulary masked, rows in a wider buffer
        _logprobs("logprobs_33_masked_f16", 33, 50277, "f16", 8, masked=True, padded=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear_attention", "linear_attention", "linear_attention_step",
                     "token_logprobs"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "token_logprobs":
        vocab = _log_uniform(rng, 1000, 150000)
        rows = _log_uniform(rng, 1, max(1, min(4096, MAX_LOGITS // vocab)))
        return {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype,
                "top": rng.choice([0, 1, 5, 8, 20]), "masked": rng.random() < 0.3,
                "padded": rng.random() < 0.3}
    dims = [32, 48, 64, 72, 80, 96, 100, 112, 128]
    groups = rng.choice([1, 2, 3, 4, 5, 8, 12])
    heads = groups * rng.choice([n for n in (1, 2, 3, 4, 5, 8, 10) if groups * n <= 40])
    case = {"op": op, "heads": heads, "groups": groups, "dk": rng.choice(dims),
            "dv": rng.choice(dims), "dtype": dtype, "decay": rng.choice(["token", "head"])}
    if op == "linear_attention_step":
        case["batch"] = _log_uniform(rng, 1, 64)
        return case
    case["batch"] = rng.randint(1, 8)
    longest = MAX_TOKEN_HEADS // (2 * case["batch"] * heads)  # fp32 moves twice the bytes
    case["length"] = _log_uniform(rng, 2, min(16384, longest))
    case["ragged"] = case["batch"] > 1 and rng.random() < 0.4
    case["h0"] = rng.random() < 0.4
    return case


# ------------------------------------------------------------------ inputs


def _decay(gen, shape, heads, kind):
    """log decays: of each token (-A dt, A in 1..16 by head, dt log-uniform in
    1e-3..1e-1) or fixed for each head (log of 1 - 2^-5 ... 1 - 2^-12)."""
    kw = {"device": "cuda", "generator": gen}
    if kind == "head":
        p = 5 + 7 * torch.rand(heads, **kw)
        return torch.log1p(-torch.exp2(-p))
    A = 1 + 15 * torch.rand(heads, **kw)
    dt = torch.exp(math.log(1e-3) + math.log(100.0) * torch.rand(*shape, heads, **kw))
    return -A * dt


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(dtype)

    if case["op"] == "token_logprobs":
        rows, vocab = case["rows"], case["vocab"]
        width = vocab + 13 if case["padded"] else vocab
        logits = (3 * torch.randn(rows, width, device="cuda", generator=gen)).to(dtype)
        logits = logits[:, :vocab]
        targets = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
        if case["masked"]:
            keep = torch.rand(rows, vocab, device="cuda", generator=gen) < 0.2
            keep.scatter_(1, targets[:, None], True)
            logits.masked_fill_(~keep, float("-inf"))
        return {"op": case["op"], "logits": logits, "targets": targets, "top": case["top"]}

    B, H, G, dk, dv = (case[n] for n in ("batch", "heads", "groups", "dk", "dv"))
    if case["op"] == "linear_attention_step":
        return {"op": case["op"], "q": normal(B, G, dk), "k": normal(B, G, dk) * dk ** -0.5,
                "v": normal(B, H, dv), "log_decay": _decay(gen, (B,), H, case["decay"]),
                "state": torch.randn(B, H, dk, dv, device="cuda", generator=gen),
                "state_out": torch.empty(B, H, dk, dv, device="cuda")}
    L = case["length"]
    state = {"op": case["op"], "q": normal(B, L, G, dk), "k": normal(B, L, G, dk) * dk ** -0.5,
             "v": normal(B, L, H, dv), "log_decay": _decay(gen, (B, L), H, case["decay"]),
             "h0": None, "lengths": None, "h_last": torch.empty(B, H, dk, dv, device="cuda")}
    if case["h0"]:
        state["h0"] = torch.randn(B, H, dk, dv, device="cuda", generator=gen)
    if case["ragged"]:
        lengths = torch.randint(0, L + 1, (B,), device="cuda", generator=gen, dtype=torch.int32)
        lengths[0] = L
        state["lengths"] = lengths
    return state


# ------------------------------------------------------------------ plain forms


def _plain_logprobs(logits, targets, top):
    x = logits.float()
    m = x.amax(dim=-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    s = e.sum(dim=-1, keepdim=True)
    logprob = (torch.gather(d, 1, targets[:, None]) - torch.log(s))[:, 0]
    t = torch.where(e > 0, e * d, torch.zeros_like(e)).sum(dim=-1)
    entropy = torch.log(s[:, 0]) - t / s[:, 0]
    if top == 0:
        return logprob, entropy
    values, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    return logprob, entropy, values[:, :top] - m - torch.log(s), ids[:, :top].contiguous()


def _plain_step(q, k, v, log_decay, state, state_out, scale):
    B, H, dk, dv = state.shape
    rep = H // q.shape[1]
    qh = q.float().repeat_interleave(rep, dim=1)
    kh = k.float().repeat_interleave(rep, dim=1)
    decay = torch.exp(log_decay).expand(B, H)
    new = decay[..., None, None] * state + kh[..., :, None] * v.float()[..., None, :]
    state_out.copy_(new)
    out = scale * (qh[..., None] * new).sum(dim=2)
    return out.to(q.dtype), state_out


def _plain_prompt(q, k, v, log_decay, h0, lengths, h_last, scale, chunk=64):
    B, L, G, dk = q.shape
    H, dv = v.shape[2:]
    n = -(-L // chunk)
    pad = n * chunk - L

    def heads_first(t, width):  # [B, L, heads, width] -> [B, H, n, chunk, width] in fp32
        t = t.float()
        if lengths is not None:
            keep = torch.arange(L, device=t.device)[None, :] < lengths[:, None]
            t = torch.where(keep[..., None, None], t, torch.zeros_like(t))
        t = torch.nn.functional.pad(t, (0, 0, 0, 0, 0, pad))
        t = t.repeat_interleave(H // t.shape[2], dim=2)
        return t.view(B, n, chunk, H, width).permute(0, 3, 1, 2, 4)

    qh, kh, vh = heads_first(q, dk), heads_first(k, dk), heads_first(v, dv)
    g = heads_first(log_decay.expand(B, L, H)[..., None], 1)[..., 0].double()
    G_ = torch.cumsum(g, dim=-1)
    causal = torch.ones(chunk, chunk, dtype=torch.bool, device=q.device).tril()
    decay = torch.exp((G_[..., :, None] - G_[..., None, :]).masked_fill(~causal, float("-inf")))
    out = torch.matmul(torch.matmul(qh, kh.transpose(-1, -2)) * decay.float(), vh)
    del decay
    to_end = torch.exp(G_[..., -1:] - G_).float()
    update = torch.matmul((kh * to_end[..., None]).transpose(-1, -2), vh)
    q_in = qh * torch.exp(G_).float()[..., None]
    carry = torch.exp(G_[..., -1]).float()
    S = torch.zeros_like(h_last) if h0 is None else h0.clone()
    for c in range(n):
        out[:, :, c] += torch.matmul(q_in[:, :, c], S)
        S = carry[:, :, c, None, None] * S + update[:, :, c]
    h_last.copy_(S)
    out = (scale * out).permute(0, 2, 3, 1, 4).reshape(B, n * chunk, H, dv)[:, :L]
    if lengths is not None:
        keep = torch.arange(L, device=q.device)[None, :] < lengths[:, None]
        out = torch.where(keep[..., None, None], out, torch.zeros_like(out))
    return out.to(q.dtype), h_last


def _package():
    if "mamba-onnx_b200" not in sys.path:
        sys.path.insert(0, "mamba-onnx_b200")
    from mamba_onnx import cuda

    return cuda


def run(state):
    op = state["op"]
    if op == "token_logprobs":
        if own:
            return _package().token_logprobs(state["logits"], state["targets"], top=state["top"])
        return _plain_logprobs(state["logits"], state["targets"], state["top"])
    scale = state["q"].shape[-1] ** -0.5
    if op == "linear_attention_step":
        args = [state[n] for n in ("q", "k", "v", "log_decay", "state")]
        if own:
            out = _package().linear_attention_step(*args, scale=scale,
                                                   state_out=state["state_out"])
            return out, state["state_out"]
        return _plain_step(*args, state["state_out"], scale)
    args = [state[n] for n in ("q", "k", "v", "log_decay")]
    if own:
        out = _package().linear_attention(*args, scale=scale, h0=state["h0"],
                                          h_last=state["h_last"], lengths=state["lengths"])
        return out, state["h_last"]
    return _plain_prompt(*args, state["h0"], state["lengths"], state["h_last"], scale)


# ------------------------------------------------------------------ 64 bits


def _exact_logprobs(logits, targets, top):
    x = logits.double()
    lse = torch.logsumexp(x, dim=-1)
    rows = torch.arange(x.shape[0], device=x.device)
    logprob = x[rows, targets] - lse
    p = torch.exp(x - lse[:, None])
    entropy = -torch.xlogy(p, p).sum(dim=-1)
    if top == 0:
        return logprob, entropy
    del p
    index = torch.arange(x.shape[1], device=x.device)
    values, ids = [], []
    for _ in range(top):
        best = x.amax(dim=-1, keepdim=True)
        first = torch.where(x == best, index, x.shape[1]).amin(dim=-1)
        values.append(best[:, 0] - lse)
        ids.append(first)
        x[rows, first] = float("-inf")
    return logprob, entropy, torch.stack(values, 1), torch.stack(ids, 1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "token_logprobs":
        return _exact_logprobs(st["logits"], st["targets"], st["top"])
    B, H, G, dk, dv = (case[n] for n in ("batch", "heads", "groups", "dk", "dv"))
    scale, step = dk ** -0.5, case["op"] == "linear_attention_step"
    q, k, v = (st[n].double() for n in ("q", "k", "v"))
    g = st["log_decay"].double()
    if step:
        q, k, v = q[:, None], k[:, None], v[:, None]
        g = g if g.dim() == 1 else g[:, None]
        S, lengths = st["state"].double(), None
    else:
        S = torch.zeros(B, H, dk, dv, dtype=torch.float64, device="cuda") \
            if st["h0"] is None else st["h0"].double()
        lengths = st["lengths"]
    L = v.shape[1]
    decay = torch.exp(g).expand(B, L, H)
    S = S.view(B, G, H // G, dk, dv).clone()
    out = torch.zeros(B, L, H, dv, dtype=torch.float64, device="cuda")
    for t in range(L):  # S <- decay S + k v^T; out = scale q S
        a = decay[:, t].reshape(B, G, H // G, 1, 1)
        kt, qt = k[:, t].view(B, G, 1, dk, 1), q[:, t].view(B, G, 1, 1, dk)
        vt = v[:, t].view(B, G, H // G, 1, dv)
        if lengths is None:
            S.mul_(a).addcmul_(kt, vt)
            out[:, t] = torch.matmul(qt, S).view(B, H, dv)
        else:
            live = (t < lengths).double().view(B, 1, 1, 1, 1)
            S.mul_(a * live + (1 - live)).addcmul_(kt * live, vt)
            out[:, t] = torch.matmul(qt * live, S).view(B, H, dv)
    out.mul_(scale)
    return out[:, 0] if step else out, S.view(B, H, dk, dv)


# ------------------------------------------------------------------ work


def work(case):
    """Each input read and each output written once; the recurrence's own
    multiplications and additions (4 dk dv for a token and head: the state's
    update and its product with the query), or four for each logit."""
    size = SIZES[case["dtype"]]
    if case["op"] == "token_logprobs":
        rows, n = case["rows"], case["rows"] * case["vocab"]
        return {"bytes": n * size + rows * (8 + 8 + 12 * case["top"]), "flops": 4 * n}
    B, H, G, dk, dv = (case[n] for n in ("batch", "heads", "groups", "dk", "dv"))
    L = case.get("length", 1)
    state_bytes = 4 * B * H * dk * dv
    tokens = B * L
    decay = 4 * (H if case["decay"] == "head" else tokens * H)
    data = size * tokens * (2 * G * dk + 2 * H * dv)
    states = 2 if case["op"] == "linear_attention_step" or case["h0"] else 1
    return {"bytes": data + decay + states * state_bytes, "flops": 4 * tokens * H * dk * dv}
