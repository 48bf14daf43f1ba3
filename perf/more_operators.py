"""More language-model operators beside the selective scan, as they are measured.

Three operators: ``gated_delta_rule`` (a prompt through attention without a
softmax whose state decays by a factor for each head and replaces, by the delta
rule, what it held under a key), ``gated_delta_rule_step`` (one token of it per
sequence) and ``linear_cross_entropy`` (a language model's loss from its last
hidden states and the weights of its head, the logits never stored; forward
alone, or with the gradients of both). ``run`` computes them in plain torch
operations, or, where ``own`` is true, by this package's entry points.
"""
import math
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
# no drawn case is larger than the largest listed one of its operator
MAX_TOKEN_HEADS = 8 * 2048 * 40
MAX_PRODUCT = 4096 * 50280 * 768


def _prompt(name, batch, length, heads, groups, dk, dv, dtype, decay="token", ragged=False,
            h0=False):
    return {"name": name, "op": "gated_delta_rule", "batch": batch, "length": length,
            "heads": heads, "groups": groups, "dk": dk, "dv": dv, "dtype": dtype,
            "decay": decay, "ragged": ragged, "h0": h0}


def _step(name, batch, heads, groups, dk, dv, dtype, decay="token"):
    return {"name": name, "op": "gated_delta_rule_step", "batch": batch, "heads": heads,
            "groups": groups, "dk": dk, "dv": dv, "dtype": dtype, "decay": decay}


def _loss(name, rows, vocab, width, dtype, train, padded=False):
    return {"name": name, "op": "linear_cross_entropy", "rows": rows, "vocab": vocab,
            "width": width, "dtype": dtype, "train": train, "padded": padded}


def listed():
    return [
        # a 1024-token prompt of a 130m-sized model: 24 heads of 64 make d_inner 1536
        _prompt("delta_1024_f32", 1, 1024, 24, 24, 64, 64, "f32"),
        # a long document, one sequence of few heads
        _prompt("delta_16384_bf16", 1, 16384, 16, 16, 128, 128, "bf16"),
        # a full prefill batch at d_inner 5120 (40 heads of 128)
        _prompt("delta_8x2048_bf16", 8, 2048, 40, 40, 128, 128, "bf16"),
        # a padded batch of odd lengths going on from states; 4 heads share queries and keys
        _prompt("delta_ragged_5x777_f16", 5, 777, 20, 5, 64, 96, "f16", ragged=True, h0=True),
        # one sequence decoding
        _step("delta_step_1_f32", 1, 24, 24, 64, 64, "f32"),
        # a serving batch decoding at d_inner 5120
        _step("delta_step_64_bf16", 64, 40, 40, 128, 128, "bf16"),
        # an odd batch with shared keys, odd head sizes and fixed decays
        _step("delta_step_7_f16", 7, 12, 3, 80, 72, "f16", decay="head"),
        # the loss of a short text over an odd vocabulary
        _loss("loss_33_f16", 33, 50277, 768, "f16", False),
        # scoring a 1024-token document with the 130m model's tied head
        _loss("loss_1024_f32", 1024, 50280, 768, "f32", False),
        # a training step of that head: loss and both gradients, part of the rows padding
        _loss("train_1024_f32", 1024, 50280, 768, "f32", True, padded=True),
        # a training batch at the same width in mixed precision
        _loss("train_4096_bf16", 4096, 50280, 768, "bf16", True),
        # an odd batch, vocabulary and width, part of the rows padding
        _loss("train_777_f16", 777, 50277, 1000, "f16", True, padded=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gated_delta_rule", "gated_delta_rule", "gated_delta_rule_step",
                     "linear_cross_entropy", "linear_cross_entropy"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "linear_cross_entropy":
        width = rng.choice([64, 100, 128, 250, 256, 384, 512, 640, 768, 1000, 1024, 1536, 2048])
        vocab = _log_uniform(rng, 1000, 150000)
        # (a float32 product costs the tensor cores three of a 16-bit one)
        most = MAX_PRODUCT // (4 if dtype == "f32" else 1) // (vocab * width)
        return {"op": op, "rows": _log_uniform(rng, 1, max(1, min(8192, most))), "vocab": vocab,
                "width": width, "dtype": dtype, "train": rng.random() < 0.6,
                "padded": rng.random() < 0.4}
    dims = [32, 48, 64, 72, 80, 96, 100, 112, 128]
    groups = rng.choice([1, 2, 3, 4, 5, 8, 12])
    heads = groups * rng.choice([n for n in (1, 2, 3, 4, 5, 8, 10) if groups * n <= 40])
    case = {"op": op, "heads": heads, "groups": groups, "dk": rng.choice(dims),
            "dv": rng.choice(dims), "dtype": dtype, "decay": rng.choice(["token", "head"])}
    if op == "gated_delta_rule_step":
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


def _prepare_loss(case, gen, dtype):
    rows, vocab, width = case["rows"], case["vocab"], case["width"]
    kw = {"device": "cuda", "generator": gen}
    targets = torch.randint(0, vocab, (rows,), **kw)
    weight = torch.randn(vocab, width, **kw) * 0.02
    # hidden states after a norm, leaning towards their target's row by as much as
    # makes it up to e^12 times as likely as an average token
    lean = 12 * torch.rand(rows, 1, **kw) * weight[targets] / (0.02 ** 2 * width)
    hidden = (torch.randn(rows, width, **kw) + lean).to(dtype)
    weight = weight.to(dtype)
    grad = None
    if case["padded"]:
        targets[torch.rand(rows, **kw) < 0.25] = -1
    if case["train"]:
        counted = (targets >= 0).sum().clamp(min=1)
        grad = torch.full((rows,), 1.0, device="cuda") / counted  # the mean's gradient
        hidden.requires_grad_()
        weight.requires_grad_()
    return {"op": case["op"], "hidden": hidden, "weight": weight, "targets": targets,
            "grad": grad}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "linear_cross_entropy":
        return _prepare_loss(case, gen, dtype)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    def unit(*shape):  # queries and keys of norm 1, as the rule wants them
        x = normal(*shape)
        return (x / x.norm(dim=-1, keepdim=True)).to(dtype)

    B, H, G, dk, dv = (case[n] for n in ("batch", "heads", "groups", "dk", "dv"))
    if case["op"] == "gated_delta_rule_step":
        return {"op": case["op"], "q": unit(B, G, dk), "k": unit(B, G, dk),
                "v": normal(B, H, dv).to(dtype), "log_decay": _decay(gen, (B,), H, case["decay"]),
                "beta": torch.sigmoid(normal(B, H)), "state": normal(B, H, dk, dv),
                "state_out": torch.empty(B, H, dk, dv, device="cuda")}
    L = case["length"]
    state = {"op": case["op"], "q": unit(B, L, G, dk), "k": unit(B, L, G, dk),
             "v": normal(B, L, H, dv).to(dtype),
             "log_decay": _decay(gen, (B, L), H, case["decay"]),
             "beta": torch.sigmoid(normal(B, L, H)),
             "h0": None, "lengths": None, "h_last": torch.empty(B, H, dk, dv, device="cuda")}
    if case["h0"]:
        state["h0"] = normal(B, H, dk, dv)
    if case["ragged"]:
        lengths = torch.randint(0, L + 1, (B,), device="cuda", generator=gen, dtype=torch.int32)
        lengths[0] = L
        state["lengths"] = lengths
    return state


# ------------------------------------------------------------------ plain forms


def _plain_step(q, k, v, log_decay, beta, state, state_out, scale):
    B, H, dk, dv = state.shape
    rep = H // q.shape[1]
    qh = q.float().repeat_interleave(rep, dim=1)
    kh = k.float().repeat_interleave(rep, dim=1)
    decayed = torch.exp(log_decay).expand(B, H)[..., None, None] * state
    held = (kh[..., None] * decayed).sum(dim=2)  # what the state has under this key
    u = beta[..., None] * (v.float() - held)
    new = decayed + kh[..., :, None] * u[..., None, :]
    state_out.copy_(new)
    out = scale * (qh[..., None] * new).sum(dim=2)
    return out.to(q.dtype), state_out


def _plain_prompt(q, k, v, log_decay, beta, h0, lengths, h_last, scale, chunk=64):
    """In chunks: with G the running log decay and A_ts = beta_t e^(G_t - G_s) k_t k_s
    below the diagonal, the chunk's updates are U = (I + A)^-1 beta (v - e^G k S)."""
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
    b = heads_first(beta.expand(B, L, H)[..., None], 1)
    g = heads_first(log_decay.expand(B, L, H)[..., None], 1)[..., 0].double()
    G_ = torch.cumsum(g, dim=-1)
    causal = torch.ones(chunk, chunk, dtype=torch.bool, device=q.device).tril()
    decay = torch.exp((G_[..., :, None] - G_[..., None, :]).masked_fill(~causal,
                                                                        float("-inf"))).float()
    A = b * torch.matmul(kh, kh.transpose(-1, -2)) * decay
    P = torch.matmul(qh, kh.transpose(-1, -2)) * decay
    del decay
    T = torch.eye(chunk, device=q.device).expand_as(A).clone()
    for i in range(1, chunk):  # the inverse of I + strictly lower A, row by row
        T[..., i, :i] = -torch.matmul(A[..., i, None, :i], T[..., :i, :i])[..., 0, :]
    from_start = torch.exp(G_).float()[..., None]
    U0 = torch.matmul(T, b * vh)
    W = torch.matmul(T, b * from_start * kh)
    q_in = qh * from_start
    k_out = kh * torch.exp(G_[..., -1:] - G_).float()[..., None]
    carry = torch.exp(G_[..., -1]).float()
    S = torch.zeros_like(h_last) if h0 is None else h0.clone()
    out = torch.empty(B, H, n, chunk, dv, device=q.device)
    for c in range(n):
        U = U0[:, :, c] - torch.matmul(W[:, :, c], S)
        out[:, :, c] = torch.matmul(q_in[:, :, c], S) + torch.matmul(P[:, :, c], U)
        S = carry[:, :, c, None, None] * S + torch.matmul(k_out[:, :, c].transpose(-1, -2), U)
    h_last.copy_(S)
    out = (scale * out).permute(0, 2, 3, 1, 4).reshape(B, n * chunk, H, dv)[:, :L]
    if lengths is not None:
        keep = torch.arange(L, device=q.device)[None, :] < lengths[:, None]
        out = torch.where(keep[..., None, None], out, torch.zeros_like(out))
    return out.to(q.dtype), h_last


def _plain_loss(hidden, weight, targets, grad):
    h, w = hidden.detach().float(), weight.detach().float()
    counts = targets >= 0
    at = targets.clamp(min=0)[:, None]
    z = torch.matmul(h, w.t())
    z -= z.amax(dim=-1, keepdim=True)
    target = torch.gather(z, 1, at)[:, 0]
    e = torch.exp(z)
    s = e.sum(dim=-1)
    loss = torch.where(counts, torch.log(s) - target, torch.zeros_like(s))
    if grad is None:
        return loss
    g = torch.where(counts, grad, torch.zeros_like(grad))
    dz = e * (g / s)[:, None]
    dz.scatter_add_(1, at, -g[:, None])
    d_hidden, d_weight = torch.matmul(dz, w), torch.matmul(dz.t(), h)
    return loss, d_hidden.to(hidden.dtype), d_weight.to(weight.dtype)


def _package(name):
    if "mamba-onnx_b200" not in sys.path:
        sys.path.insert(0, "mamba-onnx_b200")
    from mamba_onnx import cuda, model

    return cuda if name == "cuda" else model


def run(state):
    op = state["op"]
    if op == "linear_cross_entropy":
        hidden, weight, targets, grad = (state[n] for n in ("hidden", "weight", "targets", "grad"))
        if not own:
            return _plain_loss(hidden, weight, targets, grad)
        loss = _package("model").linear_cross_entropy(hidden, weight, targets)
        if grad is None:
            return loss
        return (loss.detach(), *torch.autograd.grad(loss, (hidden, weight), grad))
    scale = state["q"].shape[-1] ** -0.5
    if op == "gated_delta_rule_step":
        args = [state[n] for n in ("q", "k", "v", "log_decay", "beta", "state")]
        if own:
            out = _package("cuda").gated_delta_rule_step(*args, scale=scale,
                                                         state_out=state["state_out"])
            return out, state["state_out"]
        return _plain_step(*args, state["state_out"], scale)
    args = [state[n] for n in ("q", "k", "v", "log_decay", "beta")]
    if own:
        out = _package("cuda").gated_delta_rule(*args, scale=scale, h0=state["h0"],
                                                h_last=state["h_last"], lengths=state["lengths"])
        return out, state["h_last"]
    return _plain_prompt(*args, state["h0"], state["lengths"], state["h_last"], scale)


# ------------------------------------------------------------------ 64 bits


def _exact_loss(st):
    h, w, t = st["hidden"].detach().double(), st["weight"].detach().double(), st["targets"]
    rows = h.shape[0]
    loss = torch.zeros(rows, dtype=torch.float64, device="cuda")
    train = st["grad"] is not None
    d_hidden, d_weight = torch.zeros_like(h), torch.zeros_like(w) if train else None
    for r0 in range(0, rows, 1024):
        part = slice(r0, min(rows, r0 + 1024))
        idx = torch.nonzero(t[part] >= 0)[:, 0]
        z = h[part][idx] @ w.t()
        goal = t[part][idx]
        at = torch.arange(len(idx), device="cuda")
        lse = torch.logsumexp(z, dim=1)
        loss[r0 + idx] = lse - z[at, goal]
        if not train:
            continue
        z = torch.softmax(z, dim=1)
        z[at, goal] -= 1
        z *= st["grad"][part][idx].double()[:, None]
        d_hidden[r0 + idx] = z @ w
        d_weight += z.t() @ h[part][idx]
    return (loss, d_hidden, d_weight) if train else loss


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "linear_cross_entropy":
        return _exact_loss(st)
    B, H, G, dk, dv = (case[n] for n in ("batch", "heads", "groups", "dk", "dv"))
    R, scale, step = H // G, dk ** -0.5, case["op"] == "gated_delta_rule_step"
    q, k, v = (st[n].double() for n in ("q", "k", "v"))
    g, beta = st["log_decay"].double(), st["beta"].double()
    if step:
        q, k, v, beta = q[:, None], k[:, None], v[:, None], beta[:, None]
        g = g if g.dim() == 1 else g[:, None]
        S, lengths = st["state"].double(), None
    else:
        S = torch.zeros(B, H, dk, dv, dtype=torch.float64, device="cuda") \
            if st["h0"] is None else st["h0"].double()
        lengths = st["lengths"]
    L = v.shape[1]
    decay = torch.exp(g).expand(B, L, H).reshape(B, L, G, R, 1, 1)
    beta = beta.reshape(B, L, G, R, 1, 1)
    if lengths is not None:  # rows past a length: no decay, no update
        live = torch.arange(L, device="cuda")[None, :] < lengths[:, None]
        live = live.double().view(B, L, 1, 1, 1, 1)
        decay, beta = decay * live + (1 - live), beta * live
    S = S.view(B, G, R, dk, dv).clone()
    out = torch.zeros(B, L, H, dv, dtype=torch.float64, device="cuda")
    for t in range(L):  # S <- a S; S += beta k (v - k S); out = scale q S
        S.mul_(decay[:, t])
        kt, vt = k[:, t].view(B, G, 1, 1, dk), v[:, t].view(B, G, R, 1, dv)
        u = (vt - torch.matmul(kt, S)) * beta[:, t]
        S.addcmul_(kt.transpose(-1, -2), u)
        out[:, t] = torch.matmul(q[:, t].view(B, G, 1, 1, dk), S).view(B, H, dv)
    out.mul_(scale)
    if lengths is not None:
        out.mul_(live.view(B, L, 1, 1))
    return out[:, 0] if step else out, S.view(B, H, dk, dv)


# ------------------------------------------------------------------ work


def work(case):
    """Each input read and each output written once. The recurrence: its own
    multiplications and additions (6 dk dv for a token and head: the key's and
    the query's product with the state and its update). The loss: one product
    of the hidden states with the head, and one more for each gradient."""
    size = SIZES[case["dtype"]]
    if case["op"] == "linear_cross_entropy":
        rows, vocab, width = (case[n] for n in ("rows", "vocab", "width"))
        data = size * width * (rows + vocab)
        if case["train"]:
            return {"bytes": 2 * data + 16 * rows, "flops": 6 * rows * vocab * width}
        return {"bytes": data + 12 * rows, "flops": 2 * rows * vocab * width}
    B, H, G, dk, dv = (case[n] for n in ("batch", "heads", "groups", "dk", "dv"))
    L = case.get("length", 1)
    state_bytes = 4 * B * H * dk * dv
    tokens = B * L
    decay = 4 * (H if case["decay"] == "head" else tokens * H) + 4 * tokens * H
    data = size * tokens * (2 * G * dk + 2 * H * dv)
    states = 2 if case["op"] == "gated_delta_rule_step" or case["h0"] else 1
    return {"bytes": data + decay + states * state_bytes, "flops": 6 * tokens * H * dk * dv}
