"""CPU: the gated delta rule's and the cross entropy's entry points
(include/mamba_lm_ops.h) refuse bad arguments before any CUDA call, with a
status and a message (fake device addresses)."""
import ctypes
import re
from pathlib import Path

import pytest
import torch

from mamba_onnx import cuda, model

F = 1 << 30  # fake 16-byte aligned device addresses, 1 GiB apart
I3, I2 = ctypes.c_int64 * 3, ctypes.c_int64 * 2
INVALID, WORKSPACE, ALIASING = 1, 3, 4


def _message():
    return cuda.library().mamba_scan_last_error().decode()


def _prompt(**change):
    v = dict(q=F, k=2 * F, v=3 * F, log_decay=4 * F, beta=5 * F, h0=6 * F, lengths=7 * F,
             out=8 * F, h_last=9 * F, batch=2, seqlen=60, heads=4, groups=2, dk=16, dv=16,
             q_stride=I3(1280, 32, 16), k_stride=I3(1280, 32, 16), v_stride=I3(2560, 64, 16),
             decay_stride=I3(160, 4, 1), beta_stride=I3(160, 4, 1), scale=1.0, dtype=0)
    workspace, size = change.pop("workspace", None), change.pop("workspace_bytes", 0)
    args = cuda.GatedDeltaArgs(**{**v, **change})
    return cuda.library().mamba_gated_delta_rule(ctypes.byref(args), workspace, size, None)


@pytest.mark.parametrize("change,status,message", [
    (dict(batch=-1), INVALID, "batch"),
    (dict(seqlen=2 ** 31), INVALID, "2^31"),
    (dict(heads=0), INVALID, "heads"),
    (dict(groups=3), INVALID, "groups must divide heads"),
    (dict(dk=0), INVALID, "dk and dv"),
    (dict(dk=257), INVALID, "dk and dv"),
    (dict(dv=300), INVALID, "dk and dv"),
    (dict(dtype=3), INVALID, "dtype"),
    (dict(batch=2 ** 30, heads=2 ** 10), INVALID, "too large"),
    (dict(q_stride=I3(-1, 32, 16)), INVALID, "strides"),
    (dict(beta_stride=I3(0, 2 ** 41, 1)), INVALID, "strides"),
    (dict(q=None), INVALID, "non-NULL"),
    (dict(beta=None), INVALID, "non-NULL"),
    (dict(out=None), INVALID, "non-NULL"),
    (dict(out=F + 64), ALIASING, "out overlaps an input"),
    (dict(out=5 * F), ALIASING, "out overlaps an input"),
    (dict(h_last=6 * F), ALIASING, "h_last overlaps an input"),
    (dict(h_last=8 * F), ALIASING, "must not overlap"),
    (dict(workspace=8 * F, workspace_bytes=64), ALIASING, "must not overlap"),
    (dict(workspace=3 * F, workspace_bytes=64), ALIASING, "workspace overlaps"),
    (dict(workspace=10 * F, workspace_bytes=64), WORKSPACE, "workspace holds 64"),
    (dict(workspace=10 * F + 8, workspace_bytes=1 << 24), WORKSPACE, "16-byte"),
])
def test_gated_delta_refusals(change, status, message):
    assert _prompt(**change) == status
    assert message in _message()


@pytest.mark.parametrize("name", ["q", "k", "v", "log_decay", "beta", "h0", "lengths", "out",
                                  "h_last"])
def test_gated_delta_refuses_misaligned_addresses(name):
    at = 1 + ["q", "k", "v", "log_decay", "beta", "h0", "lengths", "out", "h_last"].index(name)
    assert _prompt(**{name: at * F + 2}) == INVALID
    assert "multiple of its type's size" in _message()


def test_gated_delta_empty_batch_null_args_and_workspace_sizes():
    lib = cuda.library()
    assert _prompt(batch=0) == 0
    assert lib.mamba_gated_delta_rule(None, None, 0, None) == INVALID
    assert lib.mamba_gated_delta_rule_step(None, None) == INVALID
    size = lib.mamba_gated_delta_rule_workspace_size
    assert size(1, 4096, 0, 1, 64, 64, 0) == 0      # bad shapes
    assert size(1, 4096, 1, 1, 64, 999, 0) == 0
    assert size(1, 48, 1, 1, 64, 64, 0) == 0        # token by token
    assert size(1, 16, 1, 1, 64, 64, 1) == 0
    assert size(1, 4096, 1, 1, 200, 64, 0) == 0
    assert size(1, 49, 1, 1, 64, 64, 0) > 0
    assert size(1, 17, 1, 1, 64, 64, 1) > 0


def _step(**change):
    v = dict(q=F, k=2 * F, v=3 * F, log_decay=4 * F, beta=5 * F, state=6 * F, state_out=6 * F,
             out=8 * F, batch=2, heads=4, groups=2, dk=16, dv=16, q_stride=I2(32, 16),
             k_stride=I2(32, 16), v_stride=I2(64, 16), decay_stride=I2(4, 1),
             beta_stride=I2(4, 1), scale=1.0, dtype=1)
    args = cuda.GatedDeltaStepArgs(**{**v, **change})
    return cuda.library().mamba_gated_delta_rule_step(ctypes.byref(args), None)


@pytest.mark.parametrize("change,status,message", [
    (dict(heads=-4), INVALID, "heads"),
    (dict(groups=0), INVALID, "groups"),
    (dict(dk=1000), INVALID, "dk and dv"),
    (dict(dtype=-1), INVALID, "dtype"),
    (dict(beta_stride=I2(-64, 16)), INVALID, "strides"),
    (dict(state=None), INVALID, "non-NULL"),
    (dict(beta=None), INVALID, "non-NULL"),
    (dict(state_out=6 * F + 16), ALIASING, "state_out must be state"),
    (dict(out=6 * F + 64), ALIASING, "out overlaps a state"),
    (dict(state_out=3 * F), ALIASING, "overlaps an input"),
    (dict(out=5 * F), ALIASING, "overlaps an input"),
    (dict(q=F + 1), INVALID, "multiple of its type's size"),
    (dict(beta=5 * F + 2), INVALID, "multiple of its type's size"),
    (dict(state_out=7 * F + 2), INVALID, "multiple of its type's size"),
])
def test_gated_delta_step_refusals(change, status, message):
    assert _step(**change) == status
    assert message in _message()


def _loss_args(**change):
    v = dict(hidden=F, weight=2 * F, target=3 * F, loss=4 * F, stats=5 * F, rows=100, vocab=1000,
             width=64, hidden_stride=64, weight_stride=64, dtype=2, reserved=0)
    return cuda.LinearCrossEntropyArgs(**{**v, **change})


def _loss(workspace=8 * F, workspace_bytes=1 << 28, **change):
    args = _loss_args(**change)
    return cuda.library().mamba_linear_cross_entropy(ctypes.byref(args), workspace,
                                                     workspace_bytes, None)


@pytest.mark.parametrize("change,status,message", [
    (dict(dtype=3), INVALID, "dtype"),
    (dict(rows=-1), INVALID, "rows"),
    (dict(rows=2 ** 31), INVALID, "rows"),
    (dict(vocab=0), INVALID, "vocab"),
    (dict(vocab=2 ** 30 + 1), INVALID, "vocab"),
    (dict(width=0), INVALID, "width"),
    (dict(width=65537, hidden_stride=65537, weight_stride=65537), INVALID, "width"),
    (dict(hidden_stride=63), INVALID, "strides"),
    (dict(weight_stride=2 ** 41), INVALID, "strides"),
    (dict(rows=2 ** 30, vocab=2 ** 30), INVALID, "too large"),
    (dict(hidden=None), INVALID, "non-NULL"),
    (dict(target=None), INVALID, "non-NULL"),
    (dict(loss=None), INVALID, "non-NULL"),
    (dict(hidden=F + 1), INVALID, "multiple of its type's size"),
    (dict(target=3 * F + 4), INVALID, "multiple of its type's size"),
    (dict(loss=4 * F + 2), INVALID, "multiple of its type's size"),
    (dict(stats=5 * F + 4), INVALID, "stats must be 8-byte aligned"),
    (dict(loss=F + 64), ALIASING, "an output overlaps an input"),
    (dict(stats=3 * F), ALIASING, "an output overlaps an input"),
    (dict(stats=4 * F + 8), ALIASING, "outputs overlap"),
    (dict(workspace=2 * F), ALIASING, "workspace overlaps an input"),
    (dict(workspace=4 * F), ALIASING, "an output overlaps the workspace"),
    (dict(workspace_bytes=64), WORKSPACE, "workspace holds 64"),
    (dict(workspace=None), WORKSPACE, "workspace holds 0"),
    (dict(workspace=8 * F + 8), WORKSPACE, "16-byte"),
])
def test_linear_cross_entropy_refusals(change, status, message):
    assert _loss(**change) == status
    assert message in _message()


def _grad(workspace=8 * F, workspace_bytes=1 << 29, grad=4 * F, grad_stride=1, d_hidden=6 * F,
          d_weight=7 * F, **change):
    args = cuda.LinearCrossEntropyGradArgs(_loss_args(loss=None, **change), grad, grad_stride,
                                           d_hidden, d_weight)
    return cuda.library().mamba_linear_cross_entropy_grad(ctypes.byref(args), workspace,
                                                          workspace_bytes, None)


@pytest.mark.parametrize("change,status,message", [
    (dict(dtype=-1), INVALID, "dtype"),
    (dict(width=0), INVALID, "width"),
    (dict(grad_stride=-1), INVALID, "grad_stride"),
    (dict(stats=None), INVALID, "non-NULL"),
    (dict(grad=None), INVALID, "non-NULL"),
    (dict(stats=5 * F + 4), INVALID, "multiple of its type's size"),
    (dict(grad=4 * F + 2), INVALID, "multiple of its type's size"),
    (dict(d_hidden=6 * F + 1), INVALID, "multiple of its type's size"),
    (dict(d_hidden=F), ALIASING, "an output overlaps an input"),
    (dict(d_weight=5 * F), ALIASING, "an output overlaps an input"),
    (dict(d_weight=4 * F), ALIASING, "an output overlaps an input"),
    (dict(d_weight=6 * F + 64), ALIASING, "outputs overlap"),
    (dict(workspace=4 * F), ALIASING, "workspace overlaps an input"),
    (dict(workspace=7 * F), ALIASING, "an output overlaps the workspace"),
    (dict(workspace_bytes=64), WORKSPACE, "workspace holds 64"),
])
def test_linear_cross_entropy_grad_refusals(change, status, message):
    assert _grad(**change) == status
    assert message in _message()


def test_linear_cross_entropy_no_rows_null_args_and_nothing_wanted():
    lib = cuda.library()
    assert _loss(rows=0) == 0
    assert _grad(rows=0, d_weight=None) == 0
    assert _grad(d_hidden=None, d_weight=None) == 0
    assert lib.mamba_linear_cross_entropy(None, None, 0, None) == INVALID
    assert lib.mamba_linear_cross_entropy_grad(None, None, 0, None) == INVALID
    assert lib.mamba_linear_cross_entropy_workspace_size(ctypes.byref(_loss_args(width=0))) == 0
    assert lib.mamba_linear_cross_entropy_workspace_size(None) == 0
    # float32 operands need their parts, misaligned 16-bit ones a copy
    plain, parts, copies = (lib.mamba_linear_cross_entropy_workspace_size(ctypes.byref(a)) for a in
                            (_loss_args(), _loss_args(dtype=0), _loss_args(hidden=F + 2)))
    assert parts > plain + 2 * 2 * 1000 * 64 and copies > plain


def test_linear_cross_entropy_never_holds_the_logits():
    """4096 rows of 50280 logits would take 824 MB in float32."""
    args = _loss_args(rows=4096, vocab=50280, width=768, hidden_stride=768, weight_stride=768)
    lib = cuda.library()
    assert lib.mamba_linear_cross_entropy_workspace_size(ctypes.byref(args)) < 32 << 20
    grads = cuda.LinearCrossEntropyGradArgs(args, 4 * F, 1, 6 * F, 7 * F)
    assert lib.mamba_linear_cross_entropy_grad_workspace_size(ctypes.byref(grads)) < 256 << 20


@pytest.mark.parametrize("name", ["gated_delta.cu", "gated_delta_mma.cu",
                                  "linear_cross_entropy.cu"])
def test_rules_that_split_work_ask_the_device_for_its_sms(name):
    source = Path(__file__).resolve().parent.parent / "mamba-onnx_b200" / "csrc" / name
    code = re.sub(r"//[^\n]*", "", source.read_text())
    assert "sm_count()" in code and not re.search(r"\b148\b", code)


@pytest.mark.parametrize("name", ["GatedDeltaArgs", "GatedDeltaStepArgs", "LinearCrossEntropyArgs",
                                  "LinearCrossEntropyGradArgs"])
def test_packed_arguments_have_the_structures_layout(name):
    """The wrappers pack the arguments by format; the structures name the fields."""
    fmt = {"GatedDeltaArgs": cuda._GD_ARGS, "GatedDeltaStepArgs": cuda._GD_STEP_ARGS,
           "LinearCrossEntropyArgs": cuda._LCE_ARGS,
           "LinearCrossEntropyGradArgs": cuda._LCE_GRAD_ARGS}[name]

    def values(args):
        got = []
        for field, t in args._fields_:
            value = getattr(args, field)
            if isinstance(value, ctypes.Structure):
                got += values(value)
            else:
                got += list(value) if hasattr(t, "_length_") else [value]
        return got

    kind = getattr(cuda, name)
    assert fmt.size == ctypes.sizeof(kind)
    want = list(range(1, len(values(kind())) + 1))
    assert values(kind.from_buffer_copy(fmt.pack(*want))) == want


# ---------------------------------------------------- the loss on CPU tensors


def _cpu_inputs(dtype=torch.float64):
    gen = torch.Generator().manual_seed(0)
    h = torch.randn(6, 12, generator=gen)
    w = torch.randn(20, 12, generator=gen)
    t = torch.tensor([3, 19, -1, 0, 7, -100])
    return h.to(dtype), w.to(dtype), t


def test_loss_on_cpu_follows_the_formula_and_its_gradients():
    h, w, t = _cpu_inputs(torch.float32)
    h[2] = float("nan")  # a row that does not count leaves no trace
    h, w = h.requires_grad_(), w.requires_grad_()
    loss = model.linear_cross_entropy(h, w, t)
    keep = t >= 0
    z = h.detach()[keep] @ w.detach().t()
    want = torch.logsumexp(z, 1) - z[torch.arange(4), t[keep]]
    assert torch.allclose(loss[keep], want, atol=1e-5) and bool((loss[~keep] == 0).all())
    loss.sum().backward()
    dz = torch.softmax(z, 1)
    dz[torch.arange(4), t[keep]] -= 1
    assert torch.allclose(h.grad[keep], dz @ w.detach(), atol=1e-5)
    assert bool((h.grad[~keep] == 0).all())
    assert torch.allclose(w.grad, dz.t() @ h.detach()[keep], atol=1e-5)


def test_rows_that_do_not_count_and_nonfinite_weights_on_cpu():
    h, w, t = _cpu_inputs(torch.float32)
    w[5, 3], w[7, 0] = float("inf"), float("nan")
    t[:] = -1
    h, w = h.requires_grad_(), w.requires_grad_()
    loss = model.linear_cross_entropy(h, w, t)
    grads = torch.autograd.grad(loss.sum(), (h, w))
    assert all(bool((x == 0).all()) for x in (loss, *grads))


def test_loss_on_cpu_past_the_vocabulary_is_nan():
    h, w, t = _cpu_inputs(torch.float32)
    t[1] = 20
    loss = model.linear_cross_entropy(h, w, t)
    assert bool(torch.isnan(loss[1])) and not bool(torch.isnan(loss[[0, 2, 3, 4, 5]]).any())


def test_model_loss_on_cpu_is_score_negated():
    """The same logits, float32 sums in another order: a few 2^-22 of logits of
    order 1."""
    def no_scan(op, u, delta, A, B, C, D, z, **kw):  # (the scan needs a GPU: any map will do)
        return u * torch.sigmoid(z)

    lm = model.MambaLM(model.MambaConfig(d_model=32, n_layer=2, vocab_size=100)).init_random(1)
    ids = torch.randint(0, 100, (2, 9), generator=torch.Generator().manual_seed(2))
    loss = lm.loss(ids, scan=no_scan)
    assert loss.shape == (2, 9) and bool((loss[:, -1] == 0).all())
    assert torch.allclose(loss, -lm.score(ids, scan=no_scan)[0], atol=1e-5)
