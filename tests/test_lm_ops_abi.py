"""CPU: the entry points of include/mamba_lm_ops.h refuse bad arguments before
any CUDA call, with a status and a message (fake device addresses)."""
import ctypes
import re
from pathlib import Path

import pytest

from mamba_onnx import cuda

F = 1 << 30  # fake 16-byte aligned device addresses, 1 GiB apart
I3, I2 = ctypes.c_int64 * 3, ctypes.c_int64 * 2
INVALID, WORKSPACE, ALIASING = 1, 3, 4


def _message():
    return cuda.library().mamba_scan_last_error().decode()


def _prompt(**change):
    v = dict(q=F, k=2 * F, v=3 * F, log_decay=4 * F, h0=5 * F, lengths=6 * F, out=7 * F,
             h_last=8 * F, batch=2, seqlen=8, heads=4, groups=2, dk=16, dv=16,
             q_stride=I3(256, 32, 16), k_stride=I3(256, 32, 16), v_stride=I3(512, 64, 16),
             decay_stride=I3(32, 4, 1), scale=1.0, dtype=0)
    workspace, size = change.pop("workspace", None), change.pop("workspace_bytes", 0)
    args = cuda.LinearAttentionArgs(**{**v, **change})
    return cuda.library().mamba_linear_attention(ctypes.byref(args), workspace, size, None)


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
    (dict(decay_stride=I3(0, 2 ** 41, 1)), INVALID, "strides"),
    (dict(q=None), INVALID, "non-NULL"),
    (dict(log_decay=None), INVALID, "non-NULL"),
    (dict(out=None), INVALID, "non-NULL"),
    (dict(out=F + 64), ALIASING, "out overlaps an input"),
    (dict(out=4 * F), ALIASING, "out overlaps an input"),
    (dict(h_last=5 * F), ALIASING, "h_last overlaps an input"),
    (dict(h_last=7 * F), ALIASING, "must not overlap"),
    (dict(workspace=7 * F, workspace_bytes=64), ALIASING, "must not overlap"),
    (dict(workspace=3 * F, workspace_bytes=64), ALIASING, "workspace overlaps"),
])
def test_linear_attention_refusals(change, status, message):
    assert _prompt(**change) == status
    assert message in _message()


def test_linear_attention_empty_batch_and_null_args():
    assert _prompt(batch=0) == 0
    assert cuda.library().mamba_linear_attention(None, None, 0, None) == INVALID
    assert cuda.library().mamba_linear_attention_step(None, None) == INVALID
    size = cuda.library().mamba_linear_attention_workspace_size
    assert size(1, 4096, 0, 1, 64, 64, 0) == 0      # a bad shape
    assert size(1, 4096, 1, 1, 64, 999, 0) == 0


def _step(**change):
    v = dict(q=F, k=2 * F, v=3 * F, log_decay=4 * F, state=5 * F, state_out=5 * F, out=7 * F,
             batch=2, heads=4, groups=2, dk=16, dv=16, q_stride=I2(32, 16), k_stride=I2(32, 16),
             v_stride=I2(64, 16), decay_stride=I2(4, 1), scale=1.0, dtype=1)
    args = cuda.LinearAttentionStepArgs(**{**v, **change})
    return cuda.library().mamba_linear_attention_step(ctypes.byref(args), None)


@pytest.mark.parametrize("change,status,message", [
    (dict(heads=-4), INVALID, "heads"),
    (dict(groups=0), INVALID, "groups"),
    (dict(dk=1000), INVALID, "dk and dv"),
    (dict(dtype=-1), INVALID, "dtype"),
    (dict(v_stride=I2(-64, 16)), INVALID, "strides"),
    (dict(state=None), INVALID, "non-NULL"),
    (dict(state_out=5 * F + 16), ALIASING, "state_out must be state"),
    (dict(out=5 * F + 64), ALIASING, "out overlaps a state"),
    (dict(state_out=3 * F), ALIASING, "overlaps an input"),
    (dict(out=4 * F), ALIASING, "overlaps an input"),
])
def test_linear_attention_step_refusals(change, status, message):
    assert _step(**change) == status
    assert message in _message()


def _logprobs(logits=F, row_stride=100, dtype=0, target=2 * F, logprob=3 * F, entropy=4 * F,
              top_logprob=5 * F, top_id=6 * F, rows=4, vocab=100, top=3):
    return cuda.library().mamba_token_logprobs(logits, row_stride, dtype, target, logprob, entropy,
                                               top_logprob, top_id, rows, vocab, top, None)


@pytest.mark.parametrize("change,status,message", [
    (dict(dtype=7), INVALID, "dtype"),
    (dict(rows=-1), INVALID, "rows"),
    (dict(rows=2 ** 31), INVALID, "rows"),
    (dict(vocab=0), INVALID, "vocab"),
    (dict(vocab=2 ** 31, row_stride=2 ** 32), INVALID, "vocab"),
    (dict(top=-1), INVALID, "top"),
    (dict(top=65), INVALID, "top"),
    (dict(vocab=2), INVALID, "top"),
    (dict(row_stride=99), INVALID, "row_stride"),
    (dict(row_stride=-1), INVALID, "row_stride"),
    (dict(logits=None), INVALID, "NULL"),
    (dict(target=None), INVALID, "target"),
    (dict(top_id=None), INVALID, "top_id"),
    (dict(logprob=F), ALIASING, "overlaps an input"),
    (dict(entropy=2 * F + 8), ALIASING, "overlaps an input"),
    (dict(top_id=3 * F), ALIASING, "outputs overlap"),
])
def test_token_logprobs_refusals(change, status, message):
    assert _logprobs(**change) == status
    assert message in _message()


def test_token_logprobs_no_rows():
    assert _logprobs(rows=0) == 0


def test_token_logprobs_largest_vocabulary():
    """Indices and their steps have to stay within 32 bits: 2^30 logits pass the
    checks (0 rows: nothing runs), one more is refused."""
    assert _logprobs(vocab=2 ** 30, row_stride=2 ** 30, rows=0) == 0
    for vocab in (2 ** 30 + 1, 2 ** 31 - 8, 2 ** 31 - 1):
        assert _logprobs(vocab=vocab, row_stride=2 ** 32, rows=0) == INVALID
        assert "1..2^30" in _message()


@pytest.mark.parametrize("name", ["q", "k", "v", "log_decay", "h0", "lengths", "out", "h_last"])
def test_linear_attention_refuses_misaligned_addresses(name):
    at = 1 + ["q", "k", "v", "log_decay", "h0", "lengths", "out", "h_last"].index(name)
    assert _prompt(**{name: at * F + 2}) == INVALID
    assert "multiple of its type's size" in _message()


@pytest.mark.parametrize("change", [dict(q=F + 1), dict(v=3 * F + 1), dict(log_decay=4 * F + 2),
                                    dict(state_out=6 * F + 2), dict(out=7 * F + 1)])
def test_linear_attention_step_refuses_misaligned_addresses(change):
    assert _step(**change) == INVALID
    assert "multiple of its type's size" in _message()


@pytest.mark.parametrize("change", [dict(logits=F + 2), dict(target=2 * F + 4),
                                    dict(logprob=3 * F + 2), dict(entropy=4 * F + 1),
                                    dict(top_logprob=5 * F + 2), dict(top_id=6 * F + 4),
                                    dict(logits=F + 1, dtype=2)])
def test_token_logprobs_refuses_misaligned_addresses(change):
    assert _logprobs(**change) == INVALID
    assert "multiple of its type's size" in _message()


@pytest.mark.parametrize("name", ["linear_attention.cu", "linear_attention_mma.cu",
                                  "token_logprobs.cu"])
def test_rules_that_split_work_ask_the_device_for_its_sms(name):
    source = Path(__file__).resolve().parent.parent / "mamba-onnx_b200" / "csrc" / name
    code = re.sub(r"//[^\n]*", "", source.read_text())
    assert "sm_count()" in code and not re.search(r"\b148\b", code)


@pytest.mark.parametrize("name", ["LinearAttentionArgs", "LinearAttentionStepArgs"])
def test_packed_arguments_have_the_structures_layout(name):
    """The wrappers pack the arguments by format; the structures name the fields."""
    fmt = {"LinearAttentionArgs": cuda._LA_ARGS, "LinearAttentionStepArgs": cuda._LA_STEP_ARGS}[name]
    kind = getattr(cuda, name)
    assert fmt.size == ctypes.sizeof(kind)
    count = sum(getattr(t, "_length_", 1) for _, t in kind._fields_)
    args = kind.from_buffer_copy(fmt.pack(*range(1, count + 1)))
    got = []
    for field, t in kind._fields_:
        value = getattr(args, field)
        got += list(value) if hasattr(t, "_length_") else [value]
    assert got == list(range(1, count + 1))
