"""A wait that ran out in the attention reaches the caller of ParallelGenerator
as an error, not as a run of tokens from NaN logits. The status is a stand-in:
no wait is made to run out."""

import pytest
import torch

from megakernels import ops
from test_gpu_parallel_generator import NEW, PROMPT, generate

pytestmark = pytest.mark.gpu


def test_status_is_checked(monkeypatch):
    model, gen, out, _ = generate("bf16", 2)
    calls = []

    def status(device=None, clear=True):
        calls.append((torch.device(device), clear))
        return 1

    monkeypatch.setattr(ops, "attention_status", status)
    with pytest.raises(RuntimeError, match="wait"):
        gen.hand_over(1)
    assert calls == [(model.device, True)]
    type(gen).prefill(gen, torch.zeros(PROMPT, dtype=torch.int64, device="cuda"))
    with pytest.raises(RuntimeError, match="wait"):
        gen.generate(out, PROMPT, NEW)
    assert len(calls) == 2  # once for all steps


def test_nothing_is_reported_without_a_reason():
    _, gen, _, _ = generate("int8", 2)
    assert gen.hand_over(0) == PROMPT + NEW and ops.attention_status() == 0
