"""`sample_tokens` on rows with more equal logits than 16 bits count, held in
shared memory or read again in each pass: sums of equal weights are exact, so
the number of ties that a cut keeps is that of 64-bit arithmetic."""

import pytest
import torch

from megakernels import ops
from test_gpu_ops import BF16, check_sample, gen

pytestmark = pytest.mark.gpu


def check_first(rows, B, u, **settings):
    """Row i is rows[i % len(rows)]; the first 2 * len(rows) are looked at."""
    n = 2 * len(rows)
    index = torch.arange(B, device="cuda") % len(rows)
    x = rows[index]
    uniforms = torch.zeros(B, device="cuda")
    uniforms[:n] = u[:n]
    tokens = ops.sample_tokens(x, uniforms, **settings)
    want = check_sample(rows[index[:n]], u[:n], **settings)  # few rows: held in shared memory
    assert torch.equal(tokens[:n], want)


@pytest.mark.parametrize("settings", [{"top_p": 0.17}, {"top_p": 0.3}, {"top_p": 0.43}, {"top_p": 0.9}, {"top_p": 0.999},
                                      {"top_p": 0.9, "top_k": 100_000}, {"top_k": 90_001}, {"top_p": 0.6, "min_p": 1e-4},
                                      {"min_p": 1e-4}, {}], ids=str)
@pytest.mark.parametrize("dtype", [BF16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("B,V", [(8, 128256), (148, 128256), (300, 128256), (149, ops.MAX_VOCAB)])
def test_equal_logits_below_the_maximum(B, V, dtype, settings):
    """One logit 8 to 10 above all others, as clamped rows have it."""
    g = gen(80)
    rows = torch.zeros(4, V, device="cuda")
    rows[0, 4321] = 8.1
    rows[1, V - 1] = 9.2
    rows[2, 0] = 9.6
    rows[3] = -7.3
    rows[3, V // 2] = 2.7
    check_first(rows.to(dtype), B, torch.rand(8, generator=g, device="cuda"), **settings)


@pytest.mark.parametrize("settings", [{"top_p": 0.99, "temperature": 1.2}, {"top_p": 0.9, "temperature": 1.2},
                                      {"top_p": 0.99, "temperature": 1.2, "top_k": 120_000}, {"temperature": 1.2, "top_k": 110_000}], ids=str)
@pytest.mark.parametrize("dtype", [BF16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("B,V", [(8, 128256), (150, 128256), (150, ops.MAX_VOCAB)])
def test_two_levels_close_to_each_other(B, V, dtype, settings):
    """The cut lies among the lower of two groups of equal logits; the last uniforms draw near it."""
    rows = torch.zeros(2, V, device="cuda")
    rows[0, :100_000] = 0.0005
    rows[1, 1::4] = 0.0005
    rows[1, 2::4] = 0.0005
    rows[1, 3::4] = 0.0005
    rows[:, 77] = 1.0
    u = torch.tensor([1 - 2.0**-24, 0.5, 0.9999, 0.99999], device="cuda")
    check_first(rows.to(dtype), B, u, **settings)
