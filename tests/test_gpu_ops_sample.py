"""`sample_tokens` at the sizes where its way of searching changes: rows short
enough to be ranked as a whole, numbers of rows that fill the GPU, and bf16
values inside and outside the table of values. Against the definition in 64
bits, as in test_gpu_ops."""

import math

import pytest
import torch

from megakernels import ops
from test_gpu_ops import BF16, SETTINGS, check_sample, gen

pytestmark = pytest.mark.gpu

DTYPES = pytest.mark.parametrize("dtype", [BF16, torch.float32], ids=["bf16", "f32"])
MORE = SETTINGS + [{"top_k": 20}, {"top_k": 100, "top_p": 0.8}, {"top_k": 512}, {"top_k": 513, "top_p": 0.99},
                   {"top_k": 1000, "min_p": 0.01}, {"top_p": 0.7, "min_p": 0.2}, {"min_p": 0.5}]


@DTYPES
@pytest.mark.parametrize("settings", MORE, ids=str)
@pytest.mark.parametrize("V", [3, 64, 127, 128, 129, 257, 512, 513, 1455, 2048, 4096, 4104])
def test_short_rows(V, dtype, settings):
    g = gen(50)
    x = torch.randn(6, V, generator=g, device="cuda") * 2
    x[1, ::2] = -math.inf
    x[2] = 0.25
    x[3, 1:] = -math.inf
    x[4, :: max(2, V // 3)] = math.nan
    x[5] = torch.linspace(-3, 3, V, device="cuda")
    check_sample(x.to(dtype), torch.rand(6, generator=g, device="cuda"), **settings)


@DTYPES
@pytest.mark.parametrize("settings", [{}, {"top_p": 0.9}, {"top_k": 30}, {"top_k": 600, "top_p": 0.9}, {"min_p": 0.05}], ids=str)
@pytest.mark.parametrize("B,V", [(300, 126), (148, 1455), (149, 1455), (297, 2000), (149, 20480), (149, 20496), (15, 32768),
                                 (34, 50257), (71, 50257), (72, 50257), (75, 50257), (16, 128256), (34, 128256),
                                 (75, 128256), (147, 128256), (148, 128256)])
def test_many_rows(B, V, dtype, settings):
    g = gen(51)
    x = (torch.randn(B, V, generator=g, device="cuda") * 2).to(dtype)
    u = torch.rand(B, generator=g, device="cuda")
    tokens = ops.sample_tokens(x, u, **settings)
    rows = torch.tensor(sorted({0, 1, B // 2, B - 1}), device="cuda")
    assert torch.equal(tokens[rows], check_sample(x[rows], u[rows], **settings))
    assert torch.equal(ops.sample_tokens(x, u, **settings), tokens)


@pytest.mark.parametrize("settings", [{}, {"top_p": 0.9}, {"top_p": 0.3, "min_p": 0.2}, {"top_p": 0.999, "temperature": 0.02},
                                      {"top_p": 0.6, "temperature": 50.0}, {"temperature": 5.0}], ids=str)
@pytest.mark.parametrize("B,V", [(8, 700), (8, 9000), (40, 40000), (74, 16001), (160, 5000)])
def test_values_inside_and_outside_the_table(B, V, settings):
    """bf16 logits with a table entry have 2^-9 <= |l| < 2^7."""
    g = gen(52)
    x = torch.randn(B, V, generator=g, device="cuda")
    x[0] *= 1e-4  # all below the table
    x[1] *= 2.0**-9  # both sides of its end
    x[2] *= 60  # beyond its upper end
    x[3] = x[3].clamp(max=1.9) + 126  # just below the upper end
    x[4] = -x[4].abs() * 30  # negative values only
    x[5, ::2] = 0.0
    x[5, 1::4] = -0.0
    x[6] = torch.where(x[6] > 0, 127.5, -127.5)
    x[7] = torch.where(x[7] > 0, 2.0**-9, 2.0**-10)
    x = x.to(BF16)
    u = torch.rand(B, generator=g, device="cuda")
    tokens = ops.sample_tokens(x, u, **settings)
    rows = torch.tensor(sorted({0, 1, 2, 3, 4, 5, 6, 7, B - 1}), device="cuda")
    assert torch.equal(tokens[rows], check_sample(x[rows], u[rows], **settings))


@DTYPES
def test_rows_of_different_kinds_in_one_call(dtype):
    """Settings per row: whatever a row's neighbours ask for, its token is the one that it gets alone."""
    g = gen(53)
    B, V = 24, 30_011
    x = (torch.randn(B, V, generator=g, device="cuda") * 2).to(dtype)
    u = torch.rand(B, generator=g, device="cuda")
    kw = {"temperature": torch.linspace(0, 2, B, device="cuda"),
          "top_k": torch.tensor([0, 5, 700, V] * 6, device="cuda", dtype=torch.int32),
          "top_p": torch.tensor([1.0, 0.9, 0.4] * 8, device="cuda"),
          "min_p": torch.tensor([0.0, 0.0, 0.0, 0.0, 0.0, 0.1] * 4, device="cuda")}
    tokens = check_sample(x, u, **kw)
    for b in (0, 3, 6, 11, 23):
        alone = {name: value[b].item() for name, value in kw.items()}
        assert ops.sample_tokens(x[b : b + 1], u[b : b + 1], **alone)[0] == tokens[b]
