"""`sample_tokens` at temperatures so small that all but the largest logits weigh
less than the fixed point resolves. Against the definition in 64 bits: where the
next logit's weight is below 2^-43 of the largest, the token is a largest logit
whatever the uniform is."""

import math

import pytest
import torch

from megakernels import ops
from test_gpu_ops import BF16, check_sample, gen

pytestmark = pytest.mark.gpu

TOPS = [5.0, 20.0, 100.0, 130.0, 0.0078125, -0.5, -20.0]


def rows_under(tops, V, dtype, g):
    """A row per maximum: two largest logits, a quarter of the row one bf16 step below, the rest further down."""
    x = torch.empty(len(tops), V, device="cuda")
    for row, top in zip(x, tops):
        step = 2.0 ** (math.frexp(abs(top))[1] - 8)
        row.copy_(top - step * torch.randint(2, 60, (V,), generator=g, device="cuda"))
        row[torch.randperm(V, generator=g, device="cuda")[: V // 4]] = top - step
        row[torch.randint(0, V, (2,), generator=g, device="cuda")] = top
    return x.to(dtype)


@pytest.mark.parametrize("settings", [{}, {"top_k": 700}, {"top_k": 700, "top_p": 0.9}, {"top_p": 0.9}, {"top_k": 20}, {"min_p": 0.1}], ids=str)
@pytest.mark.parametrize("temperature", [1e-2, 1e-3, 5e-4, 1e-4, 3e-5, 1e-5, 1e-6, 1e-30, 1e-40])
@pytest.mark.parametrize("dtype", [BF16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("B,V", [(7, 900), (7, 20011), (7, 128256), (160, 100_003)])
def test_cold_rows(B, V, dtype, temperature, settings):
    g = gen(70)
    x = rows_under(TOPS, V, dtype, g)
    u = torch.rand(len(TOPS), generator=g, device="cuda")
    u[1], u[2] = 0.0, 1 - 2.0**-24
    if B > len(TOPS):  # more rows than resident clusters; the first are looked at
        many = torch.zeros(B, V, device="cuda", dtype=dtype)
        many[: len(TOPS)] = x
        tokens = ops.sample_tokens(many, torch.cat([u, torch.zeros(B - len(TOPS), device="cuda")]), temperature=temperature, **settings)
        assert torch.equal(tokens[: len(TOPS)], check_sample(x, u, temperature=temperature, **settings))
    else:
        tokens = check_sample(x, u, temperature=temperature, **settings)
    if temperature <= 1e-6:  # the smallest step is 2^-14: weights of exp(-61) of the largest
        t = tokens[: len(TOPS), None]
        assert (x.gather(1, t)[:, 0] == x.max(1).values).all()


def test_temperatures_of_rows_down_to_the_smallest():
    g = gen(71)
    V, T = 30_011, [0.02, 1e-3, 1e-4, 3e-5, 1e-6, 1e-38, 1e-45]
    x = rows_under([20.0] * len(T), V, BF16, g)
    u = torch.rand(len(T), generator=g, device="cuda")
    check_sample(x, u, temperature=torch.tensor(T, device="cuda"))
    check_sample(x, u, temperature=torch.tensor(T, device="cuda"), top_k=torch.full((len(T),), 600, device="cuda", dtype=torch.int32))
