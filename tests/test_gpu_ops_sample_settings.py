"""`sample_tokens` with settings per row, which the host does not see, outside
their ranges: every row still gives a token of its own that the formula allows."""

import math

import pytest
import torch

from megakernels import ops
from test_gpu_ops import BF16, check_sample, gen

pytestmark = pytest.mark.gpu


def column(x, B, dtype=torch.float32):
    return torch.full((B,), x, device="cuda", dtype=dtype)


@pytest.mark.parametrize("settings", [{}, {"min_p": 0.1}, {"min_p": 1.0}, {"top_k": 30}, {"top_k": 700}, {"top_p": 0.5},
                                      {"top_k": 5000, "top_p": 0.7}], ids=str)
@pytest.mark.parametrize("dtype", [BF16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("B,V", [(3, 100), (3, 20_011), (160, 100_003)])
def test_infinite_temperature(B, V, dtype, settings):
    """Every logit above -inf weighs 1, so min_p keeps all of them; without it, the token is that of the largest finite
    temperature."""
    g = gen(120)
    x = torch.randn(B, V, generator=g, device="cuda")
    x[0, : V // 2] = -math.inf
    x[1, 1::2] = -math.inf
    x = x.to(dtype)
    u = torch.rand(B, generator=g, device="cuda")
    got = ops.sample_tokens(x, u, temperature=column(math.inf, B), **settings)
    others = {name: value for name, value in settings.items() if name != "min_p"}
    assert torch.equal(got, ops.sample_tokens(x, u, temperature=column(torch.finfo(torch.float32).max, B), **others))
    assert (x.gather(1, got[:, None]) > -math.inf).all()
    if not others:
        for b in range(3):
            left = x[b].isfinite().nonzero().reshape(-1)
            assert int(got[b]) == int(left[int(u[b].double().item() * len(left))])


@pytest.mark.parametrize("dtype", [BF16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("B,V", [(3, 100), (3, 20_011), (160, 100_003)])
def test_settings_that_mean_none(B, V, dtype):
    """temperature <= 0 or NaN: the largest logit. top_k <= 0, top_p >= 1 or NaN, min_p <= 0 or NaN: no filter. top_p <= 0:
    one token. min_p > 1: as 1."""
    g = gen(121)
    x = (torch.randn(B, V, generator=g, device="cuda") * 2).to(dtype)
    u = torch.rand(B, generator=g, device="cuda")
    for t in (0.0, -1.0, math.nan, -math.inf):
        assert torch.equal(ops.sample_tokens(x, u, temperature=column(t, B)), x.float().argmax(-1))
    plain = ops.sample_tokens(x, u)
    for kw in [{"top_k": column(k, B, torch.int32)} for k in (0, -5, V, V + 7)] + [{"top_p": column(p, B)} for p in (1.0, 2.0, math.inf, math.nan)] + \
            [{"min_p": column(p, B)} for p in (0.0, -3.0, math.nan)]:
        assert torch.equal(ops.sample_tokens(x, u, **kw), plain), kw
    for kw in [{"top_p": column(p, B)} for p in (0.0, -1.0, -math.inf)]:
        assert torch.equal(ops.sample_tokens(x, u, **kw), x.float().argmax(-1)), kw
    assert torch.equal(ops.sample_tokens(x, u, min_p=column(5.0, B)), ops.sample_tokens(x, u, min_p=1.0))
    rows = torch.arange(3, device="cuda")
    assert torch.equal(plain[rows], check_sample(x[rows], u[rows]))
