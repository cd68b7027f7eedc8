"""The scale of `shared_prefix_attention`: 0 gives the mean of V, whatever the
scores are, and negative and tiny scales their formula.

Tolerances. With scale 0 every probability is exactly 1: the sum of n values
rounds by at most 2^-23 of sum |v| per addition, the result by 2^-8 of itself.
The others are bounded as in test_gpu_ops."""

import math

import pytest
import torch

from megakernels import ops
from test_gpu_ops import BF16, EPS, attention64, gen, int8_rows, normal, wide

pytestmark = pytest.mark.gpu


def inputs(g, B, H, group, P, T, D, kind):
    if kind == "int8":
        prefix, own = int8_rows(g, 1, P, H, D), int8_rows(g, B, T, H, D)
    else:
        prefix, own = (normal(g, P, H, D), normal(g, P, H, D)), (normal(g, B, T, H, D), normal(g, B, T, H, D))
    return normal(g, B, H * group, D), prefix, own


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,group,P", [(2, 3, 200), (64, 8, 4096), (40, 7, 5001)])  # few query rows; many
@pytest.mark.parametrize("size", [1.0, 1e17])
def test_scale_zero_is_the_mean(size, B, group, P, D, kind):
    g, H, T = gen(110), 2, 70
    q, prefix, own = inputs(g, B, H, group, P, T, D, kind)
    q *= size  # scores of 1e34 and more
    for store in (prefix, own):
        if kind == "int8":
            store.k_scales.mul_(size)
        else:
            store[0].mul_(size)
    lens = torch.full((B,), 33, device="cuda", dtype=torch.int32)
    out, lse = ops.shared_prefix_attention(q, prefix, own, lens, scale=0.0, return_lse=True)
    n = P + 33
    vp, vo = wide(prefix)[1][0], wide(own)[1][:, :33]
    mean = ((vp.sum(0) + vo.sum(1)) / n).repeat_interleave(group, 1)
    most = ((vp.abs().sum(0) + vo.abs().sum(1)) / n).repeat_interleave(group, 1)
    weight = 2.0**-8 if kind == "int8" else 0.0  # with 8-bit rows V's scale is the probability's factor
    assert ((out.double() - mean).abs() <= EPS * mean.abs() + (n * 2.0**-23 + weight) * most).all()
    assert ((lse.double() - math.log(n)).abs() <= 2.0**-20 * math.log(n)).all()


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_scale_zero_with_infinities(kind):
    """0 * infinity is NaN: q of a sequence, K of a head."""
    g, B, H, group, P, D = gen(111), 64, 2, 8, 8192, 64
    q, prefix, own = inputs(g, B, H, group, P, 4, D, kind)
    lens = torch.zeros(B, device="cuda", dtype=torch.int32)
    q[5, 3, 7], q[6, 2, 0], q[7, 1, 63] = math.inf, -math.inf, math.nan
    bad = ops.shared_prefix_attention(q, prefix, own, lens, scale=0.0).isnan()
    rows = bad.all(-1)
    assert rows[5, 3] and rows[6, 2] and rows[7, 1] and rows.sum() == 3 and bad.sum() == 3 * D
    if kind == "bf16":
        prefix[0][100, 1, 0] = -math.inf
        rows = ops.shared_prefix_attention(q, prefix, own, lens, scale=0.0).isnan().all(-1)
        assert rows[:, group:].all() and rows[:, :group].sum() == 3


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("scale", [-0.2, -1e-30, 1e-30, 1e-38, 1e-45])
@pytest.mark.parametrize("B,group,P", [(2, 3, 200), (64, 8, 8192)])
def test_negative_and_tiny_scales(B, group, P, scale, kind):
    g, H, D = gen(112), 2, 64
    q, prefix, own = inputs(g, B, H, group, P, 8, D, kind)
    lens = torch.full((B,), 5, device="cuda", dtype=torch.int32)
    rows = torch.tensor([0, B - 1], device="cuda")
    out = ops.shared_prefix_attention(q, prefix, own, lens, scale=scale)[rows]
    part = ops.KVCacheInt8(*(t[rows] for t in own._tensors())) if kind == "int8" else tuple(t[rows] for t in own)
    exact, _, size = attention64(q[rows], prefix, part, lens[rows], scale)
    assert ((out.double() - exact).abs() <= EPS * exact.abs() + (EPS + P * 2.0**-23) * size).all()
