"""NaN in the caches of `shared_prefix_attention`: what a result reads makes it
NaN, however small its weight, whichever kernel computes it; what it does not
read has no effect."""

import math

import pytest
import torch

from megakernels import ops
from test_gpu_ops import BF16, gen, int8_rows, normal

pytestmark = pytest.mark.gpu


def prefix_of(kind, g, P, H, D):
    """(prefix, own of 40 rows, writes NaN into V of a row): every key has a score far below that of key 0."""
    def unlike(k):  # scores of -8 sqrt(D) for q of ones, and 8 sqrt(D) for key 0
        k[:] = -8
        k[:, 0] = 8
        return k

    if kind == "bf16":
        prefix = (unlike(normal(g, 1, P, H, D))[0], normal(g, P, H, D))
        return prefix, lambda row, head: prefix[1][row, head].fill_(math.nan)
    cache = int8_rows(g, 1, P, H, D)
    unlike(cache.k_codes)
    cache.k_scales.fill_(1.0)
    return cache, lambda row, head: cache.v_scales[0, row, head].fill_(math.nan)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,group,P", [(1, 1, 30), (2, 4, 200), (64, 8, 8192), (40, 7, 40_001)])
@pytest.mark.parametrize("row", [1, 9, 70, -1])
def test_nan_values_of_weight_zero(row, B, group, P, D, kind):
    """Next to key 0, or among other keys. In the prefix: all sequences, the query heads of that KV head. exp(-16 sqrt(D)) is 0 in 32 bits."""
    g, H = gen(90), 2
    prefix, spoil = prefix_of(kind, g, P, H, D)
    q = torch.ones(B, H * group, D, device="cuda", dtype=BF16)
    lens = torch.zeros(B, device="cuda", dtype=torch.int32)
    own = ops.KVCacheInt8.empty(B, 4, H, D) if kind == "int8" else tuple(normal(g, B, 4, H, D) for _ in range(2))
    clean = ops.shared_prefix_attention(q, prefix, own, lens)
    assert clean.isfinite().all()
    spoil(row % P, 1)
    out = ops.shared_prefix_attention(q, prefix, own, lens)
    assert torch.equal(out[:, :group], clean[:, :group]) and out[:, group:].isnan().all()


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("D", [64, 128])
def test_nan_values_of_own_rows(D, kind):
    """In the own rows: that sequence, and only inside its length."""
    g, B, H, group, T = gen(91), 5, 2, 3, 150
    prefix, _ = prefix_of(kind, g, 64, H, D)
    if kind == "int8":
        own = int8_rows(g, B, T, H, D)
        own.k_codes.fill_(-8), own.k_scales.fill_(1.0)
        own.k_codes[:, 96] = 8
        own.v_scales[2, 99, 0] = own.v_scales[3, 100, 0] = math.nan
    else:
        own = normal(g, B, T, H, D), normal(g, B, T, H, D)
        own[0].fill_(-8)
        own[0][:, 96] = 8
        own[1][2, 99, 0, :] = own[1][3, 100, 0, :] = math.nan
    q = torch.ones(B, H * group, D, device="cuda", dtype=BF16)
    out = ops.shared_prefix_attention(q, prefix, own, torch.full((B,), 100, device="cuda", dtype=torch.int32))
    bad = out.isnan().all(-1)
    assert bad[2, :group].all() and bad.sum() == group and out.isnan().sum() == group * D
