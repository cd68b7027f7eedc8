"""Settings of the wrong type: ValueError, like any other bad setting."""

import pytest
import torch

from megakernels import ops
from megakernels.build import build

build()  # no-op when the libraries are newer than their sources

BF16 = torch.bfloat16
BAD = [1.5, "x", [1], object()]


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_attention_settings_without_a_gpu(bad):
    q, lens = torch.zeros(1, 8, 64, dtype=BF16), torch.zeros(1, dtype=torch.int32)
    pair, own = (torch.zeros(4, 2, 64, dtype=BF16),) * 2, (torch.zeros(1, 4, 2, 64, dtype=BF16),) * 2
    with pytest.raises(ValueError):
        ops.shared_prefix_attention(q, pair, own, lens, max_own_len=bad)
    if not isinstance(bad, float):
        with pytest.raises(ValueError):
            ops.shared_prefix_attention(q, pair, own, lens, scale=bad)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", BAD, ids=str)
def test_settings(bad):
    q, lens = torch.zeros(1, 8, 64, dtype=BF16, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    pair, own = (q[0, :2].expand(2, 64)[None],) * 2, (torch.zeros(1, 4, 2, 64, dtype=BF16, device="cuda"),) * 2
    cache, k = ops.KVCacheInt8.empty(1, 4, 2, 64), torch.zeros(1, 1, 2, 64, dtype=BF16, device="cuda")
    calls = [("max_own_len", lambda: ops.shared_prefix_attention(q, pair, own, lens, max_own_len=bad)),
             ("start", lambda: ops.kv_cache_write(cache, k, k, bad)), ("start", lambda: ops.kv_cache_read(cache, bad, 1)),
             ("length", lambda: ops.kv_cache_read(cache, 0, bad))]
    if not isinstance(bad, float):
        calls += [("scale", lambda: ops.shared_prefix_attention(q, pair, own, lens, scale=bad)),
                  ("top_k", lambda: ops.sample_tokens(q[0], torch.zeros(8, device="cuda"), top_k=bad)),
                  ("out", lambda: ops.kv_cache_read(cache, 0, 1, out=bad))]
    for name, call in calls:
        with pytest.raises(ValueError, match=name):
            call()


@pytest.mark.gpu
def test_other_settings_that_are_not_there_or_too_large():
    cache, k = ops.KVCacheInt8.empty(1, 4, 2, 64), torch.zeros(1, 1, 2, 64, dtype=BF16, device="cuda")
    for start in (None, 1 << 70, -(1 << 70), torch.zeros(1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="start"):
            ops.kv_cache_write(cache, k, k, start)
    for length in (None, 1 << 70, 1 << 40, 5):
        with pytest.raises(ValueError, match="length"):
            ops.kv_cache_read(cache, 0, length)
    for out in (7, (k,), (k, k, k), (k, None)):
        with pytest.raises(ValueError, match="out"):
            ops.kv_cache_read(cache, 0, 1, out=out)


@pytest.mark.gpu
def test_whole_numbers_of_other_types_are_taken():
    import numpy as np

    cache, k = ops.KVCacheInt8.empty(1, 4, 2, 64), torch.ones(1, 1, 2, 64, dtype=BF16, device="cuda")
    ops.kv_cache_write(cache, k, k, np.int64(2))
    got = ops.kv_cache_read(cache, np.int32(2), np.int64(1))[0]
    assert got.all() and not cache.k_codes[0, [0, 1, 3]].any()
