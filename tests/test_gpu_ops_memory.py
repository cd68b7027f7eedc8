"""Memory that the arguments of an operator have in common: refused where blocks
would write it while others read or write it, in any order; taken where it is
only read, or interleaved without a common element."""

import random

import pytest
import torch

from megakernels import ops
from test_gpu_ops import BF16, gen, normal

pytestmark = pytest.mark.gpu


def refuses(call, *args, **kw):
    with pytest.raises(ValueError, match="same memory"):
        call(*args, **kw)


def test_caches_that_overlap_by_a_row():
    g = gen(100)
    k = normal(g, 2, 3, 2, 64)
    codes = torch.zeros(2, 9, 2, 64, device="cuda", dtype=torch.int8)
    scales = torch.zeros(2, 9, 2, device="cuda", dtype=BF16)
    for a, b in [(slice(0, 5), slice(4, 9)), (slice(4, 9), slice(0, 5)), (slice(0, 8), slice(1, 9))]:
        other = ops.KVCacheInt8.empty(2, a.stop - a.start, 2, 64)
        refuses(ops.kv_cache_write, ops.KVCacheInt8(codes[:, a], other.k_scales, codes[:, b], other.v_scales), k, k, 0)
        refuses(ops.kv_cache_write, ops.KVCacheInt8(other.k_codes, scales[:, a], other.v_codes, scales[:, b]), k, k, 0)
    # halves of the rows, and rows in turn, have nothing in common
    for a, b in [(slice(0, 4), slice(4, 8)), (slice(0, 8, 2), slice(1, 8, 2))]:
        cache = ops.KVCacheInt8(codes[:, a], scales[:, a], codes[:, b], scales[:, b])
        ops.kv_cache_write(cache, k, -k, 1)
        plain = ops.KVCacheInt8.empty(2, 4, 2, 64)
        ops.kv_cache_write(plain, k, -k, 1)
        for x, y in zip(plain._tensors(), cache._tensors()):
            assert torch.equal(x[:, 1:], y[:, 1:])


def test_rows_and_outputs_inside_the_cache():
    g = gen(101)
    raw = torch.zeros(1 << 16, device="cuda", dtype=torch.int8)
    codes = raw[: 2 * 8 * 2 * 64].view(2, 8, 2, 64)
    inside, behind = (raw[at : at + 2 * 4 * 2 * 64 * 2].view(BF16).view(2, 4, 2, 64) for at in (1024, 2048))
    other = ops.KVCacheInt8.empty(2, 8, 2, 64)
    cache = ops.KVCacheInt8(codes, other.k_scales, other.v_codes, other.v_scales)
    k = normal(g, 2, 4, 2, 64)
    refuses(ops.kv_cache_write, cache, inside, k, 0)
    refuses(ops.kv_cache_write, cache, k, inside, 0)
    refuses(ops.kv_cache_read, cache, 0, 4, out=(inside, k))
    refuses(ops.kv_cache_read, cache, 0, 4, out=(k, inside))
    refuses(ops.kv_cache_read, cache, 0, 4, out=(k, k))
    ops.kv_cache_write(cache, behind, k, 0)
    ops.kv_cache_read(cache, 0, 4, out=(behind, k))
    starts = raw[:8].view(torch.int32)
    refuses(ops.kv_cache_write, cache, k, k, starts)
    refuses(ops.kv_cache_read, other, k.view(torch.int32).reshape(-1)[:2], 4, out=(k, behind))


def test_outputs_inside_the_inputs():
    q, prefix, own = normal(gen(102), 3, 8, 64), (normal(gen(103), 5, 2, 64),) * 2, (normal(gen(104), 3, 6, 2, 64),) * 2
    lens = q.view(torch.int32).reshape(-1)[:3]
    refuses(ops.shared_prefix_attention, torch.zeros_like(q), prefix, own, lens, out=q)
    # in place of q, K or V: they have been read by then
    lens = torch.tensor([0, 3, 6], device="cuda", dtype=torch.int32)
    want = ops.shared_prefix_attention(q, prefix, own, lens)
    again = q.clone()
    assert torch.equal(ops.shared_prefix_attention(again, prefix, own, lens, out=again), want)
    v = own[1].clone()
    assert torch.equal(ops.shared_prefix_attention(q, prefix, (own[0], v), lens, out=v.view(-1)[: q.numel()].view(q.shape)), want)
    x, u = torch.zeros(4, 64, device="cuda"), torch.zeros(8, device="cuda")
    refuses(ops.sample_tokens, x, u[:4], out=u.view(torch.int64))
    refuses(ops.sample_tokens, x, u[:4], out=x.view(torch.int64)[1, :4])
    t = torch.zeros(8, device="cuda")
    refuses(ops.sample_tokens, x, u[:4], temperature=t[:4], out=t.view(torch.int64))
    ops.sample_tokens(x[:, :56], u[:4], out=x.view(torch.int64)[3, 28:])  # behind the last row


def test_views_of_one_buffer_at_random():
    """Refused exactly where the index sets meet."""
    rng = random.Random(5)
    cache = ops.KVCacheInt8.empty(2, 3, 2, 64)
    buffer = torch.zeros(40_000, device="cuda", dtype=BF16)
    met = apart = 0
    while met < 60 or apart < 60:
        views, sets = [], []
        for _ in range(2):
            n = rng.randrange(1, 4)
            unit = rng.choice([64, 72, 128])
            strides = rng.sample([unit, unit * rng.choice([2, 3, 4]), unit * rng.choice([6, 7, 9, 12])], 3)
            start = 8 * rng.randrange(0, 300)
            view = torch.as_strided(buffer, (2, n, 2, 64), (*strides, 1), start)
            index = [start + b * strides[0] + r * strides[1] + h * strides[2] + d
                     for b in range(2) for r in range(n) for h in range(2) for d in range(64)]
            assert max(index) < buffer.numel()
            views.append(view), sets.append(index)
        n = min(v.shape[1] for v in views)
        views = [v[:, :n] for v in views]
        sets = [{int(i) for i in torch.as_strided(torch.arange(buffer.numel()), v.shape, v.stride(), v.storage_offset()).reshape(-1)}
                for v in views]
        if any(len(s) < v.numel() for s, v in zip(sets, views)):
            continue  # elements of one view meet
        try:
            ops.kv_cache_read(cache, 0, n, out=tuple(views))
        except ValueError as e:
            if "elements overlap" in str(e):
                continue  # refused for itself: rows of one view in another's gaps
            assert "same memory" in str(e) and sets[0] & sets[1], (e, [(v.shape, v.stride(), v.storage_offset()) for v in views])
            met += 1
        else:
            assert not sets[0] & sets[1], [(v.shape, v.stride(), v.storage_offset()) for v in views]
            apart += 1
