"""What the operators of `megakernels.ops` refuse before anything is launched.
Types, ranks and devices are checked first, so those refusals need no GPU."""

import ctypes
import math

import pytest
import torch

from megakernels import ek, ops
from megakernels.build import build

build()  # no-op when the libraries are newer than their sources

BF16 = torch.bfloat16


def zeros(*shape, dtype=BF16, device="cpu"):
    return torch.zeros(shape, dtype=dtype, device=device)


@pytest.mark.parametrize("logits,uniforms,what", [
    ([1.0], zeros(1, dtype=torch.float32), "expected a tensor"),
    (zeros(2, 8, dtype=torch.float16), zeros(2, dtype=torch.float32), "logits: dtype"),
    (zeros(8), zeros(1, dtype=torch.float32), "logits: 1-D"),
    (zeros(2, 8), zeros(2, dtype=torch.float32), "logits: must be a CUDA tensor"),
])
def test_sample_tokens_refuses(logits, uniforms, what):
    with pytest.raises(ValueError, match=what):
        ops.sample_tokens(logits, uniforms)


def test_attention_refuses():
    q, lens = zeros(1, 8, 64), zeros(1, dtype=torch.int32)
    pair, own = (zeros(4, 2, 64), zeros(4, 2, 64)), (zeros(1, 4, 2, 64), zeros(1, 4, 2, 64))
    for args, what in [((q.float(), pair, own, lens), "q: dtype"), ((q[0], pair, own, lens), "q: 2-D"),
                       ((q, pair, own, lens), "q: must be a CUDA tensor"), ((q, pair[0], own, lens), "prefix: expected"),
                       ((q, pair, None, lens), "own: expected"), ((q, (*pair, 1), own, lens), "prefix: expected")]:
        with pytest.raises(ValueError, match=what):
            ops.shared_prefix_attention(*args)


def test_cache_refuses():
    codes, scales = zeros(1, 4, 2, 64, dtype=torch.int8), zeros(1, 4, 2)
    for tensors, what in [((codes.to(torch.uint8), scales, codes, scales), "k_codes: dtype"),
                          ((codes[0], scales, codes, scales), "k_codes: 3-D"),
                          ((codes, scales, codes, scales), "k_codes: must be a CUDA tensor")]:
        with pytest.raises(ValueError, match=what):
            ops.KVCacheInt8(*tensors)
    for call in (lambda: ops.kv_cache_write(None, codes, codes, 0), lambda: ops.kv_cache_read(codes, 0, 1)):
        with pytest.raises(ValueError, match="expected KVCacheInt8"):
            call()


def test_c_entries_refuse_null_and_bad_sizes():
    lib = ek.load_library()
    for name in ("ek_kv_write", "ek_kv_read", "ek_prefix_attention", "ek_sample"):
        assert getattr(lib, name)(None, None) == 1
        assert b"NULL" in lib.ek_last_error()
    lib.ek_prefix_attention_workspace.restype = ctypes.c_int64
    assert lib.ek_prefix_attention_workspace(None) == -1
    assert lib.ek_prefix_attention_status(0, None, 0) == 1


# ---------------------------------------------------------------------------
# with a GPU


def cuda(*shape, dtype=BF16):
    return zeros(*shape, dtype=dtype, device="cuda")


def refuses(what, call, *args, **kw):
    with pytest.raises(ValueError, match=what):
        call(*args, **kw)


@pytest.mark.gpu
def test_sample_tokens_refuses_on_the_gpu():
    x, u = cuda(3, 10), cuda(3, dtype=torch.float32)
    refuses("uniforms: expected", ops.sample_tokens, x, u[:2])
    refuses("uniforms: dtype", ops.sample_tokens, x, u.double())
    refuses("uniforms: must be a CUDA", ops.sample_tokens, x, u.cpu())
    refuses("uniforms: expected a contiguous", ops.sample_tokens, x, cuda(6, dtype=torch.float32)[::2])
    refuses("last dimension", ops.sample_tokens, cuda(10, 3).T, u)
    refuses("vocabulary 0", ops.sample_tokens, cuda(3, 0), u)
    refuses("vocabulary", ops.sample_tokens, cuda(3, ops.MAX_VOCAB + 1), u)
    for kw, what in [({"temperature": -1.0}, "temperature"), ({"temperature": math.inf}, "temperature"),
                     ({"temperature": math.nan}, "temperature"), ({"temperature": "hot"}, "temperature"),
                     ({"top_k": -1}, "top_k"), ({"top_k": 1.5}, "top_k"), ({"top_p": 1.1}, "top_p"),
                     ({"top_p": -0.1}, "top_p"), ({"top_p": math.nan}, "top_p"), ({"min_p": 2.0}, "min_p"),
                     ({"top_k": cuda(3, dtype=torch.int64)}, "top_k: dtype"),
                     ({"top_p": cuda(2, dtype=torch.float32)}, "top_p: expected"),
                     ({"out": cuda(3, dtype=torch.int32)}, "out: dtype"),
                     ({"out": cuda(2, dtype=torch.int64)}, "out: expected")]:
        refuses(what, ops.sample_tokens, x, u, **kw)
    grad = torch.zeros(3, 10, device="cuda", requires_grad=True)
    refuses("requires grad", ops.sample_tokens, grad, u)
    with torch.no_grad():
        assert ops.sample_tokens(grad, u).tolist() == [0, 0, 0]
    assert ops.sample_tokens(cuda(0, 10), cuda(0, dtype=torch.float32)).shape == (0,)


@pytest.mark.gpu
def test_attention_refuses_on_the_gpu():
    q, lens = cuda(3, 8, 64), cuda(3, dtype=torch.int32)
    prefix, own = (cuda(5, 2, 64), cuda(5, 2, 64)), (cuda(3, 6, 2, 64), cuda(3, 6, 2, 64))
    f = ops.shared_prefix_attention
    refuses("head_dim 32", f, cuda(3, 8, 32), prefix, own, lens)
    refuses("inconsistent", f, cuda(2, 8, 64), prefix, own, lens)
    refuses("inconsistent", f, cuda(3, 8, 128), prefix, own, lens)
    refuses("inconsistent", f, q, (cuda(5, 4, 64), cuda(5, 4, 64)), own, lens)
    refuses("multiple of kv_heads", f, cuda(3, 7, 64), prefix, own, lens)
    refuses("same shape", f, q, (prefix[0], cuda(4, 2, 64)), own, lens)
    refuses("own_lens: dtype", f, q, prefix, own, lens.long())
    refuses("own_lens: expected", f, q, prefix, own, lens[:2])
    refuses("max_own_len", f, q, prefix, own, lens, max_own_len=7)
    refuses("max_own_len", f, q, prefix, own, lens, max_own_len=-1)
    refuses("scale", f, q, prefix, own, lens, scale=math.inf)
    refuses("16-byte", f, cuda(3, 8, 65)[..., :64], prefix, own, lens)
    refuses("16-byte", f, cuda(3, 8, 72)[..., 4:68], prefix, own, lens)
    refuses("last dimension", f, cuda(3, 64, 8).transpose(1, 2), prefix, own, lens)
    refuses("out: ", f, q, prefix, own, lens, out=cuda(3, 8, 64, dtype=torch.float32))
    refuses("overlap", f, q, prefix, own, lens, out=cuda(1, 8, 64).expand(3, 8, 64))
    cache = ops.KVCacheInt8.empty(3, 6, 2, 64)
    refuses("both", f, q, prefix, cache, lens)
    refuses("batch 3, expected 1", f, q, cache, cache, lens)
    refuses("requires grad", f, torch.zeros(3, 8, 64, device="cuda", dtype=BF16, requires_grad=True), prefix, own, lens)
    assert f(cuda(0, 8, 64), prefix, (cuda(0, 6, 2, 64), cuda(0, 6, 2, 64)), lens[:0]).shape == (0, 8, 64)


@pytest.mark.gpu
def test_cache_refuses_on_the_gpu():
    cache = ops.KVCacheInt8.empty(2, 6, 2, 64)
    k = cuda(2, 3, 2, 64)
    refuses("outside the cache", ops.kv_cache_write, cache, k, k, 4)
    refuses("outside the cache", ops.kv_cache_write, cache, k, k, -1)
    refuses("outside the cache", ops.kv_cache_read, cache, 5, 2)
    refuses("start: dtype", ops.kv_cache_write, cache, k, k, cuda(2, dtype=torch.int64))
    refuses("start: expected", ops.kv_cache_write, cache, k, k, cuda(1, dtype=torch.int32))
    refuses("expected \\[batch", ops.kv_cache_write, cache, cuda(2, 3, 4, 64), cuda(2, 3, 4, 64), 0)
    refuses("v: dtype", ops.kv_cache_write, cache, k, k.float(), 0)
    refuses("length -1", ops.kv_cache_read, cache, 0, -1)
    refuses("out: 3 rows", ops.kv_cache_read, cache, 0, 2, out=(k, k))
    refuses("overlap", ops.kv_cache_read, cache, 0, 3, out=(cuda(1, 3, 2, 64).expand(2, 3, 2, 64), k))
    c = cache._tensors()
    refuses("do not match", ops.KVCacheInt8, c[0], c[1][:, :5], c[2], c[3])
    refuses("do not match", ops.KVCacheInt8, c[0], c[1], c[2][:, :5], c[3])
    refuses("head_dim 32", ops.KVCacheInt8.empty, 1, 4, 2, 32)
    expanded = ops.KVCacheInt8(*(t[:1].expand(2, *t.shape[1:]) for t in c))
    refuses("overlap", ops.kv_cache_write, expanded, k, k, 0)
    assert ops.kv_cache_read(cache, 6, 0)[0].shape == (2, 0, 2, 64)
    ops.kv_cache_write(cache, k[:, :0], k[:, :0], 6)


@pytest.mark.gpu
def test_memory_shared_within_a_call_is_refused():
    q, lens = cuda(3, 8, 64), cuda(3, dtype=torch.int32)
    prefix, own = (cuda(5, 2, 64), cuda(5, 2, 64)), (cuda(3, 6, 2, 64), cuda(3, 6, 2, 64))
    row = cuda(1, 2, 64).expand(5, 2, 64)  # one row shown as five
    refuses("prefix k: a row repeated", ops.shared_prefix_attention, q, (row, prefix[1]), own, lens)
    refuses("own v: a row repeated", ops.shared_prefix_attention, q, prefix, (own[0], cuda(3, 1, 2, 64).expand(3, 6, 2, 64)), lens)
    c = ops.KVCacheInt8.empty(3, 6, 2, 64)
    one = ops.KVCacheInt8(*(t[:, :1].expand(t.shape) for t in c._tensors()))
    refuses("own k_codes: a row repeated", ops.shared_prefix_attention, q, c.sequence(0), one, lens)
    same = ops.KVCacheInt8(c.k_codes, c.k_scales, c.k_codes, c.v_scales)
    k = cuda(3, 1, 2, 64)
    refuses("same memory", ops.kv_cache_write, same, k, k, 0)
    refuses("same memory", ops.kv_cache_read, c, 0, 1, out=(k, k))


@pytest.mark.gpu
def test_sizes_beyond_the_kernels_are_value_errors():
    many = ops.KVCacheInt8.empty(65536, 1, 1, 64)
    k = cuda(65536, 1, 1, 64)
    refuses("batch 65536", ops.kv_cache_write, many, k, k, 0)
    refuses("batch 65536", ops.kv_cache_read, many, 0, 1)
    n = (1 << 22) + 1
    q, lens = cuda(1, 1, 64).expand(n, 1, 64), cuda(n, dtype=torch.int32)
    prefix, own = (cuda(5, 1, 64), cuda(5, 1, 64)), tuple(cuda(1, 1, 1, 64).expand(n, 1, 1, 64) for _ in range(2))
    refuses("batch \\* q_heads", ops.shared_prefix_attention, q, prefix, own, lens)
