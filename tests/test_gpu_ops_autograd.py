"""How the operators of `megakernels.ops` meet autograd: they have no
derivatives, so tensors that ask for one are refused."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from megakernels import ops
from test_gpu_ops import BF16

pytestmark = pytest.mark.gpu


def attention_inputs():
    def zeros(*shape):
        return torch.zeros(shape, device="cuda", dtype=BF16)

    return zeros(3, 8, 64), (zeros(5, 2, 64), zeros(5, 2, 64)), (zeros(3, 6, 2, 64), zeros(3, 6, 2, 64))


def test_tangents_are_refused():
    """A dual tensor's tangent would be dropped without a word."""
    q, prefix, own = attention_inputs()
    lens = torch.ones(3, device="cuda", dtype=torch.int32)
    x, u = torch.zeros(3, 10, device="cuda"), torch.zeros(3, device="cuda")
    cache, k = ops.KVCacheInt8.empty(3, 6, 2, 64), own[0][:, :2]
    with fwd.dual_level():
        def dual(t):
            return fwd.make_dual(t, torch.ones_like(t))

        for call in (lambda: ops.sample_tokens(dual(x), u), lambda: ops.sample_tokens(x, u, temperature=dual(u + 1)),
                     lambda: ops.shared_prefix_attention(dual(q), prefix, own, lens),
                     lambda: ops.shared_prefix_attention(q, (prefix[0], dual(prefix[1])), own, lens),
                     lambda: ops.shared_prefix_attention(q, prefix, own, lens, out=dual(q.clone())),
                     lambda: ops.kv_cache_write(cache, dual(k), k, 0), lambda: ops.kv_cache_write(cache, k, dual(k), 0),
                     lambda: ops.shared_prefix_attention(dual(q)[:, :4], prefix, own, lens)):
            with pytest.raises(ValueError, match="tangent"):
                call()
        assert ops.sample_tokens(x, u).tolist() == [0, 0, 0]
        plain = fwd.unpack_dual(dual(q)).primal
        assert ops.shared_prefix_attention(plain, prefix, own, lens).shape == q.shape
    assert ops.shared_prefix_attention(q, prefix, own, lens).shape == q.shape


def test_written_tensors_count_a_version():
    """As torch's own in-place operations do, so that autograd notices when a tensor that it saved was written."""
    q, prefix, own = attention_inputs()
    lens = torch.ones(3, device="cuda", dtype=torch.int32)
    cache, k = ops.KVCacheInt8.empty(3, 6, 2, 64), own[0][:, :2]
    out, rows = torch.zeros_like(q), (torch.zeros_like(k), torch.zeros_like(k))
    tokens = torch.zeros(3, device="cuda", dtype=torch.int64)
    x, u = torch.zeros(3, 10, device="cuda"), torch.zeros(3, device="cuda")
    inputs = [q, *prefix, *own, lens, x, u]
    for call, written in [(lambda: ops.shared_prefix_attention(q, prefix, own, lens, out=out), [out]),
                          (lambda: ops.kv_cache_write(cache, k, k, 0), cache._tensors()),
                          (lambda: ops.kv_cache_write(cache, k, k, lens), cache._tensors()),
                          (lambda: ops.kv_cache_read(cache, 0, 2, out=rows), rows),
                          (lambda: ops.sample_tokens(x, u, out=tokens), [tokens])]:
        before, read = [t._version for t in written], [t._version for t in inputs]
        call()
        assert [t._version for t in written] == [v + 1 for v in before]
        assert [t._version for t in inputs] == read
    with torch.inference_mode():
        out = torch.zeros_like(q)  # has no versions
        ops.shared_prefix_attention(q, prefix, own, lens, out=out)


def test_backward_notices_a_write():
    q, prefix, own = attention_inputs()
    lens = torch.ones(3, device="cuda", dtype=torch.int32)
    w, out = torch.ones(64, device="cuda", dtype=BF16, requires_grad=True), torch.zeros_like(q)
    y = (out * w).sum()
    ops.shared_prefix_attention(q, prefix, own, lens, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
