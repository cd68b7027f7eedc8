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
