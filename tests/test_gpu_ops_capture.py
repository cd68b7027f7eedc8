"""Operators whose first call in a process is captured into a CUDA graph, on a
stream of its own, and their largest numbers of rows."""

import subprocess
import sys

import pytest
import torch

from megakernels import ops
from test_gpu_ops import BF16, gen

pytestmark = pytest.mark.gpu

FIRST_CALLS = """
import torch
from megakernels import ops

bf16 = torch.bfloat16
q = torch.randn(40, 64, 128, device="cuda").to(bf16)
lens = torch.randint(0, 9, (40,), device="cuda", dtype=torch.int32)
kv = lambda *s: tuple(torch.randn(*s, 2, 128, device="cuda").to(bf16) for _ in range(2))
few, many, own = kv(100), kv(3000), kv(40, 8)
cache = ops.KVCacheInt8.empty(40, 16, 2, 128)
logits, uniforms = torch.randn(40, 1000, device="cuda"), torch.rand(40, device="cuda")

def step():
    a = ops.shared_prefix_attention(q, few, own, lens)
    b = ops.shared_prefix_attention(q, many, own, lens)
    ops.kv_cache_write(cache, *own, 3)
    c = ops.kv_cache_read(cache, 3, 8)
    return a, b, *c, ops.sample_tokens(logits, uniforms, top_p=0.9), ops.sample_tokens(logits.to(bf16), uniforms, top_k=9)

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = step()
graph.replay()
torch.cuda.synchronize()
for x, y in zip(captured, step()):
    assert torch.equal(x, y)
assert ops.attention_status() == 0
print("same")
"""


def test_first_calls_are_captured():
    import os

    env = dict(os.environ, PYTHONPATH=os.pathsep.join(p for p in sys.path if p))
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS], capture_output=True, text=True, timeout=300, env=env)
    assert done.returncode == 0 and "same" in done.stdout, done.stderr[-2000:]


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_one_own_row_for_four_million_query_rows(kind):
    """The most query rows of a call, each with a single key of its own sequence: every result is that key's V."""
    B, H, D = 1 << 16, 64, 64
    g = gen(60)
    q = torch.randn((B, H, D), generator=g, device="cuda", dtype=BF16)
    lens = torch.ones(B, device="cuda", dtype=torch.int32)
    lens[5] = 0
    if kind == "int8":
        codes = torch.randint(-127, 128, (B, 1, H, D), generator=g, device="cuda", dtype=torch.int8)
        scales = (torch.rand((B, 1, H), generator=g, device="cuda") * 0.02 + 0.005).to(BF16)
        own = ops.KVCacheInt8(codes, scales, codes, scales)
        prefix = ops.KVCacheInt8.empty(1, 0, H, D)
    else:
        k = torch.randn((B, 1, H, D), generator=g, device="cuda", dtype=BF16)
        own, prefix = (k, k), tuple(torch.empty(0, H, D, device="cuda", dtype=BF16) for _ in range(2))
    out = ops.shared_prefix_attention(q, prefix, own, lens)
    assert not out[5].any()
    for b in range(0, B, 4096):
        if kind == "int8":
            v = codes[b : b + 4096, 0].float() * scales[b : b + 4096, 0].float()[..., None]
        else:
            v = k[b : b + 4096, 0].float()
        v[lens[b : b + 4096] == 0] = 0
        # 8-bit rows: V's scale enters with the probability, rounded to bf16, and the result is rounded once more
        bound = (2.0**-7 + 2.0**-15) * v.abs() if kind == "int8" else 0 * v
        assert ((out[b : b + 4096].float() - v).abs() <= bound).all()
