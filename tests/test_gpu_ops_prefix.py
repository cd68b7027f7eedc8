"""`shared_prefix_attention` where the prefix serves so many query rows that the
tensor-core kernel takes it (more than 16 per KV head, and 2^25 elements of K
over all tiles of 8 query rows), against the definition in 64 bits. Tolerances
as in test_gpu_ops."""

import math

import pytest
import torch

from megakernels import ops
from test_gpu_ops import BF16, check_attention, gen, int8_rows, make, normal

pytestmark = pytest.mark.gpu

KINDS = pytest.mark.parametrize("kind", ["bf16", "int8"])


def serves(B, P, Hq, H, D):
    rows = B * Hq // H
    return rows > 16 and -(-rows // 8) * H * P * D >= 2**25


def case(seed, kind, B, P, T, Hq, H, D):
    assert serves(B, P, Hq, H, D)
    return make(seed, kind, B, P, T, Hq, H, D)


@KINDS
# 4096, 4160, 4224 and 4256 query rows of a KV head: blocks of 256 and a rest of 0, 64, 128 and 160
@pytest.mark.parametrize("B", [128, 130, 132, 133])
@pytest.mark.parametrize("P", [256, 257, 319, 383, 384, 385, 1000])
def test_lengths_and_blocks(kind, B, P):
    check_attention(*case(1, kind, B, P, 9, 64, 2, 128))


@KINDS
@pytest.mark.parametrize("P", [16, 17, 127, 128, 129])
def test_short_prefixes(kind, P):
    check_attention(*case(2, kind, 256, P, 5, 512, 16, 128))


@KINDS
@pytest.mark.parametrize("B,P,T,heads", [
    (8, 10923, 40, (24, 8, 128)), (8, 11111, 1, (24, 8, 128)), (1, 87425, 3, (17, 1, 128)), (17, 10930, 70, (16, 16, 64)),
    (100, 2979, 33, (14, 2, 64)), (61, 8200, 100, (32, 8, 64)), (9, 60001, 20, (14, 2, 64)), (300, 5000, 12, (24, 8, 128)),
], ids=str)
def test_heads(kind, B, P, T, heads):
    check_attention(*case(3, kind, B, P, T, *heads))


@KINDS
def test_one_row_of_prefix_for_four_million(kind):
    """The most query rows of a call; one key each, so every row is that key's V."""
    B, H, D = 1 << 16, 64, 64
    assert serves(B, 1, H, H, D)
    g = gen(4)
    if kind == "int8":
        prefix, own = int8_rows(g, 1, 1, H, D), int8_rows(g, B, 0, H, D)
        v = (prefix.v_codes.float() * prefix.v_scales.float()[..., None])[0, 0]
    else:
        prefix = (normal(g, 1, H, D), normal(g, 1, H, D))
        own = tuple(torch.empty(B, 0, H, D, device="cuda", dtype=BF16) for _ in range(2))
        v = prefix[1][0].float()
    q = torch.randn((B, H, D), generator=g, device="cuda", dtype=BF16)
    lens = torch.zeros(B, device="cuda", dtype=torch.int32)
    out = ops.shared_prefix_attention(q, prefix, own, lens)
    # 8-bit rows: the scale enters through the probability, rounded to bf16, and the result is rounded once more
    bound = (2.0**-7 + 2.0**-15) * v.abs() if kind == "int8" else 0 * v
    for part in out.split(4096):
        assert ((part.float() - v).abs() <= bound).all()


@KINDS
@pytest.mark.parametrize("scale", [0.0, -0.125, 2.0])
def test_scales(kind, scale):
    check_attention(*case(5, kind, 66, 8000, 10, 32, 2, 64), scale=scale)


@KINDS
def test_lens_are_clamped_and_bounded(kind):
    q, prefix, own, lens = case(6, kind, 60, 8777, 50, 32, 2, 64)
    lens[0], lens[1], lens[2] = -5, 1000, 50
    check_attention(q, prefix, own, lens)
    check_attention(q, prefix, own, lens, max_own_len=23)
    check_attention(q, prefix, own, lens, max_own_len=0)


def test_large_scores():
    """Scores that grow along the keys: the running maximum moves in every tile."""
    q, prefix, own, lens = case(7, "bf16", 150, 3500, 40, 32, 2, 64)
    prefix[0].mul_(torch.linspace(0, 12, 3500, device="cuda").view(-1, 1, 1).to(BF16))
    check_attention(q, prefix, own, lens)


def test_nan_stays_in_its_row():
    q, prefix, own, lens = case(8, "bf16", 90, 6000, 10, 32, 2, 64)
    clean = ops.shared_prefix_attention(q, prefix, own, lens)
    q[1, 2, 5] = math.nan
    got = ops.shared_prefix_attention(q, prefix, own, lens)
    assert got[1, 2].isnan().all()
    got[1, 2] = clean[1, 2]
    assert torch.equal(got, clean)


@KINDS
def test_rows_behind_the_prefix_are_not_read(kind):
    q, prefix, own, lens = case(9, kind, 70, 3333, 50, 32, 2, 128)
    P = 3300  # the last tile is cut

    def cut():
        return prefix.narrow(0, P) if kind == "int8" else tuple(t[:P] for t in prefix)

    expected = ops.shared_prefix_attention(q, cut(), own, lens)
    for t in (prefix.k_scales, prefix.v_scales) if kind == "int8" else prefix:
        (t[:, P:] if kind == "int8" else t[P:]).fill_(math.nan)
    got = ops.shared_prefix_attention(q, cut(), own, lens)
    assert torch.equal(got, expected) and not got.isnan().any()


@KINDS
def test_strides(kind):
    """q inside a fused product, the prefix stored [heads, rows, D] inside a wider buffer, one head shown as several."""
    g = gen(10)
    B, H, D, P, T = 45, 2, 64, 11900, 21
    assert serves(B, P, 32, H, D)
    q = normal(g, B, (32 + 2 * H) * D)[:, : 32 * D].view(B, 32, D)
    lens = torch.randint(0, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    if kind == "bf16":
        prefix = tuple(normal(g, H, P + 9, 2 * D)[:, 4 : 4 + P, D:].transpose(0, 1) for _ in range(2))
        own = (normal(g, B, T, H, D), normal(g, B, T, H, D))
    else:
        full = int8_rows(g, H, P + 9, 1, D)

        def turned(codes, scales):
            return codes[:, 9:].permute(2, 1, 0, 3), scales[:, 9:].permute(2, 1, 0)

        prefix = ops.KVCacheInt8(*turned(full.k_codes, full.k_scales), *turned(full.v_codes, full.v_scales))
        own = int8_rows(g, B, T, H, D)
    check_attention(q, prefix, own, lens)
    wide_out = torch.zeros(B, 48, D, device="cuda", dtype=BF16)
    got = ops.shared_prefix_attention(q, prefix, own, lens, out=wide_out[:, 8:40])
    assert torch.equal(got, ops.shared_prefix_attention(q, prefix, own, lens))
    assert not wide_out[:, :8].any() and not wide_out[:, 40:].any()
    if kind == "bf16":
        one = tuple(t[:, :1].expand(P, H, D) for t in prefix)
        check_attention(q, one, own, lens)


@KINDS
def test_repeats_captures_and_streams(kind):
    q, prefix, own, lens = case(11, kind, 80, 5700, 64, 16, 2, 128)
    first = ops.shared_prefix_attention(q, prefix, own, lens)
    for _ in range(10):
        assert torch.equal(ops.shared_prefix_attention(q, prefix, own, lens), first)
    sides = [torch.cuda.Stream() for _ in range(2)]
    others = []
    for side in sides:  # two calls at once, each with its own workspace
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            others.append(ops.shared_prefix_attention(q, prefix, own, lens))
    for side, other in zip(sides, others):
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.shared_prefix_attention(q, prefix, own, lens)
    q.copy_(normal(gen(12), *q.shape))
    lens.copy_(lens.flip(0))
    graph.replay()
    graph.replay()
    expected = ops.shared_prefix_attention(q, prefix, own, lens)
    assert torch.equal(out, expected) and not torch.equal(out, first)
    assert ops.attention_status(q.device) == 0
