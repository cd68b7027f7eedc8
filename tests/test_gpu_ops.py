"""The operators of `megakernels.ops` against plain implementations in 64 bits,
at the sizes, lengths and masks where they can go wrong.

Tolerances. bf16 rounds a result by at most 2^-8 of its size. In the attention
each probability is also rounded to bf16 before it multiplies V, an error of at
most 2^-8 * sum(p |v|) in the normalised sum; fp32 sums and the exponential add
less than 2^-16 of the same. So |out - exact| <= 2^-8 |exact| + (2^-8 + 2^-16) *
sum(p |v|), and for 8-bit rows the probability times V's scale is rounded, which
bounds the same way. Cache values (code * scale) are compared exactly."""

import math

import pytest
import torch

from megakernels import ops

pytestmark = pytest.mark.gpu

EPS = 2.0**-8
BF16 = torch.bfloat16


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(BF16)


def int8_rows(g, b, n, h, d):
    def one():
        return (torch.randint(-127, 128, (b, n, h, d), generator=g, device="cuda", dtype=torch.int8),
                (torch.rand((b, n, h), generator=g, device="cuda") * 0.02 + 0.005).to(BF16))

    return ops.KVCacheInt8(*one(), *one())


def wide(store):
    """(k, v) in 64 bits, [batch, rows, heads, D]."""
    if isinstance(store, ops.KVCacheInt8):
        return (store.k_codes.double() * store.k_scales.double()[..., None],
                store.v_codes.double() * store.v_scales.double()[..., None])
    return tuple(t.double() if t.dim() == 4 else t.double()[None] for t in store)


def attention64(q, prefix, own, lens, scale=None):
    """(out, lse, sum p |v|) per sequence and head, from the definition."""
    B, Hq, D = q.shape
    (kp, vp), (ko, vo) = wide(prefix), wide(own)
    H = ko.shape[2]
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device=q.device)
    for b in range(B):
        n = int(lens[b])
        k, v = torch.cat([kp[0], ko[b, :n]]), torch.cat([vp[0], vo[b, :n]])
        if len(k) == 0:
            continue
        s = torch.einsum("hgd,khd->hgk", q[b].double().view(H, -1, D), k) * scale
        p = torch.softmax(s, -1)
        out[b] = torch.einsum("hgk,khd->hgd", p, v).reshape(Hq, D)
        size[b] = torch.einsum("hgk,khd->hgd", p, v.abs()).reshape(Hq, D)
        lse[b] = torch.logsumexp(s, -1).reshape(Hq)
    return out, lse, size


def check_attention(q, prefix, own, lens, **kw):
    out, lse = ops.shared_prefix_attention(q, prefix, own, lens, return_lse=True, **kw)
    limit = kw.get("max_own_len", (own.k_codes if isinstance(own, ops.KVCacheInt8) else own[0]).shape[1])
    ref, ref_lse, size = attention64(q, prefix, own, lens.clamp(0, limit), kw.get("scale"))
    assert out.dtype == BF16 and out.shape == q.shape
    err = (out.double() - ref).abs() - (EPS * ref.abs() + (EPS + 2.0**-16) * size)
    assert err.max().item() <= 1e-30, f"{err.max().item()} beyond the bound at {err.argmax().item()}"
    empty = ref_lse.isinf()
    assert torch.equal(lse.isinf() & (lse < 0), empty)
    assert not out[empty].any()
    # fp32 scores of size |s| carry about D 2^-24 sum |q k| and the sum 2^-20
    assert ((lse.double() - ref_lse)[~empty].abs() <= 1e-4 * (1 + ref_lse[~empty].abs())).all()
    return out


HEADS = [(32, 8, 64), (24, 8, 128), (16, 16, 64), (14, 2, 64), (17, 1, 128), (1, 1, 128)]


def make(seed, kind, B, P, T, Hq, H, D, lens=None):
    g = gen(seed)
    q = normal(g, B, Hq, D, std=1.5)
    if kind == "int8":
        prefix, own = int8_rows(g, 1, P, H, D), int8_rows(g, B, T, H, D)
    else:
        prefix = (normal(g, P, H, D), normal(g, P, H, D))
        own = (normal(g, B, T, H, D), normal(g, B, T, H, D))
    if lens is None:
        lens = torch.randint(0, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        lens[0] = 0
        lens[-1] = T
    return q, prefix, own, lens


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("B,P,T", [(1, 1, 1), (2, 15, 17), (5, 129, 65), (7, 1000, 3), (64, 300, 33), (130, 257, 20)])
def test_attention(kind, heads, B, P, T):
    check_attention(*make(1, kind, B, P, T, *heads))


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("P", [1, 127, 128, 129, 255, 256, 384, 4099, 20000])
@pytest.mark.parametrize("B", [6, 40, 65])
def test_attention_prefix_lengths(kind, P, B):
    check_attention(*make(2, kind, B, P, 9, 8, 2, 128))


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("P,T", [(0, 40), (40, 0), (0, 0)])
@pytest.mark.parametrize("B", [3, 50])
def test_attention_without_prefix_or_own(kind, P, T, B):
    q, prefix, own, lens = make(3, kind, B, P, T, 8, 2, 64)
    check_attention(q, prefix, own, torch.minimum(lens, torch.tensor(T, device="cuda", dtype=torch.int32)))


def test_attention_empty_rows_are_zero():
    q, prefix, own, lens = make(4, "bf16", 6, 0, 30, 8, 2, 64)
    lens[1] = lens[4] = 0
    out = check_attention(q, prefix, own, lens)
    assert not out[1].any() and not out[4].any()


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("B", [3, 60])
def test_attention_lens_are_clamped_and_bounded(kind, B):
    q, prefix, own, lens = make(5, kind, B, 77, 50, 8, 2, 64)
    lens[0], lens[1], lens[2] = -5, 1000, 50
    check_attention(q, prefix, own, lens)
    check_attention(q, prefix, own, lens, max_own_len=23)
    check_attention(q, prefix, own, lens, max_own_len=0)


@pytest.mark.parametrize("B", [4, 70])
def test_attention_never_reads_past_the_end(B):
    """NaN and infinity in the rows behind each sequence and behind the prefix."""
    q, prefix, own, lens = make(6, "bf16", B, 400, 50, 8, 2, 128)
    expected = ops.shared_prefix_attention(q, tuple(t[:333] for t in prefix), own, lens)
    for t in prefix:
        t[333:] = math.nan
    for b in range(B):
        for i, t in enumerate(own):
            t[b, int(lens[b]):] = (math.nan, math.inf)[i]
    got = ops.shared_prefix_attention(q, tuple(t[:333] for t in prefix), own, lens)
    assert torch.equal(got, expected) and not got.isnan().any()


@pytest.mark.parametrize("B", [4, 70])
def test_attention_int8_never_reads_past_the_end(B):
    q, prefix, own, lens = make(7, "int8", B, 400, 50, 8, 2, 128)
    expected = ops.shared_prefix_attention(q, prefix.narrow(0, 333), own, lens)
    for s in (prefix.k_scales, prefix.v_scales):
        s[:, 333:] = math.nan
    for b in range(B):
        own.k_scales[b, int(lens[b]):] = math.nan
        own.v_scales[b, int(lens[b]):] = math.inf
    got = ops.shared_prefix_attention(q, prefix.narrow(0, 333), own, lens)
    assert torch.equal(got, expected) and not got.isnan().any()


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("B", [3, 66])
@pytest.mark.parametrize("scale", [0.0, -0.125, 2.0])
def test_attention_scales(kind, B, scale):
    check_attention(*make(8, kind, B, 200, 10, 4, 2, 64), scale=scale)


@pytest.mark.parametrize("B", [2, 33, 150])
def test_attention_large_scores(B):
    """Scores that grow along the keys: the running maximum moves in every tile."""
    q, prefix, own, lens = make(9, "bf16", B, 1500, 40, 4, 2, 64)
    prefix[0].mul_(torch.linspace(0, 12, 1500, device="cuda").view(-1, 1, 1).to(BF16))
    check_attention(q, prefix, own, lens)


@pytest.mark.parametrize("B", [2, 90])
def test_attention_nan_stays_in_its_row(B):
    q, prefix, own, lens = make(10, "bf16", B, 200, 10, 4, 2, 64)
    clean = ops.shared_prefix_attention(q, prefix, own, lens)
    q[1, 2, 5] = math.nan
    got = ops.shared_prefix_attention(q, prefix, own, lens)
    assert got[1, 2].isnan().all()
    got[1, 2] = clean[1, 2]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("B", [3, 45])
def test_attention_strides(kind, B):
    """q inside a fused product, caches as views of larger ones (a layer, another order of heads and rows)."""
    g = gen(11)
    H, D, P, T = 2, 64, 150, 21
    qkv = normal(g, B, (8 + 2 * H) * D)
    q = qkv[:, : 8 * D].view(B, 8, D)
    lens = torch.randint(0, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)

    def views(x_bf16, codes):
        # stored [heads, rows, D] inside a wider buffer
        if codes:
            c = torch.randint(-127, 128, x_bf16, generator=g, device="cuda", dtype=torch.int8)
            s = (torch.rand(x_bf16[:-1], generator=g, device="cuda") * 0.02 + 0.005).to(BF16)
            return c, s
        return normal(g, *x_bf16)

    if kind == "bf16":
        prefix = tuple(views((H, P + 9, 2 * D), False)[:, 4 : 4 + P, D:].transpose(0, 1) for _ in range(2))
        own = tuple(views((B, H, T + 3, D), False)[:, :, 3:].transpose(1, 2) for _ in range(2))
    else:
        def pair(b, n, extra):
            c, s = views((b, H, n + extra, D), True)
            return c[:, :, extra:].transpose(1, 2), s[:, :, extra:].transpose(1, 2)

        prefix = ops.KVCacheInt8(*pair(1, P, 9), *pair(1, P, 9))
        own = ops.KVCacheInt8(*pair(B, T, 3), *pair(B, T, 3))
    check_attention(q, prefix, own, lens)
    wide_out = torch.zeros(B, 16, D, device="cuda", dtype=BF16)
    got = ops.shared_prefix_attention(q, prefix, own, lens, out=wide_out[:, 4:12])
    assert torch.equal(got, ops.shared_prefix_attention(q, prefix, own, lens))
    assert not wide_out[:, :4].any() and not wide_out[:, 12:].any()


@pytest.mark.parametrize("B", [3, 45])
def test_attention_expanded_prefix(B):
    """One stored head shown as several (a zero stride)."""
    g = gen(12)
    q = normal(g, B, 8, 64)
    k, v = normal(g, 100, 1, 64), normal(g, 100, 1, 64)
    own = (normal(g, B, 5, 4, 64), normal(g, B, 5, 4, 64))
    lens = torch.full((B,), 5, device="cuda", dtype=torch.int32)
    check_attention(q, (k.expand(100, 4, 64), v.expand(100, 4, 64)), own, lens)


def test_attention_64_bit_offsets():
    """Own rows of the last sequences lie past 2^31 elements."""
    B, T, H, D = 5, 4_200_000, 2, 64
    own = tuple(torch.empty(B, T, H, D, device="cuda", dtype=BF16) for _ in range(2))
    assert own[0].numel() > 2**31
    g = gen(13)
    lens = torch.tensor([3, 0, 64, 1, 200], device="cuda", dtype=torch.int32)
    for b in range(B):
        for t in own:
            t[b, : int(lens[b])] = normal(g, int(lens[b]), H, D)
    q = normal(g, B, 8, D)
    prefix = (normal(g, 50, H, D), normal(g, 50, H, D))
    small = tuple(t[:, :200].clone() for t in own)
    a = ops.shared_prefix_attention(q, prefix, own, lens, max_own_len=200)
    assert torch.equal(a, ops.shared_prefix_attention(q, prefix, small, lens))
    check_attention(q, prefix, small, lens)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("B", [4, 80])
def test_attention_repeats_captures_and_streams(kind, B):
    q, prefix, own, lens = make(14, kind, B, 700, 64, 8, 2, 128)
    first = ops.shared_prefix_attention(q, prefix, own, lens)
    for _ in range(3):
        assert torch.equal(ops.shared_prefix_attention(q, prefix, own, lens), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.shared_prefix_attention(q, prefix, own, lens)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, first)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.shared_prefix_attention(q, prefix, own, lens)
        graphs.append((graph, out))
    q2 = normal(gen(15), *q.shape)
    q.copy_(q2)
    lens.copy_(lens.flip(0))
    for graph, out in graphs + graphs:
        graph.replay()
    torch.cuda.synchronize()
    expected = ops.shared_prefix_attention(q, prefix, own, lens)
    assert not torch.equal(expected, first)
    for _, out in graphs:
        assert torch.equal(out, expected)
    assert ops.attention_status(q.device) == 0
