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


# ---------------------------------------------------------------------------
# 8-bit cache


def quantise64(x):
    """(codes, scales) from the definition, in 64 bits."""
    x = x.double()
    f, e = torch.frexp(x.abs().amax(-1) / 127)
    scale = torch.ldexp(torch.ceil(f * 256) / 256, e).clamp_min(2.0**-126)
    codes = torch.trunc(x / scale[..., None] + torch.copysign(torch.full_like(x, 0.5), x))
    return codes, scale


def check_rows(cache, k, v, starts):
    n = k.shape[1]
    for x, codes, scales in ((k, cache.k_codes, cache.k_scales), (v, cache.v_codes, cache.v_scales)):
        rc, rs = quantise64(x)
        for b, s in enumerate(starts):
            assert torch.equal(scales[b, s : s + n].double(), rs[b])
            assert torch.equal(codes[b, s : s + n].double(), rc[b])


@pytest.mark.parametrize("B,n,H,D", [(1, 1, 1, 64), (3, 7, 5, 64), (2, 33, 8, 128), (64, 1, 8, 128), (1, 1000, 3, 128)])
def test_cache_write_and_read(B, n, H, D):
    g = gen(20)
    qkv = normal(g, B, n, 3 * H * D, std=2.0)
    k, v = qkv[..., H * D : 2 * H * D].unflatten(-1, (H, D)), qkv[..., 2 * H * D :].unflatten(-1, (H, D))
    cache = ops.KVCacheInt8.empty(B, n + 11, H, D)
    start = torch.randint(0, 12, (B,), generator=g, device="cuda", dtype=torch.int32)
    before = [t.fill_(3).clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    ops.kv_cache_write(cache, k, v, start)
    check_rows(cache, k, v, start.tolist())
    for t, old in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), before):
        for b, s in enumerate(start.tolist()):  # other rows are left as they were
            assert torch.equal(t[b, :s], old[b, :s]) and torch.equal(t[b, s + n :], old[b, s + n :])
    rk, rv = ops.kv_cache_read(cache, start, n)
    for got, codes, scales in ((rk, cache.k_codes, cache.k_scales), (rv, cache.v_codes, cache.v_scales)):
        for b, s in enumerate(start.tolist()):
            exact = codes[b, s : s + n].double() * scales[b, s : s + n].double()[..., None]
            assert torch.equal(got[b], exact.to(BF16))
    # a value is off by at most half a scale, and bf16 rounds by at most 2^-8 of it
    for got, x, scales in ((rk, k, cache.k_scales), (rv, v, cache.v_scales)):
        s = torch.stack([scales[b, i : i + n] for b, i in enumerate(start.tolist())]).double()[..., None]
        assert ((got.double() - x.double()).abs() <= s / 2 + EPS * got.double().abs()).all()


def test_cache_ties_round_away_from_zero():
    """Codes that lie exactly between two integers, for every scale mantissa."""
    x = torch.zeros(1, 128, 1, 64, device="cuda", dtype=BF16)
    m = torch.arange(128, 256, device="cuda")
    x[0, :, 0, 0] = m.to(BF16)
    values = m[:, None] * torch.arange(1, 32, device="cuda")[None, :] / 64.0
    x[0, :, 0, 1:32] = values.to(BF16)
    x[0, :, 0, 32:63] = -values.to(BF16)
    cache = ops.KVCacheInt8.empty(1, 128, 1, 64)
    ops.kv_cache_write(cache, x, x, 0)
    check_rows(cache, x, x, [0])


def test_cache_all_bf16_values():
    """Every finite bf16 value, each next to maxima of many sizes."""
    bits = torch.arange(0, 65536, device="cuda", dtype=torch.int32).to(torch.int16)
    x = bits.view(BF16)
    x = x[x.isfinite()].view(1, -1, 1, 64)[:, :, :, :].contiguous()
    x = torch.cat([x, x.flip(1)[:, torch.randperm(x.shape[1], generator=gen(21), device="cuda")]], 1)
    shuffled = x.reshape(-1)[torch.randperm(x.numel(), generator=gen(22), device="cuda")].view_as(x).contiguous()
    cache = ops.KVCacheInt8.empty(1, x.shape[1], 1, 64)
    ops.kv_cache_write(cache, x, shuffled, 0)
    check_rows(cache, x, shuffled, [0])


def test_cache_zero_tiny_and_bad_rows():
    x = torch.zeros(1, 6, 2, 64, device="cuda", dtype=BF16)
    x[0, 1] = 9.2e-41  # the smallest subnormals
    x[0, 2, 0, 3] = math.nan
    x[0, 3, 1, 63] = -math.inf
    x[0, 4] = 3.3e38
    cache = ops.KVCacheInt8.empty(1, 6, 2, 64)
    ops.kv_cache_write(cache, x, x, 0)
    k, _ = ops.kv_cache_read(cache, 0, 6)
    assert not k[0, 0].any()
    assert ((k[0, 1].double() - x[0, 1].double()).abs() <= 2.0**-127).all()
    assert k[0, 2, 0].isnan().all() and not k[0, 2, 1].any()
    assert k[0, 3, 1].isnan().all() and not k[0, 3, 0].any()
    assert ((k[0, 4].double() / x[0, 4].double() - 1).abs() <= 2.0**-8 + 1 / 254).all()
    assert not cache.k_codes[0, 2, 0].any()


def test_cache_rows_outside_are_skipped():
    g = gen(23)
    k, v = normal(g, 4, 3, 2, 64), normal(g, 4, 3, 2, 64)
    cache = ops.KVCacheInt8.empty(4, 8, 2, 64)
    guard = [t.clone() for t in (cache.k_codes, cache.v_codes)]
    start = torch.tensor([-3, -1, 7, 8], device="cuda", dtype=torch.int32)
    ops.kv_cache_write(cache, k, v, start)
    rk, _ = ops.kv_cache_read(cache, start, 3)
    assert torch.equal(cache.k_codes[0], guard[0][0]) and torch.equal(cache.v_codes[3], guard[1][3])
    assert not rk[0].any() and not rk[3].any() and not rk[1, 0].any() and not rk[2, 1:].any()
    assert rk[1, 1:].any() and rk[2, 0].any()
    assert torch.equal(cache.k_codes[1, :2].double(), quantise64(k)[0][1, 1:])
    assert torch.equal(cache.k_codes[2, 7].double(), quantise64(k)[0][2, 0])


def test_cache_views_and_out():
    g = gen(24)
    big = ops.KVCacheInt8.empty(3, 40, 2, 128)
    k, v = normal(g, 1, 10, 2, 128), normal(g, 1, 10, 2, 128)
    part = big.sequence(1).narrow(5, 20)
    ops.kv_cache_write(part, k, v, 4)
    check_rows(big.sequence(1), k, v, [9])
    assert not big.k_codes[0].any() and not big.k_codes[2].any()
    model = torch.zeros(2, 1, 50, 2, 128, device="cuda", dtype=BF16)
    rk, rv = ops.kv_cache_read(part, 4, 10, out=(model[0][:, 7:17], model[1][:, 7:17]))
    assert torch.equal(rk, ops.kv_cache_read(part, 4, 10)[0]) and rk.data_ptr() == model[0][:, 7:].data_ptr()
    assert not model[:, :, :7].any() and not model[:, :, 17:].any()


def test_cache_64_bit_offsets():
    cache = ops.KVCacheInt8.empty(1, 8_500_000, 4, 64)
    assert cache.k_codes.numel() > 2**31
    g = gen(25)
    k, v = normal(g, 1, 3, 4, 64), normal(g, 1, 3, 4, 64)
    ops.kv_cache_write(cache, k, v, 8_499_990)
    check_rows(cache, k, v, [8_499_990])
    rk, _ = ops.kv_cache_read(cache, 8_499_990, 3)
    assert rk.any() and not cache.k_codes[0, :100].any()


# ---------------------------------------------------------------------------
# sampling


def sample64(logits, u, temperature, top_k, top_p, min_p):
    """The definition in 64 bits, one row: (token, distance of the draw to the nearest border)."""
    import numpy as np

    x = logits.double().cpu().numpy().copy()
    x[np.isnan(x)] = -np.inf
    if temperature <= 0 or x.max() == -np.inf:
        return int(x.argmax()), 1.0
    with np.errstate(invalid="ignore"):
        w = np.exp((x - x.max()) / temperature)
    w[x == x.max()] = 1.0
    order = np.argsort(-x, kind="stable")
    if 0 < top_k < len(x):
        order = order[:top_k]
    if top_p < 1:
        cum = np.cumsum(w[order])
        order = order[: max(1, 1 + np.searchsorted(cum, top_p * cum[-1], side="left"))]
    order = np.sort(order[w[order] >= min_p])
    cum = np.cumsum(w[order])
    at = min(np.searchsorted(cum, u * cum[-1], side="right"), len(order) - 1)
    return int(order[at]), float(np.abs(cum[:-1] / cum[-1] - u).min(initial=1.0))


def check_sample(logits, uniforms, **kw):
    def row(name, default, b):
        value = kw.get(name, default)
        return value[b].item() if isinstance(value, torch.Tensor) else float(torch.tensor(value, dtype=torch.float32))

    tokens = ops.sample_tokens(logits, uniforms, **kw)
    assert tokens.dtype == torch.int64 and tokens.shape == uniforms.shape
    for b in range(len(uniforms)):
        u = min(max(uniforms[b].item(), 0.0), 1 - 2.0**-24)
        want, gap = sample64(logits[b], u, row("temperature", 1.0, b), int(row("top_k", 0, b)), row("top_p", 1.0, b),
                             row("min_p", 0.0, b))
        # fixed point resolves 2^-43 of the largest weight; a draw within 1e-10 of a border may fall on either side
        assert int(tokens[b]) == want or gap < 1e-10, f"row {b}: {int(tokens[b])}, expected {want} (gap {gap})"
    assert torch.equal(ops.sample_tokens(logits, uniforms, **kw), tokens)
    return tokens


SETTINGS = [{}, {"temperature": 0.6}, {"top_k": 1}, {"top_k": 7}, {"top_k": 300, "temperature": 1.7},
            {"top_p": 0.9}, {"top_p": 0.5, "top_k": 40}, {"top_p": 0.999}, {"top_p": 0.0}, {"min_p": 0.1},
            {"min_p": 1.0}, {"top_k": 50, "top_p": 0.95, "min_p": 0.05, "temperature": 0.8},
            {"temperature": 0.0}, {"temperature": 30.0, "top_p": 0.7}]


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("dtype", [BF16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("B,V", [(1, 1), (2, 2), (3, 17), (5, 1000), (2, 32003), (3, 128256), (40, 4097)])
def test_sample(B, V, dtype, settings):
    g = gen(30)
    logits = (torch.randn(B, V, generator=g, device="cuda") * 2).to(dtype)
    check_sample(logits, torch.rand(B, generator=g, device="cuda"), **settings)


@pytest.mark.parametrize("settings", SETTINGS + [{"min_p": 0.5}, {"top_k": 2000, "top_p": 0.8}], ids=str)
@pytest.mark.parametrize("dtype", [BF16, torch.float32], ids=["bf16", "f32"])
def test_sample_many_rows(dtype, settings):
    """More rows than resident clusters; ragged row starts, rising rows (the maximum comes last), masked rows."""
    g = gen(37)
    B, V = 160, 100_003
    x = torch.randn(B, V, generator=g, device="cuda").mul_(2)
    x[1] = torch.arange(V, device="cuda") / 9000.0
    x[2] = 0.5
    x[3, 1:] = -math.inf
    x[4] = -math.inf
    x[5, ::2] = math.nan
    x[6, 50_000] = x[6, 70_000] = math.inf
    x[7, 99_999] = 40.0
    x = x.to(dtype)
    rows = torch.tensor([0, 1, 2, 3, 4, 5, 6, 7, 20, 99, 159], device="cuda")
    u = torch.rand(B, generator=g, device="cuda")
    tokens = ops.sample_tokens(x, u, **settings)
    assert torch.equal(tokens[rows], check_sample(x[rows], u[rows], **settings))


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("kind", ["equal", "two values", "one high", "wide", "signed zeros", "close", "steps"])
@pytest.mark.parametrize("dtype", [BF16, torch.float32], ids=["bf16", "f32"])
def test_sample_shapes_of_rows(kind, dtype, settings):
    g = gen(31)
    V = 20011
    x = torch.randn(2, V, generator=g, device="cuda")
    if kind == "equal":
        x = torch.full_like(x, -3.25)
    elif kind == "two values":
        x = (x > 1).float()
    elif kind == "one high":
        x[:, 777] = 60.0
    elif kind == "wide":
        x *= 1e30
    elif kind == "signed zeros":
        x = torch.where(x > 0, 0.0, -0.0)
    elif kind == "close":
        x = 1000 + x * 1e-3
    else:
        x = torch.arange(V, device="cuda").float().expand(2, V).contiguous() / 500
    check_sample(x.to(dtype), torch.rand(2, generator=g, device="cuda"), **settings)


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("dtype", [BF16, torch.float32], ids=["bf16", "f32"])
def test_sample_masked_rows(dtype, settings):
    """-inf, the type's lowest value, NaN and +inf among the logits; rows with nothing, or one token, left."""
    g = gen(32)
    V = 5003
    x = (torch.randn(9, V, generator=g, device="cuda") * 2).to(dtype)
    x[0, torch.randperm(V, generator=g, device="cuda")[:4900]] = -math.inf
    x[1] = -math.inf
    x[2] = -math.inf
    x[2, 4321] = -7.5
    x[3] = math.nan
    x[4, ::2] = math.nan
    x[5, ::3] = torch.finfo(dtype).min
    x[6] = torch.finfo(dtype).min
    x[7, 100] = x[7, 2000] = math.inf
    x[8, 1:] = -math.inf
    tokens = check_sample(x, torch.rand(9, generator=g, device="cuda"), **settings)
    assert tokens[1] == 0 and tokens[3] == 0 and tokens[2] == 4321 and tokens[8] == 0


def test_sample_rows_with_settings_of_their_own():
    g = gen(33)
    B, V = 64, 12289
    x = torch.randn(B, V, generator=g, device="cuda") * 3
    r = lambda: torch.rand(B, generator=g, device="cuda")  # noqa: E731
    temperature, top_p, min_p = r() * 2, r() * 1.2, r() * 0.2
    top_k = torch.randint(-3, 100, (B,), generator=g, device="cuda", dtype=torch.int32)
    temperature[::7] = 0
    check_sample(x, r(), temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)


def test_sample_uniforms_at_the_ends():
    g = gen(34)
    x = torch.randn(1, 999, generator=g, device="cuda").expand(6, 999).contiguous()
    u = torch.tensor([0.0, 1 - 2.0**-24, 1.0, 2.0, -1.0, 1e-30], device="cuda")
    t = check_sample(x, u)
    assert t[0] == 0 and t[1] == 998 and t[2] == t[3] == t[1] and t[4] == 0
    assert int(ops.sample_tokens(x[:1], torch.full((1,), math.nan, device="cuda"))) == 0


def test_sample_frequencies():
    """Equally spaced uniforms draw every token as often as its weight says, to within one."""
    n = 4096
    p = torch.tensor([0.5, 0.25, 0.125, 0.0625, 0.0625], device="cuda")
    x = p.log().expand(n, 5).contiguous()
    u = (torch.arange(n, device="cuda") + 0.5) / n
    counts = torch.bincount(ops.sample_tokens(x, u), minlength=5)
    assert ((counts - p * n).abs() <= 1).all()


def test_sample_strided_rows_out_and_capture():
    g = gen(35)
    wide_rows = torch.randn(5, 9000, generator=g, device="cuda").to(BF16)
    x = wide_rows[:, 3:8123]
    u = torch.rand(5, generator=g, device="cuda")
    want = check_sample(x, u, top_p=0.9)
    out = torch.full((7,), -1, device="cuda", dtype=torch.int64)
    got = ops.sample_tokens(x, u, top_p=0.9, out=out[1:6])
    assert torch.equal(got, want) and out[0] == -1 and out[6] == -1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = ops.sample_tokens(x, u, top_p=0.9)
    u.copy_(torch.rand(5, generator=g, device="cuda"))
    graph.replay()
    assert torch.equal(again, ops.sample_tokens(x, u, top_p=0.9))


@pytest.mark.parametrize("dtype", [BF16, torch.float32], ids=["bf16", "f32"])
def test_sample_largest_vocabulary(dtype):
    g = gen(36)
    x = torch.randn(2, ops.MAX_VOCAB, generator=g, device="cuda").to(dtype)
    check_sample(x, torch.rand(2, generator=g, device="cuda"), top_p=0.97, top_k=100_000)
    check_sample(x, torch.rand(2, generator=g, device="cuda"), top_p=0.97, temperature=5.0)
