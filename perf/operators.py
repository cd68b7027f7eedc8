"""Measured cases of the operators for several sampled continuations of one
prompt: attention over a shared prefix (`shared_prefix_attention`), the 8-bit
KV cache (`kv_cache_write`, `kv_cache_read`) and token sampling
(`sample_tokens`).

With `own = False`, `run` computes an operator from its definition in
elementary torch operations; with `own = True` it makes the call that a user
makes of `megakernels.ops`.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "epic-kernel_b200")


def _ops():
    """The framework's operators, as a user's program finds them."""
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from megakernels import ops

    return ops


# ---------------------------------------------------------------------------
# cases


def _attention(batch, prefix, own_len, q_heads, kv_heads, head_dim, kind):
    return {"op": "attention", "batch": batch, "prefix": prefix, "own": own_len,
            "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "kind": kind}


def _cache(op, batch, length, capacity, kv_heads, head_dim, ragged):
    return {"op": op, "batch": batch, "length": length, "capacity": capacity,
            "kv_heads": kv_heads, "head_dim": head_dim, "ragged": ragged}


def _sample(batch, vocab, dtype, temperature, top_k, top_p, min_p, per_row=False, spread=2.0):
    return {"op": "sample", "batch": batch, "vocab": vocab, "dtype": dtype,
            "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "per_row": per_row, "spread": spread}


def listed():
    return [
        # one continuation of a short prompt: a single layer of the 1B at the start of a chat, latency only
        {"name": "attn_one"} | _attention(1, 128, 40, 32, 8, 64, "bf16"),
        # sixteen answers to one 2048-token prompt, 1B heads
        {"name": "attn_n16_kv2048"} | _attention(16, 2048, 256, 32, 8, 64, "bf16"),
        # sixty-one continuations of a long document in an 8-bit cache, odd lengths, Mixtral heads
        {"name": "attn_n61_int8"} | _attention(61, 16001, 1023, 32, 8, 128, "int8"),
        # a large best-of-n over a long context, 3B heads (three query heads share a KV head)
        {"name": "attn_n256_long"} | _attention(256, 32768, 512, 24, 8, 128, "bf16"),
        # the rows of one decode step of sixty-four sequences, each at its own position, written and read back
        {"name": "cache_step"} | _cache("write", 64, 1, 1024, 8, 128, True),
        # a prompt of 32001 tokens (one layer) written to the 8-bit cache and read back
        {"name": "cache_prompt"} | _cache("write", 1, 32001, 32768, 8, 128, False),
        # the tail of nine continuations of the 1B read back for the bf16 engine
        {"name": "cache_read_tail"} | _cache("read", 9, 333, 1024, 8, 64, True),
        # a long context read back for the bf16 engine
        {"name": "cache_read_long"} | _cache("read", 1, 65536, 65536, 8, 128, False),
        # one token of a chat: the 1B's vocabulary, the usual top-k with top-p
        {"name": "sample_one"} | _sample(1, 128256, "bf16", 0.7, 50, 0.9, 0.0),
        # Mixtral's vocabulary size made odd, fp32 logits, every row with settings of its own
        {"name": "sample_rows"} | _sample(17, 32003, "f32", 1.0, 40, 0.95, 0.05, per_row=True),
        # sixty-four continuations, nucleus only: the cut lies deep in the vocabulary
        {"name": "sample_nucleus"} | _sample(64, 128256, "bf16", 1.0, 0, 0.95, 0.0),
        # the largest batch, fp32 logits, plain temperature with min-p
        {"name": "sample_n256"} | _sample(256, 128256, "f32", 0.8, 0, 1.0, 0.02),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "sample", "sample", "write", "read"])
    if op == "attention":
        q_heads, kv_heads, head_dim = rng.choice(
            [(32, 8, 64), (24, 8, 128), (32, 8, 128), (16, 16, 64), (14, 2, 64), (16, 1, 128)])
        kind = rng.choice(["bf16", "int8"])
        batch = _log_int(rng, 1, 256)
        prefix = _log_int(rng, 1, 32768)
        own_len = _log_int(rng, 1, 512 if batch > 64 else 1024)
        return _attention(batch, prefix, own_len, q_heads, kv_heads, head_dim, kind)
    if op in ("write", "read"):
        kv_heads, head_dim = rng.choice([(8, 64), (8, 128), (2, 64), (1, 128)])
        ragged = rng.random() < 0.5
        batch = _log_int(rng, 1, 64)
        length = _log_int(rng, 1, 65536 // batch if op == "read" else max(1, 32001 // batch))
        return _cache(op, batch, length, length + (rng.randrange(1, 300) if ragged else 0), kv_heads, head_dim, ragged)
    top_k = rng.choice([0, _log_int(rng, 1, 2000)])
    top_p = rng.choice([1.0, rng.uniform(0.05, 0.999)])
    min_p = rng.choice([0.0, rng.uniform(0.001, 0.5)])
    return _sample(_log_int(rng, 1, 256), _log_int(rng, 64, 128256), rng.choice(["bf16", "f32"]),
                   rng.uniform(0.3, 2.0), top_k, top_p, min_p, rng.random() < 0.3, rng.uniform(0.5, 4.0))


def _own_lens(case):
    """Own lengths of the sequences, 0 to case["own"], spread evenly; the last one is full."""
    n, top = case["batch"], case["own"]
    return [(b * 2654435761 % 2**32) * (top + 1) // 2**32 for b in range(n - 1)] + [top]


# ---------------------------------------------------------------------------
# inputs


def _quantised_store(gen, shape):
    """Codes and scales as a cache holds them: every (token, head) row reaches +-127."""
    codes = torch.randint(-127, 128, shape, generator=gen, device="cuda", dtype=torch.int8)
    scales = (torch.rand(shape[:-1], generator=gen, device="cuda") * 0.02 + 0.01).to(torch.bfloat16)
    return codes, scales


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(shape, std=1.0):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16).mul_(std)

    d = {}
    if case["op"] == "attention":
        B, P, T, H, D = case["batch"], case["prefix"], case["own"], case["kv_heads"], case["head_dim"]
        # the query rows lie inside the fused QKV product, as the model's step leaves them
        qkv = normal((B, (case["q_heads"] + 2 * H) * D), 1.5)
        d["q"] = qkv[:, : case["q_heads"] * D].view(B, case["q_heads"], D)
        order = torch.randperm(B, generator=gen, device="cuda")
        d["lens"] = torch.tensor(_own_lens(case), device="cuda", dtype=torch.int32)[order]
        if case["kind"] == "bf16":
            d["prefix"] = (normal((P, H, D)), normal((P, H, D)))
            d["own"] = (normal((B, T, H, D)), normal((B, T, H, D)))
        else:
            d["prefix"] = _quantised_store(gen, (1, P, H, D)) + _quantised_store(gen, (1, P, H, D))
            d["own"] = _quantised_store(gen, (B, T, H, D)) + _quantised_store(gen, (B, T, H, D))
    elif case["op"] in ("write", "read"):
        B, n, T, H, D = case["batch"], case["length"], case["capacity"], case["kv_heads"], case["head_dim"]
        d["start"] = (torch.randint(0, T - n + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
                      if case["ragged"] else 0)
        if case["op"] == "write":
            # K and V rows lie inside the fused QKV product (four query heads per KV head)
            qkv = normal((B, n, 6 * H * D))
            d["k"] = qkv[..., 4 * H * D : 5 * H * D].unflatten(-1, (H, D))
            d["v"] = qkv[..., 5 * H * D :].unflatten(-1, (H, D))
            d["store"] = (torch.zeros((B, T, H, D), device="cuda", dtype=torch.int8),
                          torch.zeros((B, T, H), device="cuda", dtype=torch.bfloat16),
                          torch.zeros((B, T, H, D), device="cuda", dtype=torch.int8),
                          torch.zeros((B, T, H), device="cuda", dtype=torch.bfloat16))
        else:
            d["store"] = _quantised_store(gen, (B, T, H, D)) + _quantised_store(gen, (B, T, H, D))
    else:
        B, V = case["batch"], case["vocab"]
        logits = torch.randn((B, V), generator=gen, device="cuda").mul_(case["spread"])
        d["logits"] = logits.to(torch.bfloat16) if case["dtype"] == "bf16" else logits
        d["uniforms"] = torch.rand((B,), generator=gen, device="cuda")
        for name in ("temperature", "top_k", "top_p", "min_p"):
            value = case[name]
            if case["per_row"]:
                if name == "top_k":
                    value = torch.randint(0, 2 * value + 2, (B,), generator=gen, device="cuda", dtype=torch.int32)
                else:
                    value = value * torch.rand((B,), generator=gen, device="cuda").mul_(0.5).add_(0.5)
            d[name] = value
    return d


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own:
        ops = _ops()
        if case["op"] == "attention" and case["kind"] == "int8":
            state["prefix"] = ops.KVCacheInt8(*state["prefix"])
            state["own"] = ops.KVCacheInt8(*state["own"])
        if "store" in state:
            state["cache"] = ops.KVCacheInt8(*state["store"])
    return state


# ---------------------------------------------------------------------------
# one pass


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"attention": _plain_attention, "write": _plain_write, "read": _plain_read,
                "sample": _plain_sample}[op](state)
    ops = _ops()
    if op == "attention":
        return ops.shared_prefix_attention(state["q"], state["prefix"], state["own"], state["lens"])
    if op == "write":  # written rows are returned as the values that the cache now holds for them
        ops.kv_cache_write(state["cache"], state["k"], state["v"], state["start"])
        return ops.kv_cache_read(state["cache"], state["start"], state["case"]["length"])
    if op == "read":
        return ops.kv_cache_read(state["cache"], state["start"], state["case"]["length"])
    return ops.sample_tokens(state["logits"], state["uniforms"], temperature=state["temperature"],
                             top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"])


def _float_store(store):
    """K and V in fp32 of a (k, v) pair or of (k codes, k scales, v codes, v scales)."""
    if len(store) == 2:
        return store[0].float(), store[1].float()
    kc, ks, vc, vs = store
    return kc.float() * ks.float().unsqueeze(-1), vc.float() * vs.float().unsqueeze(-1)


def _plain_attention(state):
    q = state["q"].float()
    B, Hq, D = q.shape
    kp, vp = (t.reshape(-1, *t.shape[-2:]) for t in _float_store(state["prefix"]))  # [P, H, D]
    ko, vo = _float_store(state["own"])  # [B, T, H, D]
    H, G = kp.shape[1], Hq // kp.shape[1]
    scale = 1.0 / math.sqrt(D)
    q = q.view(B, H, G, D) * scale
    shared = q.transpose(0, 1).reshape(H, B * G, D) @ kp.permute(1, 2, 0)  # [H, B G, P]
    shared = shared.view(H, B, G, -1).transpose(0, 1)
    private = q @ ko.permute(0, 2, 3, 1)  # [B, H, G, T]
    hidden = torch.arange(ko.shape[1], device=q.device) >= state["lens"].view(B, 1, 1, 1)
    private = private.masked_fill(hidden, float("-inf"))
    top = private.amax(-1, keepdim=True)
    if shared.shape[-1]:
        top = torch.maximum(top, shared.amax(-1, keepdim=True))
    top = torch.where(top.isinf(), 0.0, top)  # a row without any key
    ws, wp = torch.exp(shared - top), torch.exp(private - top)
    total = ws.sum(-1, keepdim=True) + wp.sum(-1, keepdim=True)
    o = (ws.transpose(0, 1).reshape(H, B * G, -1) @ vp.transpose(0, 1)).view(H, B, G, D).transpose(0, 1)
    o = o + wp @ vo.transpose(1, 2)
    o = torch.where(total > 0, o / total, 0.0)
    return o.reshape(B, Hq, D).to(torch.bfloat16)


def _plain_quantise(x):
    x = x.float()
    scale = (x.abs().amax(-1) / 127).contiguous()
    scale = ((scale.view(torch.int32) + 0xFFFF) & ~0xFFFF).view(torch.float32).clamp_min(2.0**-126)
    codes = torch.floor(x.abs() / scale.unsqueeze(-1) + 0.5) * x.sign()
    return codes.to(torch.int8), scale.to(torch.bfloat16)


def _rows(state):
    case = state["case"]
    n = torch.arange(case["length"], device="cuda")
    start = state["start"]
    if not case["ragged"]:
        start = torch.full((case["batch"],), start, device="cuda", dtype=torch.int32)
    return torch.arange(case["batch"], device="cuda").unsqueeze(1), start.long().unsqueeze(1) + n


def _plain_read(state):
    at = _rows(state)
    k, v = _float_store([t[at] for t in state["store"]])
    return k.to(torch.bfloat16), v.to(torch.bfloat16)


def _plain_write(state):
    at = _rows(state)
    for t, value in zip(state["store"], _plain_quantise(state["k"]) + _plain_quantise(state["v"])):
        t[at] = value
    return _plain_read(state)


def _column(value, like):
    if not isinstance(value, torch.Tensor):
        value = torch.full((like.shape[0],), value, device=like.device,
                           dtype=torch.int32 if isinstance(value, int) else torch.float32)
    return value.unsqueeze(1)


def _plain_sample(state):
    x = state["logits"].double()
    x = torch.where(x.isnan(), float("-inf"), x)
    temperature, top_p, min_p = (_column(state[n], x).double() for n in ("temperature", "top_p", "min_p"))
    top_k = _column(state["top_k"], x)
    top_k = torch.where(top_k > 0, top_k, x.shape[1])
    w = torch.exp((x - x.amax(1, keepdim=True)) / temperature)
    ranked, order = torch.sort(w, dim=1, descending=True, stable=True)
    keep = torch.arange(x.shape[1], device=x.device) < top_k
    ranked = ranked * keep
    before = ranked.cumsum(1) - ranked
    keep &= (before < top_p * ranked.sum(1, keepdim=True)) | (top_p >= 1)
    keep[:, 0] = True
    keep &= ranked >= min_p
    kept = torch.zeros_like(w).scatter_(1, order, (ranked * keep))
    cum = kept.cumsum(1)
    goal = state["uniforms"].double().unsqueeze(1) * cum[:, -1:]
    return (cum > goal).to(torch.int8).argmax(1)


# ---------------------------------------------------------------------------
# the definitions in 64 bits, apart from the plain forms


def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, d)
    if case["op"] == "sample":
        return _exact_sample(d)
    B, n = case["batch"], case["length"]
    starts = d["start"].tolist() if case["ragged"] else [0] * B
    if case["op"] == "read":
        kc, ks, vc, vs = d["store"]
        return tuple(torch.stack([c[b, s : s + n].double() * z[b, s : s + n].double()[..., None]
                                  for b, s in enumerate(starts)]) for c, z in ((kc, ks), (vc, vs)))
    out = []
    for x in (d["k"].double(), d["v"].double()):
        fraction, exponent = torch.frexp(x.abs().amax(-1, keepdim=True) / 127)
        scale = torch.ldexp(torch.ceil(fraction * 256) / 256, exponent)  # eight bits, rounded up
        scale = torch.where(scale < 2.0**-126, 2.0**-126, scale)
        out.append(torch.trunc(x / scale + torch.copysign(torch.full_like(x, 0.5), x)) * scale)
    return tuple(out)


def _exact_attention(case, d):
    def wide(store, b):
        if len(store) == 2:
            return [t[b].double() for t in store]
        return [store[i][b].double() * store[i + 1][b].double()[..., None] for i in (0, 2)]

    B, Hq, D = d["q"].shape
    H = case["kv_heads"]
    kp, vp = wide(d["prefix"], slice(None) if case["kind"] == "bf16" else 0)
    kp, vp = kp.transpose(0, 1).contiguous(), vp.transpose(0, 1).contiguous()  # [H, P, D]
    out = torch.zeros((B, Hq, D), device="cuda", dtype=torch.float64)
    for b, n in enumerate(d["lens"].tolist()):
        ko, vo = (t[:n].transpose(0, 1) for t in wide(d["own"], b))
        q = d["q"][b].double().view(H, Hq // H, D) / math.sqrt(D)
        s = torch.cat([q @ kp.transpose(1, 2), q @ ko.transpose(1, 2)], dim=2)  # [H, G, P + n]
        if s.shape[2] == 0:
            continue
        p = torch.softmax(s, dim=2)
        cut = kp.shape[1]
        out[b] = (p[..., :cut] @ vp + p[..., cut:] @ vo).view(Hq, D)
    return out


def _exact_sample(d):
    logits = d["logits"].double().cpu().numpy()
    B, V = logits.shape

    def column(name):
        value = d[name]
        if isinstance(value, torch.Tensor):
            return value.double().cpu().numpy()
        # scalars reach the operator in single precision
        return np.full(B, np.float32(value), dtype=np.float64)

    temperature, top_k, top_p, min_p = (column(n) for n in ("temperature", "top_k", "top_p", "min_p"))
    u = d["uniforms"].double().cpu().numpy()
    tokens = np.zeros(B, dtype=np.int64)
    for b in range(B):
        w = np.exp((logits[b] - logits[b].max()) / temperature[b])
        order = np.argsort(-logits[b], kind="stable")
        if top_k[b] > 0:
            order = order[: int(top_k[b])]
        if top_p[b] < 1:
            cum = np.cumsum(w[order])
            order = order[: max(1, 1 + np.searchsorted(cum, top_p[b] * cum[-1], side="left"))]
        order = np.sort(order[w[order] >= min_p[b]])
        cum = np.cumsum(w[order])
        tokens[b] = order[min(np.searchsorted(cum, u[b] * cum[-1], side="right"), len(order) - 1)]
    return torch.from_numpy(tokens).cuda()


# ---------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    if case["op"] == "attention":
        B, P, H, D, Hq = case["batch"], case["prefix"], case["kv_heads"], case["head_dim"], case["q_heads"]
        rows = P + sum(_own_lens(case))
        row = H * (D * 2 if case["kind"] == "bf16" else D + 2)  # one token's K (or V)
        keys = B * P + sum(_own_lens(case))
        return {"bytes": 2 * rows * row + 2 * B * Hq * D * 2 + 4 * B, "flops": 4 * keys * Hq * D}
    if case["op"] in ("write", "read"):
        heads = case["batch"] * case["length"] * case["kv_heads"]
        held = 2 * heads * (case["head_dim"] + 2)  # codes and scales of K and V
        values = 2 * heads * case["head_dim"] * 2
        if case["op"] == "read":
            return {"bytes": held + values, "flops": values // 2}
        return {"bytes": values + held + values, "flops": 3 * values // 2}
    size = 2 if case["dtype"] == "bf16" else 4
    n = case["batch"] * case["vocab"]
    return {"bytes": n * size + case["batch"] * 12, "flops": 4 * n}
