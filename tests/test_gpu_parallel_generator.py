"""Sampling in `MK_Generator` and the operators together in `ParallelGenerator`:
prompt, shared prefix, caches of both kinds, sampling, and the hand-over of one
continuation to the megakernel."""

import pytest
import torch

import cases
from megakernels import ops

pytestmark = pytest.mark.gpu

PROMPT = 40
NEW = 6


def ids(n=PROMPT, seed=3):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, cases.TINY["vocab_size"], (n,), generator=g).cuda()


def params(seed=0, **kw):
    from megakernels.generators import SamplingParams

    return SamplingParams(generator=torch.Generator(device="cuda").manual_seed(seed), **kw)


def mk_generator(model, seq_len, sampling=None):
    from megakernels.demos.latency.mk import LatencyMK_Interpreter
    from megakernels.demos.latency.scheduler import LatencyScheduleBuilder
    from megakernels.generators import MK_Generator
    from megakernels.scheduler import assign_to_sms, tensorize_instructions

    s = LatencyScheduleBuilder.build(model, seq_len=seq_len)
    tensorize_instructions(s.globs, assign_to_sms("rr", schedule=s))
    return MK_Generator(model, LatencyMK_Interpreter(), s, sampling=sampling)


def generate(kind, n, **kw):
    from megakernels.generators import ParallelGenerator

    model = cases.tiny_model("cuda")
    gen = ParallelGenerator(model, n, NEW, sampling=params(**kw), kv_cache=kind)
    out = torch.zeros(n, NEW + 1, dtype=torch.int64, device="cuda")
    out[:, 0] = gen.prefill(ids())
    logits = []
    for i in range(NEW):
        gen.generate(out, PROMPT, 1, ntok_already_generated=1 + i)
        logits.append(gen.logits.float())
    return model, gen, out, logits


@pytest.mark.parametrize("n", [1, 5, 20])
def test_continuations_match_the_prompt_pass(n):
    """Every step's logits equal those of the whole text in one dense pass, within
    the bounds that the prompt pass itself is held to against the decode path (0.1
    and 0.03 standard deviations: both sum the same bf16 products in other orders)."""
    model, gen, out, logits = generate("bf16", n, temperature=1.5)
    assert n == 1 or len({tuple(r) for r in out.tolist()}) > 1  # they diverge
    other = cases.tiny_model("cuda")
    for b in range(min(n, 3)):
        for i in (0, NEW - 1):
            ref = other.prefill(torch.cat([ids(), out[b, : i + 1]]), 0).float()
            d = (logits[i][b] - ref).abs()
            assert d.max() <= 0.1 * ref.std() and d.pow(2).mean().sqrt() <= 0.03 * ref.std()


def test_int8_caches_hold_the_quantised_rows():
    """Layer 0's rows depend on the tokens alone, so the 8-bit run holds exactly the quantised rows of the bf16 run."""
    model, gen, out, _ = generate("int8", 4, temperature=1.0)
    from megakernels.generators import ParallelGenerator

    plain = ParallelGenerator(cases.tiny_model("cuda"), 4, NEW, sampling=params())
    plain.prefill(ids())
    for i in range(NEW):
        plain.run(out[:, i])
    for src, cache in ((plain.prefix[0], gen.prefix[0]), (plain.own[0], gen.own[0])):
        k, v = (t.unsqueeze(0) if t.dim() == 3 else t for t in src)
        expected = ops.KVCacheInt8.empty(*k.shape)
        ops.kv_cache_write(expected, k, v, 0)
        for a, b in zip(expected._tensors(), cache._tensors()):
            assert torch.equal(a, b)


def test_greedy_continuations_agree_and_follow_the_logits():
    _, _, out, logits = generate("bf16", 3, temperature=0.0)
    assert (out == out[:1]).all()
    for i, x in enumerate(logits):
        assert torch.equal(out[:, i + 1], x.argmax(-1))


def test_same_seed_same_tokens():
    a, b, c = (generate("int8", 6, seed=s, temperature=1.2, top_k=50, top_p=0.9)[2] for s in (7, 7, 8))
    assert torch.equal(a, b) and not torch.equal(a, c)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_hand_over_to_the_megakernel(kind):
    """The handed-over rows are the sequence's, and the megakernel's next step
    agrees with the generator's own next step on the same token (bf16: within
    the bounds of test_prefill; 8-bit rows: the same bounds against a dense
    pass over the same cached rows)."""
    import mk_llama

    model, gen, out, _ = generate(kind, 3, temperature=1.3)
    end = gen.hand_over(1)
    assert end == PROMPT + NEW
    for l, own in enumerate(gen.own):
        rows = (ops.kv_cache_read(own.sequence(1), 0, NEW) if kind == "int8" else [t[1:2] for t in own])
        for cache, r in zip(model.stacked_kv_cache, rows):
            assert torch.equal(cache[l, :1, PROMPT:end], r)
    mk = mk_generator(model, end + 2)
    mk.run(out[1:2, NEW:], end)
    torch.cuda.synchronize()
    mk_llama.check()
    got = mk.schedule.globs.logits.float()
    ref = model.prefill(out[1, NEW:], end).float()  # rewrites row `end`, over the same cached rows
    d = (got - ref).abs()
    assert d.max() <= 0.1 * ref.std() and d.pow(2).mean().sqrt() <= 0.03 * ref.std()


def test_mk_generator_samples():
    import mk_llama

    model = cases.tiny_model("cuda")
    greedy = mk_generator(model, PROMPT + 8)
    first = greedy.prefill(ids())
    expected = greedy.run(first.view(1, 1), PROMPT).clone()
    cold = mk_generator(model, PROMPT + 8, sampling=params(temperature=0.0))
    assert torch.equal(cold.prefill(ids()), first)
    assert torch.equal(cold.run(first.view(1, 1), PROMPT), expected)
    hot = mk_generator(model, PROMPT + 8, sampling=params(seed=5, temperature=2.0, top_p=0.95))
    u = torch.rand(256, 1, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    token = hot.prefill(ids())
    for i in range(4):
        logits = hot.schedule.globs.logits
        token = hot.run(token.view(1, 1), PROMPT + i).clone()
        want = ops.sample_tokens(logits.view(1, -1), u[i + 1], temperature=2.0, top_p=0.95)
        assert int(token) == int(want)
    torch.cuda.synchronize()
    mk_llama.check()


def test_generator_refuses():
    from megakernels.generators import ParallelGenerator

    model = cases.tiny_model("cuda")
    for kw, what in [({"num_sequences": 0}, "positive"), ({"max_new_tokens": 0}, "positive"), ({"kv_cache": "fp4"}, "kv_cache")]:
        with pytest.raises(ValueError, match=what):
            ParallelGenerator(**{"model": model, "num_sequences": 2, "max_new_tokens": 2, **kw})
    with pytest.raises(ValueError, match="CUDA"):
        ParallelGenerator(cases.tiny_model("cpu"), 2, 2)
    gen = ParallelGenerator(model, 2, 1)
    first = torch.zeros(2, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="prefill first"):
        gen.run(first)
    gen.prefill(ids())
    with pytest.raises(ValueError, match="expected 2"):
        gen.run(first[:1])
    gen.run(first)
    with pytest.raises(ValueError, match="hold 1 new"):
        gen.run(first)
    with pytest.raises(ValueError, match="sequence 2"):
        gen.hand_over(2)
    with pytest.raises(ValueError, match="ntok_already_generated"):
        gen.generate(torch.zeros(2, 4, dtype=torch.int64, device="cuda"), PROMPT, 1, 1)


def test_a_second_prompt_starts_over():
    """After longer use, a shorter prompt gives what a new generator gives."""
    for kind in ("bf16", "int8"):
        model, gen, _, _ = generate(kind, 3)
        fresh = type(gen)(model, 3, NEW, sampling=params(seed=9, top_k=20), kv_cache=kind)
        gen.sampler = type(gen.sampler)(params(seed=9, top_k=20), 3)
        got = []
        for g in (gen, fresh):
            out = torch.zeros(3, NEW + 1, dtype=torch.int64, device="cuda")
            out[:, 0] = g.prefill(ids(17, seed=4))
            g.generate(out, 17, NEW)
            got.append(out)
        assert torch.equal(*got)


def test_sampled_steps_are_not_captured():
    gen = generate("bf16", 2)[1]
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            gen.sampler(gen.logits)
    torch.cuda.synchronize()
    assert gen.sampler(gen.logits).shape == (2,)
