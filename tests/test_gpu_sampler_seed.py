"""A generator that is seeded anew between steps gives the same tokens again."""

import pytest
import torch

from test_gpu_parallel_generator import NEW, PROMPT, ids, mk_generator, params

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", ["own", "own state", "default"])
def test_seeding_anew_repeats_the_continuations(how):
    import cases
    from megakernels.generators import ParallelGenerator, SamplingParams

    model = cases.tiny_model("cuda")
    sampling = SamplingParams(temperature=1.5) if how == "default" else params(temperature=1.5)
    gen = ParallelGenerator(model, 4, NEW, sampling=sampling)
    state = None if how == "default" else sampling.generator.get_state()

    def tokens(seed):
        if how == "default":
            torch.manual_seed(seed)
        elif how == "own":
            sampling.generator.manual_seed(seed)
        else:
            sampling.generator.set_state(state)
        out = torch.zeros(4, NEW + 1, dtype=torch.int64, device="cuda")
        out[:, 0] = gen.prefill(ids())
        gen.generate(out, PROMPT, NEW)
        return out

    first = tokens(11)
    assert torch.equal(tokens(11), first)
    assert how == "own state" or not torch.equal(tokens(12), first)
    assert torch.equal(tokens(11), first)


def test_seeding_anew_in_mk_generator():
    import cases

    model = cases.tiny_model("cuda")
    sampling = params(temperature=3.0)
    gen = mk_generator(model, PROMPT + 8, sampling=sampling)
    runs = []
    for _ in range(2):
        sampling.generator.manual_seed(21)
        token = gen.prefill(ids())
        runs.append([int(token)])
        for i in range(5):
            token = gen.run(token.view(1, 1), PROMPT + i).clone()
            runs[-1].append(int(token))
    assert runs[0] == runs[1]
