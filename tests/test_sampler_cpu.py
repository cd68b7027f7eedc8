"""The random numbers of sampled decoding, on CPU: which steps get which, and
that all ranks of a tensor-parallel model draw with the same ones (gloo, two
processes)."""

import os
import tempfile

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from megakernels.generators import SamplingParams, _Sampler

CPU = torch.device("cpu")


def test_numbers_come_from_the_generator_in_blocks_of_steps():
    s = _Sampler(SamplingParams(generator=torch.Generator().manual_seed(3)), 4)
    got = torch.stack([s.draw(CPU).clone() for _ in range(2 * s.STEPS + 5)])
    g = torch.Generator().manual_seed(3)
    want = torch.cat([torch.rand(s.STEPS, 4, generator=g) for _ in range(3)])
    assert torch.equal(got, want[: len(got)])


class Globs:
    """What setup_tensor_parallel leaves on a rank's globals."""

    def __init__(self, world, group=None):
        self.tp_world, self.tp_group = world, group


def _rank(rank, world, init, out):
    import sys

    sys.path[:0] = [p for p in os.environ.get("EK_TEST_PATHS", "").split(os.pathsep) if p]
    dist.init_process_group("gloo", init_method=f"file://{init}", rank=rank, world_size=world)
    try:
        group = dist.new_group(list(range(world)))
        for i, g in enumerate((None, group)):
            params = SamplingParams(generator=torch.Generator().manual_seed(100 + rank))  # not in the same state
            s = _Sampler(params, 1, Globs(world, g))
            torch.save(torch.stack([s.draw(CPU).clone() for _ in range(s.STEPS + 3)]), f"{out}.{i}.{rank}")
    finally:
        dist.destroy_process_group()


def test_all_ranks_draw_with_the_same_numbers():
    import sys

    os.environ["EK_TEST_PATHS"] = os.pathsep.join(p for p in sys.path if p)
    with tempfile.TemporaryDirectory() as tmp:
        mp.spawn(_rank, args=(2, f"{tmp}/init", f"{tmp}/u"), nprocs=2, join=True)
        for i in range(2):
            a, b = (torch.load(f"{tmp}/u.{i}.{r}") for r in range(2))
            assert torch.equal(a, b)
            assert torch.equal(a[:256], torch.rand(256, 1, generator=torch.Generator().manual_seed(100)))
