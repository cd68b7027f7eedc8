"""Token loops around the megakernel (`megakernels/generators.py` of
epic-kernel, :11-166).

`MK_Generator.run` does per token what the reference does: embed the input
token into `hidden_states`, reset the barrier counters, zero the logits, launch
the megakernel, and take the argmax of the logits, all on the current stream
with no host synchronisation. With an interpreter that supports the fused
step (the Llama engine), the gather and the argmax run inside the megakernel
and a step is one barrier reset plus one launch. With `sampling`, the token is
drawn from the logits (`ops.sample_tokens`) instead of their argmax.

`ParallelGenerator` decodes several continuations of one prompt at once: the
prompt's K/V rows are kept once and shared (`ops.shared_prefix_attention`), in
bf16 or in 8 bits (`ops.KVCacheInt8`). Any continuation can be handed back to
the model's cache, to go on with the megakernel at batch 1.
"""

from dataclasses import dataclass

import torch
import torch.distributed as dist
from torch import Tensor

from megakernels import ops
from megakernels.mk import MK_Interpreter
from megakernels.model_types import BatchState
from megakernels.scheduler import Schedule


@dataclass
class SamplingParams:
    """How tokens are drawn from the logits (see `ops.sample_tokens`). `generator`
    is the torch generator of the random numbers, on the logits' device; None
    uses torch's default one; seeding it anew takes effect at the next token.
    temperature 0 takes the largest logit. With several
    tensor-parallel ranks the first one's generator serves all; the other
    settings must be the same on every rank, and a new seed waits for the next
    block of numbers."""

    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    generator: torch.Generator | None = None


class _Sampler:
    """Draws tokens with the random numbers of a generator, which are made for many steps at once.

    globs: the globals of a tensor-parallel model. All its ranks must draw the same token, so they use the numbers of
    the first rank's generator, exchanged on the host once per STEPS steps; all ranks take the same steps."""

    STEPS = 256

    def __init__(self, params: SamplingParams, rows: int, globs=None):
        self.params = params
        self.rows = rows
        self.globs = globs
        self.step = self.STEPS

    def _place(self, device):
        """Where the generator stands: numbers left over are dropped when it was seeded or used since. Several ranks,
        which must make new numbers at the same step, keep to the steps."""
        g = self.params.generator
        if device.type != "cuda" or getattr(self.globs, "tp_world", 1) > 1:
            return None
        if g is None:
            g = torch.cuda.default_generators[torch.cuda.current_device() if device.index is None else device.index]
        return g.initial_seed(), g.get_offset()

    def draw(self, device) -> Tensor:
        """The next step's uniforms `[rows]`."""
        device = torch.device(device)
        if self.step == self.STEPS or self._place(device) != self.place:
            self.uniforms = torch.rand((self.STEPS, self.rows), generator=self.params.generator, device=device)
            if getattr(self.globs, "tp_world", 1) > 1:
                group = self.globs.tp_group
                numbers = [self.uniforms.cpu()]
                dist.broadcast_object_list(numbers, src=dist.get_global_rank(group, 0) if group else 0, group=group)
                self.uniforms.copy_(numbers[0])
            self.step = 0
            self.place = self._place(device)
        self.step += 1
        return self.uniforms[self.step - 1]

    def __call__(self, logits: Tensor, out: Tensor | None = None) -> Tensor:
        p = self.params
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("sampling cannot be captured: a replay would use the same random numbers again")
        return ops.sample_tokens(logits, self.draw(logits.device), temperature=p.temperature, top_k=p.top_k,
                                 top_p=p.top_p, min_p=p.min_p, out=out)


class Generator:
    def generate(self, output_tokens: Tensor, prompt_len: int, ntok: int,
                 ntok_already_generated: int = 1):
        raise NotImplementedError

    def generate_with_eos(self, output_tokens: Tensor, prompt_len: int, ntok: int,
                          eos_token_check_interval: int, eos_token_ids: list[int]):
        """Generate in chunks, checking for EOS between chunks. Returns (pos of
        the first eos token, tokens generated)."""
        assert output_tokens.shape[0] == 1, "batch size must be 1"
        for done in range(1, ntok, eos_token_check_interval):
            chunk = min(eos_token_check_interval, ntok - done)
            self.generate(output_tokens, prompt_len=prompt_len, ntok=chunk,
                          ntok_already_generated=done)
            for j, token in enumerate(output_tokens[0, done : done + chunk].cpu()):
                if token in eos_token_ids:
                    return done + j, done + chunk - 1
        return ntok, ntok - 1


class MK_Generator(Generator):
    def __init__(self, model, interpreter: MK_Interpreter, schedule: Schedule,
                 barrier_fill_val: int = 0, skip_mk: bool = False, skip_rest: bool = False,
                 sampling: SamplingParams | None = None):
        self.model = model
        self.interpreter = interpreter
        self.schedule = schedule
        self.barrier_fill_val = barrier_fill_val
        self.skip_mk = skip_mk
        self.skip_rest = skip_rest
        self.sampler = _Sampler(sampling, 1, schedule.globs) if sampling is not None else None
        self.fill()

    def _fused_step(self) -> bool:
        if self.skip_mk or self.skip_rest or not getattr(self.interpreter, "supports_fused_step", False):
            return False
        if getattr(self.schedule.globs, "lm_head_instructions", 0) < 1:
            return False
        if not hasattr(self, "_tokens"):
            # two output tokens in turn, and the argmax that a sampled step does not use
            self._tokens = torch.zeros(3, 1, dtype=torch.int64, device=self.schedule.globs.hidden_states.device)
            self._flip = 0
        return True

    def fill(self):
        self.schedule.globs.barriers.fill_(self.barrier_fill_val)

    def replace_with_noops(self):
        self.schedule.globs.instructions.zero_()

    def run(self, input_ids: Tensor, pos_id: int) -> Tensor:
        globs = self.schedule.globs
        if self._fused_step():
            # embedding gather and argmax inside the megakernel; the output
            # token alternates between two buffers so that a step may read the
            # previous step's token while writing its own
            self.fill()
            globs.pos_id = pos_id
            out = self._tokens[self._flip]
            self._flip ^= 1
            ids = input_ids.reshape(-1)[:1]
            if ids.dtype != torch.int64:
                ids = ids.to(torch.int64)
            self.interpreter.interpret_step(globs, ids, self.model.model.embed_tokens.embed_tokens.weight,
                                            self._tokens[2] if self.sampler else out)
            if self.sampler:
                self.sampler(globs.logits.view(1, -1), out=out)
            return out[0]
        if not self.skip_rest:
            emb = self.model.model.embed_tokens(BatchState(input_ids=input_ids))
            globs.hidden_states[:] = emb.hidden_states.reshape(-1)
        self.fill()
        globs.pos_id = pos_id
        globs.logits.zero_()
        if not self.skip_mk:
            self.interpreter.interpret(globs)
        if self.skip_rest:
            return input_ids
        return self._pick(globs.logits)

    def _pick(self, logits: Tensor) -> Tensor:
        if self.sampler:
            return self.sampler(logits.view(1, -1))[0]
        return torch.argmax(logits, dim=-1)

    def prefill(self, prompt_ids: Tensor, start_pos: int = 0) -> Tensor:
        """Fill the KV cache with the prompt (the model's dense prefill, as
        the reference's model forward does before MK decoding) and return the
        first generated token (argmax of, or draw from, the last prompt token's
        logits)."""
        return self._pick(self.model.prefill(prompt_ids, start_pos))

    def generate(self, output_tokens: Tensor, prompt_len: int, ntok: int,
                 ntok_already_generated: int = 1):
        for i in range(ntok):
            src = ntok_already_generated + i - 1
            input_ids = output_tokens[:, src : src + 1]
            out = self.run(input_ids, pos_id=prompt_len + ntok_already_generated + i - 1)
            output_tokens[:, src + 1] = out.reshape(-1)


class ParallelGenerator(Generator):
    """Decodes `num_sequences` continuations of one prompt at once.

    The prompt's K/V rows stay in the model's cache (`kv_cache="bf16"`: nothing
    else may write them meanwhile) or are quantised once (`"int8"`); each sequence has a cache of its own, of the same
    kind, for up to `max_new_tokens` tokens. The projections are dense products,
    as in the model's prefill. model: a LlamaForCausalLM on a CUDA device."""

    def __init__(self, model, num_sequences: int, max_new_tokens: int, sampling: SamplingParams | None = None,
                 kv_cache: str = "bf16"):
        if not hasattr(model, "decode_rows"):
            raise ValueError(f"ParallelGenerator: {type(model).__name__} has no decode_rows")
        if model.device.type != "cuda":
            raise ValueError("ParallelGenerator: the model must be on a CUDA device")
        if num_sequences < 1 or max_new_tokens < 1:
            raise ValueError("ParallelGenerator: num_sequences and max_new_tokens must be positive")
        if kv_cache not in ("bf16", "int8"):
            raise ValueError(f"kv_cache {kv_cache!r}: must be 'bf16' or 'int8'")
        c = model.config
        self.model = model
        self.num_sequences = num_sequences
        self.max_new_tokens = max_new_tokens
        self.sampler = _Sampler(sampling or SamplingParams(), num_sequences)
        self.int8 = kv_cache == "int8"
        self.prompt_len = 0
        self.new_tokens = 0  # tokens in the sequences' own caches
        self.logits: Tensor | None = None  # of the last step, [num_sequences, vocab]
        shape = (c.num_hidden_layers * num_sequences, max_new_tokens, c.num_key_value_heads, c.head_dim)
        if self.int8:
            own = ops.KVCacheInt8.empty(*shape, device=model.device)
            self.own = [ops.KVCacheInt8(*(t.unflatten(0, (c.num_hidden_layers, num_sequences))[l]
                                          for t in own._tensors())) for l in range(c.num_hidden_layers)]
        else:
            k, v = (torch.zeros(shape, dtype=torch.bfloat16, device=model.device)
                    .unflatten(0, (c.num_hidden_layers, num_sequences)) for _ in range(2))
            self.own = list(zip(k, v))
        self.prefix: list = []

    def prefill(self, prompt_ids: Tensor) -> Tensor:
        """Run the prompt through the model, keep its K/V rows as the shared
        prefix, and return the first token of every sequence (`[num_sequences]`
        int64). Starts over: earlier continuations are dropped."""
        logits = self.model.prefill(prompt_ids, 0)
        n = self.prompt_len = prompt_ids.numel()
        self.new_tokens = 0
        k, v = (t[:, 0, :n] for t in self.model.stacked_kv_cache)  # [L, n, Hkv, D]
        if self.int8:
            prefix = ops.KVCacheInt8.empty(*k.shape, device=k.device)
            ops.kv_cache_write(prefix, k, v, 0)
            self.prefix = [prefix.sequence(l) for l in range(k.shape[0])]
        else:
            self.prefix = list(zip(k, v))
        return self.sampler(logits.view(1, -1).expand(self.num_sequences, -1))

    def run(self, input_ids: Tensor) -> Tensor:
        """One step: the sequences' last tokens `[num_sequences]` in, their next
        ones out. `logits` keeps what they were drawn from."""
        if not self.prefix:
            raise ValueError("ParallelGenerator.run: prefill first")
        if self.new_tokens == self.max_new_tokens:
            raise ValueError(f"ParallelGenerator.run: the caches hold {self.max_new_tokens} new tokens")
        ids = input_ids.reshape(-1)
        if ids.numel() != self.num_sequences:
            raise ValueError(f"input_ids: {ids.numel()} tokens, expected {self.num_sequences}")
        at = self.new_tokens
        if self.prompt_len + at >= self.model.max_len():
            raise ValueError("ParallelGenerator.run: beyond the model's positions")
        lens = torch.full((self.num_sequences,), at + 1, dtype=torch.int32, device=self.model.device)
        pos = torch.full((self.num_sequences,), self.prompt_len + at, dtype=torch.int64, device=self.model.device)

        def attend(l, q, k, v):
            own = self.own[l]
            if self.int8:
                ops.kv_cache_write(own, k.unsqueeze(1), v.unsqueeze(1), at)
            else:
                own[0][:, at] = k
                own[1][:, at] = v
            return ops.shared_prefix_attention(q, self.prefix[l], own, lens, max_own_len=at + 1)

        self.logits = self.model.decode_rows(ids, pos, attend)
        self.new_tokens = at + 1
        return self.sampler(self.logits)

    def generate(self, output_tokens: Tensor, prompt_len: int, ntok: int, ntok_already_generated: int = 1):
        """Append `ntok` tokens per sequence to `output_tokens`
        `[num_sequences, ...]`, whose column ntok_already_generated - 1 holds the
        last ones (as `prefill` returned them, the first time)."""
        if prompt_len != self.prompt_len or ntok_already_generated != self.new_tokens + 1:
            raise ValueError(f"prompt_len {prompt_len} / ntok_already_generated {ntok_already_generated}: the caches "
                             f"hold a prompt of {self.prompt_len} and {self.new_tokens} new tokens")
        for i in range(ntok):
            src = ntok_already_generated + i - 1
            output_tokens[:, src + 1] = self.run(output_tokens[:, src])
        self.check()

    def check(self):
        """Wait for the steps so far; RuntimeError if a wait inside their attention ran out. Logits, tokens and cached
        rows since then are worthless. `generate` ends and `hand_over` begins with it; callers of `run` call it themselves."""
        if ops.attention_status(self.model.device):
            raise RuntimeError("ParallelGenerator: a wait inside the attention ran out; the tokens since the last check "
                               "are not valid")

    def hand_over(self, index: int) -> int:
        """Copy the rows of sequence `index` behind the prompt in the model's
        cache, so that `MK_Generator` goes on with it; returns the next position
        (prompt and new tokens)."""
        if not 0 <= index < self.num_sequences:
            raise ValueError(f"sequence {index} of {self.num_sequences}")
        self.check()
        n, end = self.new_tokens, self.prompt_len + self.new_tokens
        k_cache, v_cache = self.model.stacked_kv_cache
        for l, own in enumerate(self.own):
            k, v = k_cache[l, :1, self.prompt_len : end], v_cache[l, :1, self.prompt_len : end]
            if self.int8:
                ops.kv_cache_read(own.sequence(index), 0, n, out=(k, v))
            else:
                k.copy_(own[0][index : index + 1, :n])
                v.copy_(own[1][index : index + 1, :n])
        return end
