"""Operators for several sampled continuations of one prompt, on the GPU:

  KVCacheInt8, kv_cache_write, kv_cache_read
      a KV cache in 8 bits, quantised row by row as it is written
  shared_prefix_attention
      decode attention of a batch whose sequences share a prefix
  sample_tokens
      temperature, top-k, top-p and min-p sampling from given uniforms

Each call is asynchronous on the current stream of its tensors' device, which
need not be the current device. Nothing is kept between calls; outputs and
workspaces come from torch's allocator unless an output is given, so a call can
be captured into a CUDA graph. Tensors used on a stream other than the one that
they were made on need torch's usual `record_stream`.

Errors: a bad shape, dtype, stride or setting raises ValueError before
anything is launched, and so does an output or cache in whose memory another
argument lies (only results of `shared_prefix_attention` may replace q, K or
V); a CUDA failure raises RuntimeError. There is no CPU path:
CPU tensors raise ValueError. No operator has derivatives: tensors that require
grad raise ValueError while grad mode is on, dual tensors of forward-mode
differentiation always.
"""

import ctypes
import threading
from dataclasses import dataclass

import torch
from torch import Tensor

from megakernels import ek

MAX_VOCAB = 360448  # of sample_tokens

_native_module = None
_lock = threading.Lock()


def _native():
    """The compiled binding `_ekops`, connected to the loaded libek.so."""
    global _native_module
    if _native_module is None:
        with _lock:
            if _native_module is None:
                lib = ek.load_library()
                module = ek.load_extension("_ekops")
                module.bind({name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value
                             for name in ("ek_last_error", "ek_kv_write", "ek_kv_read",
                                          "ek_prefix_attention_workspace", "ek_prefix_attention", "ek_sample")})
                _native_module = module
    return _native_module


@dataclass
class KVCacheInt8:
    """K and V rows in 8 bits: int8 codes `[batch, rows, kv_heads, head_dim]`
    and one bf16 scale per (row, head), `[batch, rows, kv_heads]`; a value is
    code * scale. The tensors may be views (a layer, a range of rows)."""

    k_codes: Tensor
    k_scales: Tensor
    v_codes: Tensor
    v_scales: Tensor

    def __post_init__(self):
        _native().check_cache(self._tensors())

    def _tensors(self):
        return self.k_codes, self.k_scales, self.v_codes, self.v_scales

    @classmethod
    def empty(cls, batch: int, rows: int, kv_heads: int, head_dim: int, device="cuda") -> "KVCacheInt8":
        """A cache of zeros."""

        def codes():
            return torch.zeros(batch, rows, kv_heads, head_dim, dtype=torch.int8, device=device)

        def scales():
            return torch.zeros(batch, rows, kv_heads, dtype=torch.bfloat16, device=device)

        return cls(codes(), scales(), codes(), scales())

    @property
    def batch(self) -> int:
        return self.k_codes.shape[0]

    @property
    def rows(self) -> int:
        return self.k_codes.shape[1]

    def narrow(self, start: int, length: int) -> "KVCacheInt8":
        """A view of rows start .. start + length - 1 of every sequence."""
        return KVCacheInt8(*(t.narrow(1, start, length) for t in self._tensors()))

    def sequence(self, index: int) -> "KVCacheInt8":
        """A view of one sequence (batch 1)."""
        return KVCacheInt8(*(t.narrow(0, index, 1) for t in self._tensors()))


def _tensors_of(store, name: str) -> tuple:
    if isinstance(store, KVCacheInt8):
        return store._tensors()
    if isinstance(store, (tuple, list)) and len(store) == 2:
        return tuple(store)
    raise ValueError(f"{name}: expected KVCacheInt8 or a (k, v) pair, got {type(store).__name__}")


def _cache_tensors(cache) -> tuple:
    if not isinstance(cache, KVCacheInt8):
        raise ValueError(f"cache: expected KVCacheInt8, got {type(cache).__name__}")
    return cache._tensors()


def kv_cache_write(cache: KVCacheInt8, k: Tensor, v: Tensor, start: int | Tensor) -> None:
    """Quantise bf16 rows `k`, `v` `[batch, n, kv_heads, head_dim]` into the
    cache: row i of sequence b becomes cache row start[b] + i.

    start: one position for all sequences, or an int32 tensor `[batch]` on the
    device. An integer start must keep all rows inside the cache; with a tensor,
    rows that fall outside it are not written.

    Per (row, head): scale = max|x| / 127 rounded up to bf16 (at least 2^-126),
    code = x / scale rounded half away from zero, so a value is off by at most
    half a scale. A head holding a NaN or an infinity reads back as NaN; the
    largest finite bf16 value reads back as infinity (127 scales round to it)."""
    _native().kv_write(_cache_tensors(cache), k, v, start)


def kv_cache_read(cache: KVCacheInt8, start: int | Tensor, length: int,
                  out: tuple[Tensor, Tensor] | None = None) -> tuple[Tensor, Tensor]:
    """Rows start[b] .. start[b] + length - 1 of every sequence in bf16, as
    (k, v) of `[batch, length, kv_heads, head_dim]`, into `out` if given (two
    bf16 tensors, which may be views into the model's cache). `start` as in
    `kv_cache_write`; with a tensor, rows outside the cache read as zeros."""
    return _native().kv_read(_cache_tensors(cache), start, length, out)


def shared_prefix_attention(q: Tensor, prefix, own, own_lens: Tensor, *, scale: float | None = None,
                            max_own_len: int | None = None, out: Tensor | None = None,
                            return_lse: bool = False):
    """Decode attention of `batch` sequences, one query token each, over a
    prefix that all of them share followed by the rows of their own:

        out[b] = softmax(scale * q[b] [Kp; Ko[b, :own_lens[b]]]^T) [Vp; Vo[b, :own_lens[b]]]

    q         bf16 `[batch, q_heads, head_dim]`, head_dim 64 or 128; query head
              h reads KV head h // (q_heads // kv_heads)
    prefix    (k, v), each bf16 `[prefix_len, kv_heads, head_dim]`, or a
              KVCacheInt8 of batch 1; its rows are read once for all sequences
    own       (k, v), each bf16 `[batch, rows, kv_heads, head_dim]`, or a
              KVCacheInt8 of the batch (of the same kind as the prefix)
    own_lens  int32 `[batch]` on the device, clamped to [0, max_own_len]
    max_own_len  bound of own_lens that the host knows (default: all rows); a
              tight one saves empty work
    scale     default 1 / sqrt(head_dim)

    Returns bf16 `[batch, q_heads, head_dim]` (`out` if given), with
    `return_lse` also the natural log of the softmax sum, f32 `[batch, q_heads]`.
    A row without any key gives zeros and -inf. What lies behind the first
    own_lens[b] rows has no effect, NaN included. Caches may repeat heads or
    sequences (expand), not rows. Scores, softmax and sums are fp32; the probabilities are rounded
    to bf16 for the product with V."""
    return _native().attention(q, _tensors_of(prefix, "prefix"), _tensors_of(own, "own"), own_lens, scale,
                               max_own_len, out, return_lse)


def attention_status(device=None, clear: bool = True) -> int:
    """Synchronise; 1 if a wait inside a `shared_prefix_attention` kernel ran
    out on `device` since the last clear (the rows concerned are NaN), else 0."""
    out = ctypes.c_int32()
    index = torch.device("cuda" if device is None else device).index
    index = torch.cuda.current_device() if index is None else index
    ek.check(ek.load_library().ek_prefix_attention_status(index, ctypes.byref(out), int(clear)),
             "ek_prefix_attention_status")
    return out.value


def sample_tokens(logits: Tensor, uniforms: Tensor, *, temperature: float | Tensor = 1.0, top_k: int | Tensor = 0,
                  top_p: float | Tensor = 1.0, min_p: float | Tensor = 0.0, out: Tensor | None = None) -> Tensor:
    """One token per row of `logits` (bf16 or f32 `[batch, vocab]`), int64
    `[batch]`, drawn with the random numbers `uniforms` (f32 `[batch]`, in
    [0, 1)). Each setting is one number or a tensor `[batch]` on the device
    (int32 for top_k, f32 otherwise).

    With w_i = exp((l_i - max l) / temperature), and tokens ordered by falling
    logit, then rising index:
      top_k   the first top_k tokens stay (0: all)
      top_p   of those, the tokens stay before which less than top_p of their
              weight lies (1: all; the first always stays)
      min_p   of those, the tokens with w_i >= min_p stay (0: all)
    The result is the first token, by index, whose running weight over the
    tokens that stayed exceeds uniform * (their weight). temperature 0 gives the
    largest logit (the first one on ties, as torch.argmax).

    Weights are summed in fixed point, so the same inputs give the same token in
    every launch. NaN logits count as -inf (never drawn); several logits of
    +inf share the weight; a row without any logit above -inf gives token 0.
    Uniforms outside [0, 1) count as the nearest value inside. Settings per row
    are not checked: temperatures below 0 and NaN count as 0, +inf gives all
    logits above -inf the weight 1; other settings outside their range count as
    the nearest value inside, NaN as no filter."""
    return _native().sample(logits, uniforms, temperature, top_k, top_p, min_p, out, MAX_VOCAB)
