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
anything is launched; a CUDA failure raises RuntimeError. There is no CPU path:
CPU tensors raise ValueError. No operator has a backward pass: inputs that
require grad raise ValueError while grad mode is on.
"""

import ctypes
import math
from dataclasses import dataclass

import torch
from torch import Tensor

from megakernels import ek

_BF16 = torch.bfloat16
MAX_VOCAB = 360448  # of sample_tokens


def _need(t, name: str, dtype, ndim: int | None = None, like: Tensor | None = None) -> Tensor:
    if not isinstance(t, Tensor):
        raise ValueError(f"{name}: expected a tensor, got {type(t).__name__}")
    if t.dtype not in (dtype if isinstance(dtype, tuple) else (dtype,)):
        raise ValueError(f"{name}: dtype {t.dtype}, expected {dtype}")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{name}: {t.dim()}-D, expected {ndim}-D")
    if not t.is_cuda:
        raise ValueError(f"{name}: must be a CUDA tensor")
    if like is not None and t.device != like.device:
        raise ValueError(f"{name}: on {t.device}, expected {like.device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: requires grad, but this operator has no backward pass (use torch.no_grad)")
    return t


def _rows16(t: Tensor, name: str) -> Tensor:
    """The last dimension contiguous, everything else on 16-byte steps."""
    size = t.element_size()
    if t.numel():
        if t.stride(-1) != 1:
            raise ValueError(f"{name}: the last dimension must be contiguous")
        if t.data_ptr() % 16 or any(s * size % 16 for s, n in zip(t.stride()[:-1], t.shape) if n > 1):
            raise ValueError(f"{name}: rows must start on 16-byte boundaries")
    return t


def _no_overlap(t: Tensor, name: str) -> Tensor:
    """Refuse outputs whose elements share memory (an expanded dimension)."""
    span = 1
    for s, n in sorted((abs(s), n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if s < span:
            raise ValueError(f"{name}: elements overlap in memory")
        span = s * n
    return t


def _stream(device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _strides(t: Tensor, unit: int):
    """Strides of the leading dimensions; those of size one do not matter and
    are passed as multiples of `unit`."""
    return [s if n > 1 else 0 for s, n in zip(t.stride(), t.shape)][:unit]


def _kv_tensor(data: Tensor, scales: Tensor | None = None) -> ek.EkKvTensor:
    """Descriptor of [batch, row, head, D] rows; a 3-D tensor has no batch."""
    r = ek.EkKvTensor()
    r.data = data.data_ptr()
    strides = _strides(data, data.dim() - 1)
    r.stride_batch, r.stride_row, r.stride_head = [0] * (3 - len(strides)) + strides
    if scales is not None:
        r.scales = scales.data_ptr()
        strides = _strides(scales, scales.dim())
        r.scale_stride_batch, r.scale_stride_row, r.scale_stride_head = [0] * (3 - len(strides)) + strides
    return r


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
        for kind in "kv":
            codes = _need(getattr(self, f"{kind}_codes"), f"{kind}_codes", torch.int8, 4)
            scales = _need(getattr(self, f"{kind}_scales"), f"{kind}_scales", _BF16, 3, codes)
            _rows16(codes, f"{kind}_codes")
            if codes.shape != self.k_codes.shape or scales.shape != codes.shape[:3]:
                raise ValueError(f"{kind}_codes {tuple(codes.shape)} / {kind}_scales {tuple(scales.shape)}: shapes "
                                 f"do not match k_codes {tuple(self.k_codes.shape)}")
            if codes.device != self.k_codes.device:
                raise ValueError("KVCacheInt8: tensors on several devices")
        _check_head_dim(self.k_codes.shape[3])

    @classmethod
    def empty(cls, batch: int, rows: int, kv_heads: int, head_dim: int, device="cuda") -> "KVCacheInt8":
        """A cache of zeros."""

        def codes():
            return torch.zeros(batch, rows, kv_heads, head_dim, dtype=torch.int8, device=device)

        def scales():
            return torch.zeros(batch, rows, kv_heads, dtype=_BF16, device=device)

        return cls(codes(), scales(), codes(), scales())

    @property
    def batch(self) -> int:
        return self.k_codes.shape[0]

    @property
    def rows(self) -> int:
        return self.k_codes.shape[1]

    def narrow(self, start: int, length: int) -> "KVCacheInt8":
        """A view of rows start .. start + length - 1 of every sequence."""
        return KVCacheInt8(*(t.narrow(1, start, length) for t in
                             (self.k_codes, self.k_scales, self.v_codes, self.v_scales)))

    def sequence(self, index: int) -> "KVCacheInt8":
        """A view of one sequence (batch 1)."""
        return KVCacheInt8(*(t.narrow(0, index, 1) for t in
                             (self.k_codes, self.k_scales, self.v_codes, self.v_scales)))


def _check_head_dim(d: int):
    if d not in (64, 128):
        raise ValueError(f"head_dim {d} (supported: 64, 128)")


def _copy_args(cache: KVCacheInt8, k: Tensor, v: Tensor, start) -> ek.EkKvCopyArgs:
    if not isinstance(cache, KVCacheInt8):
        raise ValueError(f"cache: expected KVCacheInt8, got {type(cache).__name__}")
    codes = cache.k_codes
    _rows16(_need(k, "k", _BF16, 4, codes), "k")
    _rows16(_need(v, "v", _BF16, 4, codes), "v")
    if k.shape != v.shape or k.shape[0] != codes.shape[0] or k.shape[2:] != codes.shape[2:]:
        raise ValueError(f"k {tuple(k.shape)} / v {tuple(v.shape)}: expected [batch, rows, kv_heads, head_dim] as in "
                         f"the cache {tuple(codes.shape)}")
    a = ek.EkKvCopyArgs()
    a.k_values, a.v_values = _kv_tensor(k), _kv_tensor(v)
    a.k_cache = _kv_tensor(codes, cache.k_scales)
    a.v_cache = _kv_tensor(cache.v_codes, cache.v_scales)
    a.batch, a.length, a.kv_heads, a.head_dim = k.shape
    a.capacity = codes.shape[1]
    if isinstance(start, Tensor):
        _need(start, "start", torch.int32, 1, codes)
        if start.shape[0] != a.batch or not start.is_contiguous():
            raise ValueError(f"start: expected a contiguous int32 tensor of {a.batch} positions")
        a.start = start.data_ptr()
    else:
        start = int(start)
        if start < 0 or start + a.length > a.capacity:
            raise ValueError(f"rows {start} .. {start + a.length - 1} outside the cache of {a.capacity} rows")
        a.start_all = start
    a.device = codes.device.index
    return a


def kv_cache_write(cache: KVCacheInt8, k: Tensor, v: Tensor, start: int | Tensor) -> None:
    """Quantise bf16 rows `k`, `v` `[batch, n, kv_heads, head_dim]` into the
    cache: row i of sequence b becomes cache row start[b] + i.

    start: one position for all sequences, or an int32 tensor `[batch]` on the
    device. An integer start must keep all rows inside the cache; with a tensor,
    rows that fall outside it are not written.

    Per (row, head): scale = max|x| / 127 rounded up to bf16 (at least 2^-126),
    code = x / scale rounded half away from zero, so a value is off by at most
    half a scale. A head holding a NaN or an infinity reads back as NaN."""
    a = _copy_args(cache, k, v, start)
    for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
        _no_overlap(getattr(cache, name), name)
    ek.check(ek.load_library().ek_kv_write(ctypes.byref(a), _stream(k.device)), "ek_kv_write")


def kv_cache_read(cache: KVCacheInt8, start: int | Tensor, length: int,
                  out: tuple[Tensor, Tensor] | None = None) -> tuple[Tensor, Tensor]:
    """Rows start[b] .. start[b] + length - 1 of every sequence in bf16, as
    (k, v) of `[batch, length, kv_heads, head_dim]`, into `out` if given (two
    bf16 tensors, which may be views into the model's cache). `start` as in
    `kv_cache_write`; with a tensor, rows outside the cache read as zeros."""
    if not isinstance(cache, KVCacheInt8):
        raise ValueError(f"cache: expected KVCacheInt8, got {type(cache).__name__}")
    if length < 0:
        raise ValueError(f"length {length}")
    b, _, h, d = cache.k_codes.shape
    if out is None:
        out = tuple(torch.empty(b, length, h, d, dtype=_BF16, device=cache.k_codes.device) for _ in range(2))
    k, v = out
    a = _copy_args(cache, k, v, start)
    if a.length != length:
        raise ValueError(f"out: {a.length} rows, expected {length}")
    _no_overlap(k, "out[0]"), _no_overlap(v, "out[1]")
    ek.check(ek.load_library().ek_kv_read(ctypes.byref(a), _stream(k.device)), "ek_kv_read")
    return k, v


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
    A row without any key gives zeros and -inf. Only the first own_lens[b] rows
    are read. Scores, softmax and sums are fp32; the probabilities are rounded
    to bf16 for the product with V."""
    _rows16(_need(q, "q", _BF16, 3), "q")
    batch, q_heads, head_dim = q.shape
    _check_head_dim(head_dim)
    int8 = isinstance(prefix, KVCacheInt8)
    if int8 != isinstance(own, KVCacheInt8):
        raise ValueError("prefix and own must both be KVCacheInt8 or both (k, v) pairs")
    a = ek.EkPrefixAttnArgs()
    if int8:
        if prefix.batch != 1:
            raise ValueError(f"prefix: batch {prefix.batch}, expected 1")
        for t, name in ((prefix.k_codes, "prefix"), (own.k_codes, "own")):
            if t.device != q.device:
                raise ValueError(f"{name}: on {t.device}, expected {q.device}")
        pk, ok = prefix.k_codes[0], own.k_codes
        a.prefix_k, a.prefix_v = (_kv_tensor(prefix.k_codes, prefix.k_scales),
                                  _kv_tensor(prefix.v_codes, prefix.v_scales))
        a.own_k, a.own_v = _kv_tensor(own.k_codes, own.k_scales), _kv_tensor(own.v_codes, own.v_scales)
    else:
        pk, pv = prefix
        ok, ov = own
        for t, name, ndim in ((pk, "prefix k", 3), (pv, "prefix v", 3), (ok, "own k", 4), (ov, "own v", 4)):
            _rows16(_need(t, name, _BF16, ndim, q), name)
        if pk.shape != pv.shape or ok.shape != ov.shape:
            raise ValueError("k and v must have the same shape")
        a.prefix_k, a.prefix_v = _kv_tensor(pk), _kv_tensor(pv)
        a.own_k, a.own_v = _kv_tensor(ok), _kv_tensor(ov)
    kv_heads = ok.shape[2]
    if ok.shape[0] != batch or pk.shape[1:] != ok.shape[2:] or ok.shape[3] != head_dim:
        raise ValueError(f"q {tuple(q.shape)}, prefix {tuple(pk.shape)}, own {tuple(ok.shape)}: inconsistent")
    if kv_heads < 1 or q_heads < 1 or q_heads % kv_heads:
        raise ValueError(f"q_heads {q_heads} must be a positive multiple of kv_heads {kv_heads}")
    _need(own_lens, "own_lens", torch.int32, 1, q)
    if own_lens.shape[0] != batch or not own_lens.is_contiguous():
        raise ValueError(f"own_lens: expected a contiguous int32 tensor of {batch} lengths")
    if max_own_len is None:
        max_own_len = ok.shape[1]
    if not 0 <= max_own_len <= ok.shape[1]:
        raise ValueError(f"max_own_len {max_own_len} outside the {ok.shape[1]} own rows")
    scale = 1.0 / math.sqrt(head_dim) if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale {scale}")
    if out is None:
        out = torch.empty(batch, q_heads, head_dim, dtype=_BF16, device=q.device)
    else:
        _no_overlap(_rows16(_need(out, "out", _BF16, 3, q), "out"), "out")
        if out.shape != q.shape:
            raise ValueError(f"out: {tuple(out.shape)}, expected {tuple(q.shape)}")
    lse = torch.empty(batch, q_heads, dtype=torch.float32, device=q.device) if return_lse else None
    a.q, a.own_lens, a.out = q.data_ptr(), own_lens.data_ptr(), out.data_ptr()
    a.q_stride_batch, a.q_stride_head = _strides(q, 2)
    a.out_stride_batch, a.out_stride_head = _strides(out, 2)
    a.lse = lse.data_ptr() if return_lse else None
    a.batch, a.q_heads, a.kv_heads, a.head_dim = batch, q_heads, kv_heads, head_dim
    a.prefix_len, a.own_capacity, a.max_own_len = pk.shape[0], ok.shape[1], max_own_len
    a.scale = scale
    a.device = q.device.index
    lib = ek.load_library()
    size = lib.ek_prefix_attention_workspace(ctypes.byref(a))
    if size < 0:
        ek.check(1, "ek_prefix_attention_workspace")
    workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), size
    ek.check(lib.ek_prefix_attention(ctypes.byref(a), _stream(q.device)), "ek_prefix_attention")
    return (out, lse) if return_lse else out


def attention_status(device=None, clear: bool = True) -> int:
    """Synchronise; 1 if a wait inside a `shared_prefix_attention` kernel ran
    out on `device` since the last clear (the rows concerned are NaN), else 0."""
    out = ctypes.c_int32()
    index = torch.device("cuda" if device is None else device).index
    index = torch.cuda.current_device() if index is None else index
    ek.check(ek.load_library().ek_prefix_attention_status(index, ctypes.byref(out), int(clear)),
             "ek_prefix_attention_status")
    return out.value


def _setting(value, name: str, dtype, logits: Tensor):
    """(device pointer or None, scalar) of a setting given as a number or as a
    tensor with one value per row."""
    if isinstance(value, Tensor):
        _need(value, name, dtype, 1, logits)
        if value.shape[0] != logits.shape[0] or not value.is_contiguous():
            raise ValueError(f"{name}: expected a contiguous tensor of {logits.shape[0]} values")
        return value.data_ptr(), 0
    return None, value


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
    Uniforms outside [0, 1) count as the nearest value inside."""
    _need(logits, "logits", (_BF16, torch.float32), 2)
    batch, vocab = logits.shape
    if not 1 <= vocab <= MAX_VOCAB:
        raise ValueError(f"logits: vocabulary {vocab} (1 .. {MAX_VOCAB})")
    if vocab > 1 and logits.stride(1) != 1:
        raise ValueError("logits: the last dimension must be contiguous")
    _need(uniforms, "uniforms", torch.float32, 1, logits)
    if uniforms.shape[0] != batch or not uniforms.is_contiguous():
        raise ValueError(f"uniforms: expected a contiguous f32 tensor of {batch} numbers")
    a = ek.EkSampleArgs()
    a.temperature, temperature = _setting(temperature, "temperature", torch.float32, logits)
    a.top_k, top_k = _setting(top_k, "top_k", torch.int32, logits)
    a.top_p, top_p = _setting(top_p, "top_p", torch.float32, logits)
    a.min_p, min_p = _setting(min_p, "min_p", torch.float32, logits)
    if not (temperature >= 0 and math.isfinite(temperature)):
        raise ValueError(f"temperature {temperature}: must be finite and not negative")
    if top_k < 0 or top_k != int(top_k):
        raise ValueError(f"top_k {top_k}: must be a whole number >= 0")
    if not 0 <= top_p <= 1:
        raise ValueError(f"top_p {top_p}: must lie in [0, 1]")
    if not 0 <= min_p <= 1:
        raise ValueError(f"min_p {min_p}: must lie in [0, 1]")
    a.temperature_all, a.top_p_all, a.min_p_all = temperature, top_p, min_p
    a.top_k_all = min(int(top_k), vocab)
    if out is None:
        out = torch.empty(batch, dtype=torch.int64, device=logits.device)
    else:
        _need(out, "out", torch.int64, 1, logits)
        if out.shape[0] != batch or not out.is_contiguous():
            raise ValueError(f"out: expected a contiguous int64 tensor of {batch} tokens")
    a.logits, a.uniforms, a.tokens = logits.data_ptr(), uniforms.data_ptr(), out.data_ptr()
    a.row_stride = logits.stride(0) if batch > 1 else 0
    a.logits_f32 = int(logits.dtype == torch.float32)
    a.batch, a.vocab, a.device = batch, vocab, logits.device.index
    ek.check(ek.load_library().ek_sample(ctypes.byref(a), _stream(logits.device)), "ek_sample")
    return out
