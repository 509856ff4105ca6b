"""Serving operators over the C ABI (include/aps_serve.h, aps_decode.h): a
paged key/value cache, attention over it, and the rules on the logits of the
next token; rotary positions of other layouts and scalings, linear layers with
weights in 4 bits, and log probabilities of tokens.

The reference has no counterpart: its generate_decode computes the whole
prefix again for every token (src/model.cu:163-204).
decoder.Model.generate_decode runs on these.

A decode step of a batch, on torch's current stream:

    plan = PagedBatch(q_lens, kv_lens, pages, cache.page_size, device)
    q = kv_append_gpu(cache, k, v, plan.positions, plan.slots, cos, sin, q=q)
    out = attention_paged_gpu(q, cache, plan.q_offsets, plan.kv_lens, plan.page_table, plan.max_q_len,
                              plan.max_kv_len, q_heads=16, window=2047, sinks=4)

and around it, for a model with weights in 4 bits:

    w = quantise_q4_gpu(weight, group=128)
    y = linear_q4_gpu(x, w, bias)
    q, k = rope_gpu(q, k, plan.positions, freq, head_dim=128, layout="pairs", amplitude=amplitude)
    scores = token_logprobs_gpu(logits, tokens, top=5)

Calls launch kernels and read nothing back, so they can be captured into a
graph; index arrays are read on the device (PagedBatch checks its own on the
host).  Wrong shapes, types and layouts raise ValueError.
"""
from __future__ import annotations

import contextlib
import ctypes
import math
from typing import NamedTuple, Optional, Sequence, Tuple

import numpy as np
import torch

from . import capi
from .moe import _call, _require

MXFP4 = capi.KV_MXFP4
_CODE = {torch.float32: capi.DTYPE_F32, torch.bfloat16: capi.DTYPE_BF16}


def _p(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


# A decode step is a row of short launches, so what Python does around them
# counts: the stream's handle without an object for it, checks on plain numbers.
# A torch that lacks the short ways (one without a GPU backend has neither) gives
# both by its public calls.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _launch(fn, device: torch.device, *args) -> None:
    """fn(*args, the current stream of device), with device current."""
    index = device.index
    if _current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _call(rc)


def on_stream(stream, device: torch.device):
    """A context whose current stream of device is `stream`: a handle, as an
    int or a c_void_p (None or 0: the default stream)."""
    handle = (stream.value if isinstance(stream, ctypes.c_void_p) else stream) or 0
    if handle == _raw_stream(device.index):
        return contextlib.nullcontext()
    return torch.cuda.stream(torch.cuda.ExternalStream(handle, device) if handle
                             else torch.cuda.default_stream(device))


def _like(t: torch.Tensor) -> torch.Tensor:
    """An unset contiguous tensor of t's shape, type and device."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _dev(t: torch.Tensor, device: torch.device, dtype: torch.dtype, what: str) -> int:
    """The address of a contiguous tensor of that type on that device."""
    if t.dtype is not dtype or t.device != device or not t.is_contiguous():
        raise ValueError(f"{what}: expects a contiguous {dtype} tensor on {device}")
    return t.data_ptr()


class PagedKvCache:
    """One layer's cache: k and v [pages][kv_heads][page][head_dim], fp32 or
    bf16; or, given k_scale and v_scale, 4-bit codes [..][head_dim / 2] (uint8)
    with scale bytes [..][head_dim / 32] (uint8).  The tensors stay the
    caller's; allocate() makes them."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "pages", "kv_heads", "page_size", "head_dim", "dtype", "device",
                 "_desc", "_ref")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None):
        shape, dt, dev = k.shape, k.dtype, k.device
        if len(shape) != 4 or v.shape != shape or v.dtype is not dt or dev.type != "cuda" or v.device != dev or \
                not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError("paged cache: k and v [pages, kv_heads, page, head_dim] on a GPU")
        self.pages, self.kv_heads, self.page_size, self.head_dim = shape
        if k_scale is not None or v_scale is not None:
            _require(dt is torch.uint8 and k_scale is not None and v_scale is not None,
                     "paged cache: 4-bit codes are uint8 with k_scale and v_scale")
            self.head_dim *= 2
            self.dtype = MXFP4
            want = (*shape[:3], self.head_dim // 32)
            for s in (k_scale, v_scale):
                _require(s.shape == want and s.dtype is torch.uint8 and s.device == dev and s.is_contiguous(),
                         f"paged cache: scales {want}")
        else:
            _require(dt in _CODE, f"paged cache: dtype {dt}")
            self.dtype = _CODE[dt]
        self.k, self.v, self.k_scale, self.v_scale, self.device = k, v, k_scale, v_scale, dev
        self._desc = capi.KvCacheDesc(k.data_ptr(), v.data_ptr(), _p(k_scale), _p(v_scale), self.pages,
                                      self.page_size, self.kv_heads, self.head_dim, self.dtype)
        self._ref = ctypes.byref(self._desc)

    @staticmethod
    def allocate(pages: int, page_size: int, kv_heads: int, head_dim: int, dtype, device) -> "PagedKvCache":
        """dtype: torch.float32, torch.bfloat16 or "mxfp4" (4 bits)."""
        shape = (pages, kv_heads, page_size)
        if dtype in ("mxfp4", MXFP4):
            z = lambda n: torch.zeros((*shape, n), dtype=torch.uint8, device=device)  # noqa: E731
            return PagedKvCache(z(head_dim // 2), z(head_dim // 2), z(head_dim // 32), z(head_dim // 32))
        z = lambda: torch.zeros((*shape, head_dim), dtype=dtype, device=device)  # noqa: E731
        return PagedKvCache(z(), z())


class PagedBatch:
    """A batch's index arrays on the device, checked on the host: q_lens[b] new
    tokens of sequence b, kv_lens[b] cached positions with them, pages[b] its
    page ids.  positions and slots of the new tokens' rows, for the append;
    q_offsets, kv_lens, page_table and the two maxima, for the attention."""

    def __init__(self, q_lens: Sequence[int], kv_lens: Sequence[int], pages: Sequence[Sequence[int]], page_size: int,
                 device, num_pages: Optional[int] = None):
        q, kv = np.asarray(q_lens, np.int64).reshape(-1), np.asarray(kv_lens, np.int64).reshape(-1)
        _require(q.size == kv.size == len(pages), "paged batch: one length and page list a sequence")
        _require(page_size >= 1, "paged batch: page size")
        _require(bool(np.all(q >= 0)) and bool(np.all(kv >= q)) and bool(np.all(kv < 1 << 30)) and int(q.sum()) < 1 << 30,
                 "paged batch: 0 <= q_lens <= kv_lens")
        ids = [np.asarray(p, np.int64).reshape(-1) for p in pages]
        for n, p in zip(kv, ids):
            _require(p.size * page_size >= n, "paged batch: too few pages")
            _require(p.size == 0 or (p.min() >= 0 and p.max() < (num_pages if num_pages is not None else 1 << 31)),
                     "paged batch: page id")
        table = np.full((q.size, max([p.size for p in ids], default=0) or 1), -1, np.int32)
        for b, p in enumerate(ids):
            table[b, :p.size] = p
        seq = np.repeat(np.arange(q.size), q)
        pos = np.arange(seq.size) - np.repeat(np.cumsum(q) - q, q) + (kv - q)[seq]
        slots = table[seq, pos // page_size].astype(np.int64) * page_size + pos % page_size
        _require(np.unique(slots).size == slots.size, "paged batch: two new tokens share a slot")
        up = lambda a, t: torch.from_numpy(np.ascontiguousarray(a.astype(t))).to(device)  # noqa: E731
        self.rows, self.batch = int(q.sum()), int(q.size)
        self.max_q_len, self.max_kv_len = int(q.max(initial=0)), int(kv.max(initial=0))
        self.positions, self.slots = up(pos, np.int32), up(slots, np.int64)
        self.q_offsets = up(np.concatenate([[0], np.cumsum(q)]), np.int32)
        self.kv_lens, self.page_table = up(kv, np.int32), up(table, np.int32)


def _rows_of(t: torch.Tensor, width: int, what: str) -> int:
    """The row stride of a matrix whose rows are `width` neighbouring values."""
    shape = t.shape
    if len(shape) == 2 and shape[1] == width:
        row, col = t.stride()
        if col == 1 or width == 1:
            return row if shape[0] > 1 else width   # the stride of a single row says nothing
    raise ValueError(f"{what}: expects rows of {width} neighbouring values")


def kv_append_gpu(cache: PagedKvCache, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                  cos: torch.Tensor, sin: torch.Tensor, q: Optional[torch.Tensor] = None,
                  q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Writes k (rotated by positions) and v, [rows, kv_heads * head_dim] with
    any row stride, into the cache's slots; returns q [rows, q_heads *
    head_dim] rotated (into q_out; q itself rotates in place).  cos and sin:
    [positions, head_dim / 2] fp32 (rope_table).  slots int64, -1 for padding
    rows, otherwise distinct; positions int32."""
    what, dev, dim, dt = "kv_append", cache.device, cache.head_dim, k.dtype
    width, rows = cache.kv_heads * dim, k.shape[0]
    k_stride, v_stride = _rows_of(k, width, what), _rows_of(v, width, what)
    code = _CODE.get(dt)
    if code is None or v.dtype is not dt or v.shape[0] != rows or k.device != dev or v.device != dev:
        raise ValueError("kv_append: k and v of one fp32 or bf16 type on the cache's device")
    max_pos = cos.shape[0]
    if positions.numel() != rows or slots.numel() != rows or cos.shape != sin.shape or cos.dim() != 2 or \
            cos.shape[1] * 2 != dim:
        raise ValueError("kv_append shape")
    q_heads = q_stride = o_stride = 0
    qp = op = None
    if q is not None:
        q_width = q.shape[-1]
        q_stride = _rows_of(q, q_width, what)
        if q.shape[0] != rows or q_width % dim or q.dtype is not dt or q.device != dev:
            raise ValueError("kv_append: q [rows, q_heads * head_dim] of k's type")
        q_heads = q_width // dim
        if q_out is None:
            q_out, o_stride = _like(q), q_width
        elif q_out.shape != q.shape or q_out.dtype is not dt or q_out.device != dev:
            raise ValueError("kv_append: q_out of q's shape and type")
        else:
            o_stride = _rows_of(q_out, q_width, what)
        qp, op = q.data_ptr(), q_out.data_ptr()
    _launch(capi.lib().aps_kv_append, dev, cache._ref, k.data_ptr(), k_stride, v.data_ptr(), v_stride, qp, q_stride,
            op, o_stride, code, rows, q_heads, _dev(positions, dev, torch.int32, what),
            _dev(slots, dev, torch.int64, what), _dev(cos, dev, torch.float32, what),
            _dev(sin, dev, torch.float32, what), max_pos)
    return q_out if q is not None else None


def kv_gather_gpu(cache: PagedKvCache, slots: torch.Tensor, out_dtype: torch.dtype = torch.float32
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [rows, kv_heads * head_dim] of the slots (int64; zeros for one
    outside the cache), the values of the codes for a 4-bit cache."""
    _require(out_dtype in _CODE, f"kv_gather: dtype {out_dtype}")
    at, rows = _dev(slots, cache.device, torch.int64, "kv_gather"), slots.numel()
    k = torch.empty((rows, cache.kv_heads * cache.head_dim), dtype=out_dtype, device=cache.device)
    v = torch.empty_like(k)
    _launch(capi.lib().aps_kv_gather, cache.device, cache._ref, at, rows, k.data_ptr(), v.data_ptr(),
            _CODE[out_dtype])
    return k, v


def attention_paged_gpu(q: torch.Tensor, cache: PagedKvCache, q_offsets: torch.Tensor, kv_lens: torch.Tensor,
                        page_table: torch.Tensor, max_q_len: int, max_kv_len: int, q_heads: int, window: int,
                        sinks: int = 0, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                        workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Softmax attention of the batch's new tokens (rows of q) over the cached
    keys they see: the last `window` up to their own and the first `sinks`.
    scale: 1 / sqrt(head_dim) unless given.  The workspace is torch's, taken
    on the current stream, unless one is given (uint8).  Rows of a given `out`
    (not q) that no sequence names are left as they were, of a new one unset."""
    what, dev, dim = "attention_paged", cache.device, cache.head_dim
    width = q_heads * dim
    q_stride = _rows_of(q, width, what)
    dt = q.dtype
    code = _CODE.get(dt)
    if code is None or q.device != dev:
        raise ValueError("attention_paged: fp32 or bf16 queries on the cache's device")
    batch, rows, table = kv_lens.numel(), q.shape[0], page_table.shape
    if q_offsets.numel() != batch + 1 or len(table) != 2 or table[0] != batch:
        raise ValueError("attention_paged shape")
    if out is None:
        out = _like(q)
    elif out.shape != (rows, width) or out.dtype is not dt or out.device != dev or not out.is_contiguous():
        raise ValueError("attention_paged: out of q's shape and type, contiguous")
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    if window < 1 or sinks < 0:
        raise ValueError("attention_paged: window >= 1 and sinks >= 0")
    window, sinks = min(window, 0x7FFFFFFF), min(sinks, 0x7FFFFFFF)
    lib = capi.lib()
    need = lib.aps_attention_paged_workspace_size(cache._ref, rows, q_heads, batch, max_q_len, max_kv_len, window,
                                                  sinks)
    wp, wn = None, 0
    if need:
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        elif workspace.device != dev or not workspace.is_contiguous():
            raise ValueError("attention_paged: a contiguous workspace on the cache's device")
        wp, wn = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    _launch(lib.aps_attention_paged, dev, cache._ref, q.data_ptr(), q_stride, code, rows, q_heads,
            _dev(q_offsets, dev, torch.int32, what), _dev(kv_lens, dev, torch.int32, what),
            _dev(page_table, dev, torch.int32, what), table[1], batch, max_q_len, max_kv_len, window, sinks, scale,
            out.data_ptr(), wp, wn)
    return out


def logits_process_gpu(logits: torch.Tensor, history: Optional[torch.Tensor] = None,
                       history_lens: Optional[torch.Tensor] = None, prompt_lens: Optional[torch.Tensor] = None,
                       repetition: Optional[torch.Tensor] = None, frequency: Optional[torch.Tensor] = None,
                       presence: Optional[torch.Tensor] = None, bias_ids: Optional[torch.Tensor] = None,
                       bias_values: Optional[torch.Tensor] = None, bias_lens: Optional[torch.Tensor] = None,
                       mask: Optional[torch.Tensor] = None, mask_index: Optional[torch.Tensor] = None,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The logits [rows, vocab] after the rules (aps_logits_process): penalties
    by each row's history [rows, n] (int32, the first history_lens of it, the
    first prompt_lens of those the prompt), biases of the first bias_lens ids
    of bias_ids [rows, n], and a bit mask [masks, words] (int32 words, bit t %
    32 of word t / 32 allows token t; row r's is mask_index[r], or r).  A rule
    without its arrays is off.  out may be logits itself."""
    what = "logits_process"
    _require(logits.dim() == 2, "logits_process: logits [rows, vocab]")
    rows, vocab = logits.shape
    dev, dt = logits.device, logits.dtype
    code = _CODE.get(dt)
    if code is None or dev.type != "cuda":
        raise ValueError("logits_process: fp32 or bf16 logits on a GPU")
    stride = _rows_of(logits, vocab, what)
    if out is None:
        out = _like(logits)
    elif out.shape != logits.shape or out.dtype is not dt or out.device != dev:
        raise ValueError("logits_process: out of the logits' shape and type")
    rules = capi.LogitsRules()

    def each(t, dtype):  # one value a row
        if t.numel() != rows:
            raise ValueError("logits_process: one value a row")
        return _dev(t, dev, dtype, what)

    i32, f32 = torch.int32, torch.float32
    if history is not None:
        _require(history.dim() == 2 and history.shape[0] == rows and history_lens is not None,
                 "logits_process: a history [rows, n] and its history_lens")
        rules.history, rules.history_lens = _dev(history, dev, i32, what), each(history_lens, i32)
        rules.history_stride = history.shape[1]
        if prompt_lens is not None:
            rules.prompt_lens = each(prompt_lens, i32)
        if repetition is not None:
            rules.repetition = each(repetition, f32)
        if frequency is not None:
            rules.frequency = each(frequency, f32)
        if presence is not None:
            rules.presence = each(presence, f32)
    else:
        _require(repetition is frequency is presence is None, "logits_process: penalties need a history")
    if bias_ids is not None:
        _require(bias_ids.dim() == 2 and bias_ids.shape[0] == rows and bias_lens is not None and
                 bias_values is not None and bias_values.shape == bias_ids.shape,
                 "logits_process: biases are bias_ids and bias_values [rows, n] and bias_lens")
        rules.bias_ids, rules.bias_values = _dev(bias_ids, dev, i32, what), _dev(bias_values, dev, f32, what)
        rules.bias_lens, rules.bias_stride = each(bias_lens, i32), bias_ids.shape[1]
    if mask is not None:
        _require(mask.dim() == 2 and mask.shape[1] * 32 >= vocab and (mask_index is not None or mask.shape[0] >= rows),
                 "logits_process: mask [masks, words] with a word for every 32 logits")
        rules.mask = _dev(mask, dev, i32, what)
        rules.mask_rows, rules.mask_stride = mask.shape
        if mask_index is not None:
            rules.mask_index = each(mask_index, i32)
    _launch(capi.lib().aps_logits_process, dev, logits.data_ptr(), stride, code, rows, vocab, ctypes.byref(rules),
            out.data_ptr(), _rows_of(out, vocab, what))
    return out


# ---- rotary positions ---------------------------------------------------------

_LAYOUT = {"half": capi.ROPE_HALF, "pairs": capi.ROPE_PAIRS}


def rope_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                     trained: int = 4096, fast: float = 32.0, slow: float = 1.0,
                     divisors: Optional[Sequence[float]] = None) -> Tuple[np.ndarray, float]:
    """(angles per position [rotary_dim / 2] in 64 bits, amplitude) of the pairs
    theta^(-2 i / rotary_dim), for contexts `factor` times the trained length:
      "none"    as they are
      "linear"  all divided by factor: positions between the trained ones
      "base"    theta times factor^(rotary_dim / (rotary_dim - 2)): the fastest
                pair stays, the slowest is divided by factor
      "parts"   pairs that turn `fast` times or more in the trained length stay,
                those that turn `slow` times or less are divided by factor, in
                between by parts; amplitude 1 + 0.1 ln factor
      "divisors" each pair by its own"""
    _require(rotary_dim >= 2 and rotary_dim % 2 == 0, "rope_frequencies: an even rotary_dim")
    _require(theta > 0.0 and 0.0 < factor < math.inf, "rope_frequencies: theta and factor are positive")
    i = np.arange(rotary_dim // 2)
    if scaling == "base":
        _require(rotary_dim > 2, "rope_frequencies: a base needs two pairs")
        return (theta * factor ** (rotary_dim / (rotary_dim - 2))) ** (-2.0 * i / rotary_dim), 1.0
    freq = float(theta) ** (-2.0 * i / rotary_dim)
    if scaling == "linear":
        return freq / factor, 1.0
    if scaling == "parts":
        _require(fast > slow and trained >= 1, "rope_frequencies: fast > slow, a trained length")
        stay = np.clip((trained * freq / (2 * math.pi) - slow) / (fast - slow), 0.0, 1.0)
        return freq * (stay + (1 - stay) / factor), 1.0 + 0.1 * math.log(factor)
    if scaling == "divisors":
        by = np.asarray(divisors if divisors is not None else (), np.float64)
        _require(by.shape == freq.shape and bool(np.all(by > 0)), "rope_frequencies: a positive divisor for each pair")
        return freq / by, 1.0
    _require(scaling == "none", f"rope_frequencies: scaling {scaling!r}")
    return freq, 1.0


def rope_gpu(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, freq: torch.Tensor, head_dim: int,
             layout: str = "half", amplitude: float = 1.0, inverse: bool = False,
             q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None
             ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(q, k) [rows, heads * head_dim], fp32 or bf16 with any row stride, turned
    by positions (int32; a negative one copies its row) times freq (float64, an
    angle for each pair: the first 2 len(freq) values of a head turn, the rest is
    copied).  layout: the pairs are (i, i + len(freq)) ("half") or (2 i, 2 i + 1)
    ("pairs").  inverse turns back: the gradient.  k may be None.  q_out and k_out
    may be q and k themselves."""
    what, dev, dt = "rope", q.device, q.dtype
    code = _CODE.get(dt)
    if code is None or dev.type != "cuda":
        raise ValueError("rope: fp32 or bf16 rows on a GPU")
    if layout not in _LAYOUT:
        raise ValueError(f"rope: layout {layout!r}")
    rows, width = q.shape[0], q.shape[-1]
    q_stride = _rows_of(q, width, what)
    if head_dim < 2 or width % head_dim or positions.numel() != rows or freq.dim() != 1:
        raise ValueError("rope shape")
    if q_out is None:
        q_out, qo_stride = _like(q), width
    elif q_out.shape != q.shape or q_out.dtype is not dt or q_out.device != dev:
        raise ValueError("rope: q_out of q's shape and type")
    else:
        qo_stride = _rows_of(q_out, width, what)
    kp = kop = None
    k_heads = k_stride = ko_stride = 0
    if k is not None:
        k_width = k.shape[-1]
        k_stride = _rows_of(k, k_width, what)
        if k.shape[0] != rows or k_width % head_dim or k.dtype is not dt or k.device != dev:
            raise ValueError("rope: k [rows, heads * head_dim] of q's type")
        if k_out is None:
            k_out, ko_stride = _like(k), k_width
        elif k_out.shape != k.shape or k_out.dtype is not dt or k_out.device != dev:
            raise ValueError("rope: k_out of k's shape and type")
        else:
            ko_stride = _rows_of(k_out, k_width, what)
        kp, kop, k_heads = k.data_ptr(), k_out.data_ptr(), k_width // head_dim
    elif k_out is not None:
        raise ValueError("rope: k_out without k")
    _launch(capi.lib().aps_rope, dev, q.data_ptr(), q_stride, q_out.data_ptr(), qo_stride, width // head_dim, kp,
            k_stride, kop, ko_stride, k_heads, code, rows, head_dim, 2 * freq.shape[0], _LAYOUT[layout], inverse,
            _dev(positions, dev, torch.int32, what), _dev(freq, dev, torch.float64, what), amplitude)
    return q_out, k_out


def rope_table_gpu(freq: torch.Tensor, positions: int, amplitude: float = 1.0, first: int = 0
                   ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin) [positions, len(freq)] fp32 of the positions from `first`, times
    amplitude: kv_append_gpu's tables from such frequencies."""
    dev = freq.device
    if freq.dim() != 1 or dev.type != "cuda" or positions < 0:
        raise ValueError("rope_table: a vector of frequencies on a GPU")
    cos = torch.empty((positions, freq.shape[0]), dtype=torch.float32, device=dev)
    sin = torch.empty_like(cos)
    _launch(capi.lib().aps_rope_freq_table, dev, _dev(freq, dev, torch.float64, "rope_table"), freq.shape[0], first,
            positions, amplitude, cos.data_ptr(), sin.data_ptr())
    return cos, sin


# ---- weights in 4 bits --------------------------------------------------------

class Q4Weight:
    """A weight [out, in] in 4 bits, (code - zero) scale: codes uint8 [out, in /
    2] (two to a byte, the even input in the low half), scales [out, in / group]
    fp32 or bf16, zeros uint8 [out, in / group] (None: 8); groups of 32, 64 or
    128.  The tensors stay the caller's; quantise_q4_gpu makes them."""

    __slots__ = ("codes", "scales", "zeros", "out_features", "in_features", "group", "device", "_desc", "_ref")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None):
        dev, shape, per = codes.device, codes.shape, scales.shape
        code = _CODE.get(scales.dtype)
        if len(shape) != 2 or codes.dtype is not torch.uint8 or dev.type != "cuda" or not codes.is_contiguous():
            raise ValueError("4-bit weight: codes uint8 [out, in / 2] on a GPU")
        if len(per) != 2 or per[0] != shape[0] or not per[1] or 2 * shape[1] % per[1] or code is None or \
                scales.device != dev or not scales.is_contiguous():
            raise ValueError("4-bit weight: scales [out, in / group], fp32 or bf16")
        if zeros is not None and (zeros.shape != per or zeros.dtype is not torch.uint8 or zeros.device != dev or
                                  not zeros.is_contiguous()):
            raise ValueError("4-bit weight: zeros uint8 [out, in / group]")
        self.out_features, self.in_features, self.device = shape[0], 2 * shape[1], dev
        self.group = self.in_features // per[1]
        if self.group not in (32, 64, 128):
            raise ValueError(f"4-bit weight: groups of {self.group} (32, 64 or 128)")
        self.codes, self.scales, self.zeros = codes, scales, zeros
        self._desc = capi.Q4WeightDesc(codes.data_ptr(), scales.data_ptr(), _p(zeros), self.out_features,
                                       self.in_features, self.group, code)
        self._ref = ctypes.byref(self._desc)


def quantise_q4_gpu(weight: torch.Tensor, group: int = 128, zeros: bool = True,
                    scale_dtype: torch.dtype = torch.bfloat16) -> Q4Weight:
    """weight [out, in] (contiguous, fp32 or bf16) in 4 bits: the codes of each
    group spread over its range (zeros), or its largest magnitude at 7."""
    code = _CODE.get(weight.dtype)
    if weight.dim() != 2 or code is None or weight.device.type != "cuda" or not weight.is_contiguous():
        raise ValueError("quantise_q4: a contiguous fp32 or bf16 weight [out, in] on a GPU")
    n, k = weight.shape
    if group not in (32, 64, 128) or k % group or not k or scale_dtype not in _CODE:
        raise ValueError("quantise_q4: groups of 32, 64 or 128 that divide the inputs, fp32 or bf16 scales")
    if weight.data_ptr() % 16:   # the kernel reads 16 bytes at a time
        weight = weight.clone()
    new = lambda width, dt: torch.empty((n, width), dtype=dt, device=weight.device)  # noqa: E731
    to = Q4Weight(new(k // 2, torch.uint8), new(k // group, scale_dtype),
                  new(k // group, torch.uint8) if zeros else None)
    _launch(capi.lib().aps_quantise_q4, weight.device, weight.data_ptr(), code, to._ref)
    return to


def linear_q4_gpu(x: torch.Tensor, weight: Q4Weight, bias: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x W^T (+ bias, fp32) of x [rows, in], fp32 or bf16 with any row stride, in
    x's type.  The workspace is torch's, taken on the current stream, unless one
    is given (uint8)."""
    what, dev, dt = "linear_q4", weight.device, x.dtype
    code = _CODE.get(dt)
    if code is None or x.device != dev:
        raise ValueError("linear_q4: fp32 or bf16 rows on the weight's device")
    stride, rows, n = _rows_of(x, weight.in_features, what), x.shape[0], weight.out_features
    if out is None:
        out = torch.empty_strided((rows, n), (n, 1), dtype=dt, device=dev)   # (cheaper than empty)
    elif out.shape != (rows, n) or out.dtype is not dt or out.device != dev or not out.is_contiguous():
        raise ValueError("linear_q4: out [rows, out] of x's type, contiguous")
    bp = None
    if bias is not None:
        if bias.numel() != n:
            raise ValueError("linear_q4: a bias for each output")
        bp = _dev(bias, dev, torch.float32, what)
    lib = capi.lib()
    wp, wn = None, lib.aps_linear_q4_workspace_size(weight._ref, rows, code)
    if wn:
        if workspace is None:
            workspace = torch.empty(wn, dtype=torch.uint8, device=dev)
        elif workspace.device != dev or not workspace.is_contiguous():
            raise ValueError("linear_q4: a contiguous workspace on the weight's device")
        wp, wn = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    _launch(lib.aps_linear_q4, dev, x.data_ptr(), stride, code, rows, weight._ref, bp, out.data_ptr(), wp, wn)
    return out


# ---- log probabilities --------------------------------------------------------

MAX_TOP = 64   # likeliest tokens of a row


class TokenLogprobs(NamedTuple):
    """logprobs as the tokens' shape (None without tokens), entropy [rows],
    top_ids (int32) and top_logprobs [rows, top]."""
    logprobs: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor


def token_logprobs_gpu(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top: int = 0,
                       workspace: Optional[torch.Tensor] = None) -> TokenLogprobs:
    """Log probabilities under logits [rows, vocab], fp32 or bf16 with any row
    stride: of the given tokens ([rows] or [rows, n] int32; 0 for an id outside
    the vocabulary), and of the `top` likeliest (up to 64; of equal logits the
    lower id first), and the rows' entropies, all fp32.  Logits of -inf have the
    probability 0 (as a mask they are quicker than a finite value, whose ties the
    likeliest tokens are then picked from one by one).  The workspace is torch's, taken on the current stream, unless
    one is given (uint8)."""
    what, dev = "token_logprobs", logits.device
    code = _CODE.get(logits.dtype)
    if code is None or dev.type != "cuda" or logits.dim() != 2:
        raise ValueError("token_logprobs: fp32 or bf16 logits [rows, vocab] on a GPU")
    rows, vocab = logits.shape
    stride = _rows_of(logits, vocab, what)
    n, tp, lp, logprobs = 0, None, None, None
    if tokens is not None:
        shape = tokens.shape
        if len(shape) not in (1, 2) or shape[0] != rows:
            raise ValueError("token_logprobs: tokens [rows] or [rows, n]")
        n, tp = (shape[1] if len(shape) == 2 else 1), _dev(tokens, dev, torch.int32, what)
        logprobs = torch.empty_like(tokens, dtype=torch.float32)
        lp = logprobs.data_ptr()
    if top < 0:
        raise ValueError("token_logprobs: top is a number of tokens")
    f32, wide = torch.float32, ((rows, top), (top, 1))
    entropy = torch.empty(rows, dtype=f32, device=dev)
    top_ids = torch.empty_strided(*wide, dtype=torch.int32, device=dev)   # (cheaper than empty)
    top_logprobs = torch.empty_strided(*wide, dtype=f32, device=dev)
    lib = capi.lib()
    wp, wn = None, lib.aps_token_logprobs_workspace_size(rows, vocab, top, code)
    if wn:
        if workspace is None:
            workspace = torch.empty(wn, dtype=torch.uint8, device=dev)
        elif workspace.device != dev or not workspace.is_contiguous():
            raise ValueError("token_logprobs: a contiguous workspace on the logits' device")
        wp, wn = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    _launch(lib.aps_token_logprobs, dev, logits.data_ptr(), stride, code, rows, vocab, tp, n, top, lp,
            entropy.data_ptr(), top_ids.data_ptr(), top_logprobs.data_ptr(), wp, wn)
    return TokenLogprobs(logprobs, entropy, top_ids, top_logprobs)
