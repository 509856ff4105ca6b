"""Serving operators over the C ABI (include/aps_serve.h): a paged key/value
cache, attention over it, and the rules on the logits of the next token.

The reference has no counterpart: its generate_decode computes the whole
prefix again for every token (src/model.cu:163-204).
decoder.Model.generate_decode runs on these.

A decode step of a batch, on torch's current stream:

    plan = PagedBatch(q_lens, kv_lens, pages, cache.page_size, device)
    q = kv_append_gpu(cache, k, v, plan.positions, plan.slots, cos, sin, q=q)
    out = attention_paged_gpu(q, cache, plan.q_offsets, plan.kv_lens, plan.page_table, plan.max_q_len,
                              plan.max_kv_len, q_heads=16, window=2047, sinks=4)

Calls launch kernels and read nothing back, so they can be captured into a
graph; index arrays are read on the device (PagedBatch checks its own on the
host).  Wrong shapes, types and layouts raise ValueError.
"""
from __future__ import annotations

import contextlib
import ctypes
import math
from typing import Optional, Sequence, Tuple

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
