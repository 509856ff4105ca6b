"""Rotary embedding and GQA tree attention over prefix-trie rows, over the C
ABI (include/aps_moe.h).

Reference API mirrored (file:line in the reference tree):
  Linear::forward (projections)     src/layer.cu:30-42, src/tensor.cu:3120-3143
  tensor_ops::apply_rope_tree_gpu   include/tensor.h:100-103, src/tensor.cu:3342-3359
  tensor_ops::attention_tree_gpu    include/tensor.h:109-114, src/tensor.cu:3361-3377
  rope_table                        src/tensor.cu:2703-2735 (host tables)

Rows are the nodes of the prompts' prefix trie (aps2026_amd.prefix): a
node's RoPE position is its depth and its keys are its ancestor chain, so
attention needs no expansion back to token rows.  Shapes as the reference:
q [rows, q_heads * 128], k and v [rows, kv_heads * 128], fp32, q_heads =
4 kv_heads.  Errors raise ValueError with the reference's messages
("attention_tree_gpu expects GQA-4").
"""
from __future__ import annotations

from typing import Dict, List, Tuple, Union

import numpy as np
import torch

from . import capi
from .moe import _call, _ptr, _stream

NUM_ATTENTION_HEADS = 16   # reference include/config.h:10
NUM_KV_HEADS = 4           # include/config.h:11
HEAD_DIM = 128             # include/config.h:12
SLIDING_WINDOW = 2047      # include/config.h:17
ROPE_THETA = 10000.0       # include/config.h:18

_tables: Dict[Tuple[torch.device, int, float], List[Tuple[torch.Tensor, torch.Tensor]]] = {}


def rope_table(max_seq: int, head_dim: int = HEAD_DIM, theta: float = ROPE_THETA) -> Tuple[np.ndarray, np.ndarray]:
    """(cos, sin) [max_seq, head_dim / 2], the reference's host tables."""
    half = head_dim // 2
    c = np.empty((max_seq, half), np.float32)
    s = np.empty((max_seq, half), np.float32)
    _call(capi.lib().aps_rope_table(max_seq, head_dim, theta, c.ctypes.data_as(capi._c_vp),
                                    s.ctypes.data_as(capi._c_vp)))
    return c, s


def _device_table(device: torch.device, max_seq: int, head_dim: int, theta: float):
    """Device copies of the tables, kept per device and grown on demand (the
    reference keeps one static table, src/tensor.cu:2703-2712).  The ones
    outgrown stay, for kernels still under way on another stream and recorded
    graphs read them; each has at least twice the rows of the one before, so
    all of them take less than twice the newest's memory."""
    kept = _tables.setdefault((device, head_dim, float(theta)), [])
    if not kept or kept[-1][0].shape[0] < max_seq:
        rows = max(max_seq, 2 * kept[-1][0].shape[0]) if kept else max_seq
        c, s = rope_table(rows, head_dim, theta)
        kept.append((torch.from_numpy(c).to(device), torch.from_numpy(s).to(device)))
    return kept[-1]


def _rows_u32(t: Union[torch.Tensor, np.ndarray], device) -> torch.Tensor:
    if isinstance(t, torch.Tensor):
        return t.to(device=device, dtype=torch.int32).contiguous()
    return torch.from_numpy(np.ascontiguousarray(np.asarray(t, dtype=np.uint32)).view(np.int32)).to(device)


def linear_gpu(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor = None,
               out: torch.Tensor = None) -> torch.Tensor:
    """y = x weight^T (+ bias), fp32, each output one FMA chain over k
    ascending and the bias added once: the decoder's Linear layers (reference
    src/layer.cu:30-42, src/tensor.cu:3120-3143, kernel :715-800)."""
    k = x.shape[-1]
    rows = x.numel() // k if k else 0
    n = weight.shape[0]
    if weight.shape[1] != k or (bias is not None and bias.numel() != n):
        raise ValueError("matmul_transposed_bias_gpu shape")
    for t in (x, weight) + ((bias,) if bias is not None else ()):
        if t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError("linear_gpu expects contiguous fp32 tensors")
    if out is None:
        out = torch.empty((rows, n), dtype=torch.float32, device=x.device)
    elif out.numel() != rows * n or out.dtype != torch.float32 or not out.is_contiguous():
        raise ValueError("matmul_transposed_bias_gpu shape")
    _call(capi.lib().aps_linear(_ptr(x), _ptr(weight), _ptr(bias), rows, k, n, _ptr(out), _stream(x.device)))
    return out


def linear_tc_prepare(weight: torch.Tensor) -> torch.Tensor:
    """The reference's Tensor::prepare_cuda_bf16_weight(true) (src/tensor.cu:
    149-177): weight [out][in] fp32 -> packed bf16 hi / lo tile images on the
    weight's device (the USE_TC Linear's operand)."""
    n, k = weight.shape
    if weight.dtype != torch.float32 or not weight.is_contiguous():
        raise ValueError("linear_tc_prepare expects a contiguous fp32 matrix")
    nbytes = capi.lib().aps_linear_tc_packed_bytes(n, k)
    if nbytes == 0 or n % 4 != 0:
        raise ValueError("linear_tc_prepare shape: out % 4 == 0, in % 64 == 0")
    packed = torch.empty(nbytes, dtype=torch.uint8, device=weight.device)
    _call(capi.lib().aps_linear_tc_prepare(_ptr(weight), n, k, _ptr(packed), nbytes, _stream(weight.device)))
    return packed


def linear_tc_split(x: torch.Tensor) -> torch.Tensor:
    """x [rows][in] fp32 -> [2][rows][in] bf16 bits (x_hi, x_lo), the
    USE_TC kernel's on-the-fly split done once per input."""
    k = x.shape[-1]
    rows = x.numel() // k
    if x.dtype != torch.float32 or not x.is_contiguous():
        raise ValueError("linear_tc_split expects contiguous fp32")
    out = torch.empty((2, rows, k), dtype=torch.int16, device=x.device)
    _call(capi.lib().aps_linear_tc_split(_ptr(x), rows, k, _ptr(out), _stream(x.device)))
    return out


def linear_tc_gpu(x_split: torch.Tensor, packed: torch.Tensor, out_features: int, bias: torch.Tensor = None,
                  all_terms: bool = False, out: torch.Tensor = None) -> torch.Tensor:
    """y = x_hi W_hi + x_hi W_lo + x_lo W_hi (+ x_lo W_lo) (+ bias): the
    reference's USE_TC / USE_TC_ALL Linear (src/tensor.cu:514-584)."""
    _, rows, k = x_split.shape
    if out is None:
        out = torch.empty((rows, out_features), dtype=torch.float32, device=x_split.device)
    _call(capi.lib().aps_linear_tc(_ptr(x_split), rows, k, _ptr(packed), _ptr(bias), out_features, int(all_terms),
                                   _ptr(out), _stream(x_split.device)))
    return out


def apply_rope_tree_gpu(q: torch.Tensor, k: torch.Tensor, row_pos, max_seq: int,
                        q_heads: int = NUM_ATTENTION_HEADS, kv_heads: int = NUM_KV_HEADS,
                        head_dim: int = HEAD_DIM, theta: float = ROPE_THETA) -> None:
    """RoPE in place on q and k at each row's position (reference
    src/tensor.cu:3342-3359)."""
    rows = q.shape[0]
    if q.numel() != rows * q_heads * head_dim or k.numel() != rows * kv_heads * head_dim:
        raise ValueError("apply_rope_tree_gpu shape")
    if q.dtype != torch.float32 or k.dtype != torch.float32 or not q.is_contiguous() or not k.is_contiguous():
        raise ValueError("apply_rope_tree_gpu expects contiguous fp32 tensors")
    pos = _rows_u32(row_pos, q.device)
    if rows and int(pos.max().item()) >= max_seq:
        raise ValueError("apply_rope_tree_gpu position past max_seq")
    c, s = _device_table(q.device, max_seq, head_dim, theta)
    _call(capi.lib().aps_rope_tree(_ptr(q), _ptr(k), _ptr(pos), rows, q_heads, kv_heads, head_dim, _ptr(c), _ptr(s),
                                   c.shape[0], _stream(q.device)))


def attention_tree_gpu(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, row_pos, anc,
                       anc_stride: int, q_heads: int = NUM_ATTENTION_HEADS, kv_heads: int = NUM_KV_HEADS,
                       head_dim: int = HEAD_DIM, window: int = SLIDING_WINDOW) -> torch.Tensor:
    """out = softmax attention of each row over its ancestor chain (reference
    src/tensor.cu:3361-3377)."""
    if q_heads != 4 * kv_heads:
        raise ValueError("attention_tree_gpu expects GQA-4")
    rows = q.shape[0]
    for t, h in ((q, q_heads), (k, kv_heads), (v, kv_heads), (out, q_heads)):
        if t.numel() != rows * h * head_dim or t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError("attention_tree_gpu shape")
    pos = _rows_u32(row_pos, q.device)
    a = _rows_u32(anc, q.device)
    if rows:
        if int(pos.max().item()) >= anc_stride or a.numel() < rows * anc_stride:
            raise ValueError("attention_tree_gpu ancestor table")
        # every key a row can see must be a row of this batch (the u32 table
        # is viewed as int32: entries >= 2^31 read as negative)
        tab = a[:rows * anc_stride].view(rows, anc_stride)
        live = torch.arange(anc_stride, device=q.device)[None, :] <= pos[:, None]
        if bool((((tab < 0) | (tab >= rows)) & live).any()):
            raise ValueError("attention_tree_gpu ancestor index")
    _call(capi.lib().aps_attention_tree(_ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(pos), _ptr(a), anc_stride, rows,
                                        q_heads, kv_heads, head_dim, window, _stream(q.device)))
    return out
