"""Decoder layer and whole-model prefill over the C ABI: the Python mirror of
include/layer.h's PhiDecoderLayer and include/model.h's PhiTinyMoEModel.

Reference order of operations (file:line in the reference tree):
  PhiDecoderLayer::forward_carry   src/layer.cu:273-300
  PhiAttention::forward (trie)     src/layer.cu:156-194
  PhiTinyMoEModel::generate        src/model.cu:45-159

A prefill runs on the rows of the prompts' prefix trie (one row per
distinct prefix, aps2026_amd.prefix): gather the embedding rows of the
nodes, then per layer
    normed = LN(x)            (first layer)   or  LN(x += carry)
    q, k, v = normed W^T + b  (fp32 FMA chains, the reference's arithmetic)
    RoPE(q, k) at node depths; attention over ancestor chains (GQA-4)
    attn = att W_o^T + b_o
    post = LN(attn += x)      (attn becomes the carried residual)
    x = MoE(post)             (router, top-2, dispatch, experts, combine)
then the final LN of x + carry, each prompt's last row and the LM head.
Every buffer is allocated once per row count (Buffers) and every step is a
sequence of C-ABI launches on one stream with no host synchronisation, so a
prefill can be timed or captured as it is.  Activations are fp32; the MoE
experts compute in the weight set's dtype (fp32, or bf16 with the router
reading fp32 x exactly and the experts a bf16 copy of it).
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from . import capi, prefix, serve
from .attention import HEAD_DIM, NUM_ATTENTION_HEADS, NUM_KV_HEADS, ROPE_THETA, SLIDING_WINDOW, _device_table
from .moe import NORM_EPS, MoeWeights, _call, register_moe_weights_gpu

EOS_TOKEN_ID = 32000                  # reference include/config.h:25
QD = NUM_ATTENTION_HEADS * HEAD_DIM   # 2048: q and attention-output width
KD = NUM_KV_HEADS * HEAD_DIM          # 512: k and v width


def _p(t: Optional[torch.Tensor]) -> ctypes.c_void_p:
    return ctypes.c_void_p(t.data_ptr() if t is not None else 0)


@dataclass
class LayerWeights:
    """One decoder layer's weights on the device (fp32 except the registered
    expert set), under the reference's model.bin names."""
    in_w: torch.Tensor
    in_b: torch.Tensor
    post_w: torch.Tensor
    post_b: torch.Tensor
    proj: Dict[str, Tuple[torch.Tensor, torch.Tensor]]   # q_proj, k_proj, v_proj, o_proj: (weight, bias)
    gate: torch.Tensor
    moe: MoeWeights

    def release(self) -> None:
        self.moe.release()


def layer_from_tensors(W: Dict[str, torch.Tensor], i: int, moe_dtype=torch.float32) -> LayerWeights:
    """model.layers.<i>.* of a name -> tensor dict (device or host fp32)."""
    dev = W["model.layers.%d.self_attn.q_proj.weight" % i].device
    p = f"model.layers.{i}."
    m = p + "block_sparse_moe."
    f32 = lambda t: t.to(device=dev, dtype=torch.float32).contiguous()
    E = W[m + "gate.weight"].shape[0]
    experts = [[f32(W[m + f"experts.{e}.{nm}.weight"]) for e in range(E)] for nm in ("w1", "w2", "w3")]
    moe = register_moe_weights_gpu(*experts, compute_dtype=moe_dtype)
    del experts
    return LayerWeights(
        in_w=f32(W[p + "input_layernorm.weight"]), in_b=f32(W[p + "input_layernorm.bias"]),
        post_w=f32(W[p + "post_attention_layernorm.weight"]), post_b=f32(W[p + "post_attention_layernorm.bias"]),
        proj={nm: (f32(W[p + f"self_attn.{nm}.weight"]), f32(W[p + f"self_attn.{nm}.bias"]))
              for nm in ("q_proj", "k_proj", "v_proj", "o_proj")},
        gate=f32(W[m + "gate.weight"]), moe=moe)


def random_layer(H: int, F: int, E: int, device, generator: torch.Generator, moe_dtype=torch.bfloat16,
                 std: float = 0.02) -> LayerWeights:
    """A random-init layer drawn on the device: linear and expert weights and
    the projection biases ~N(0, std), LayerNorm weight 1 and bias 0 (the
    usual initialisation).  The fp32 expert weights are freed once the
    packed set is registered."""
    rn = lambda *shape: (std * torch.randn(shape, generator=generator, device=device)).contiguous()
    proj = {nm: (rn(o, k), rn(o)) for nm, (o, k) in
            (("q_proj", (QD, H)), ("k_proj", (KD, H)), ("v_proj", (KD, H)), ("o_proj", (H, QD)))}
    gate = rn(E, H)
    w1 = [rn(F, H) for _ in range(E)]
    w2 = [rn(H, F) for _ in range(E)]
    w3 = [rn(F, H) for _ in range(E)]
    moe = register_moe_weights_gpu(w1, w2, w3, compute_dtype=moe_dtype)
    del w1, w2, w3
    one = torch.ones(H, device=device)
    zero = torch.zeros(H, device=device)
    return LayerWeights(in_w=one, in_b=zero, post_w=one.clone(), post_b=zero.clone(), proj=proj, gate=gate, moe=moe)


@dataclass
class RowPlan:
    """Device arrays of a prefix-trie plan for attention on node rows,
    checked once on the host: positions below the ancestor stride,
    ancestors below the row count."""
    rows: int
    max_len: int
    pos: torch.Tensor        # int32 view of u32 [rows]
    anc: torch.Tensor        # int32 view of u32 [rows][max_len]
    node_token: torch.Tensor
    last_rows: torch.Tensor  # int32 view of u32 [batch]: each prompt's last node
    prompt_tokens: int

    @staticmethod
    def from_prompts(prompts: Sequence[Sequence[int]], device) -> "RowPlan":
        # the trie on the host, its ancestor table on the device (the host
        # table is nodes x max_len words: 42 MB at C4, which took longer to
        # fill, copy and upload than a layer of the model)
        plan = prefix.prefix_dedup(prompts, with_ancestors=False)
        depth = np.asarray(plan.node_depth, np.uint32)
        if depth.size and int(depth.max()) >= plan.max_len:
            raise ValueError("prefix plan out of range")
        to_dev = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.int32)).to(device)
        anc = prefix.ancestors_gpu(plan, device)
        return RowPlan(rows=plan.nodes, max_len=plan.max_len, pos=to_dev(depth), anc=anc,
                       node_token=to_dev(np.asarray(plan.node_token, np.uint32)),
                       last_rows=to_dev(np.asarray(plan.last_rows, np.uint32)),
                       prompt_tokens=int(np.asarray(plan.token_node).shape[0]))


    @staticmethod
    def packed(prompts: Sequence[Sequence[int]], device) -> "RowPlan":
        """Every token its own row, no deduplication: row r of a prompt that
        starts at row o has position p = r - o and keys o .. r (the packed
        sequences of the reference's non-trie path, written as chains)."""
        lens = [len(p) for p in prompts]
        if not lens or min(lens) == 0:
            raise ValueError("empty input")
        rows, max_len = sum(lens), max(lens)
        pos = np.concatenate([np.arange(n, dtype=np.uint32) for n in lens])
        starts = np.repeat(np.cumsum([0] + lens[:-1]).astype(np.uint32), lens)
        cols = np.arange(max_len, dtype=np.uint32)[None, :]
        anc = np.where(cols <= pos[:, None], starts[:, None] + cols, 0).astype(np.uint32)
        to_dev = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.int32)).to(device)
        last = np.cumsum(lens).astype(np.uint32) - 1
        return RowPlan(rows=rows, max_len=max_len, pos=to_dev(pos), anc=to_dev(anc),
                       node_token=to_dev(np.concatenate([np.asarray(p, np.uint32) for p in prompts])),
                       last_rows=to_dev(last), prompt_tokens=rows)


@dataclass
class CachedRows:
    """The rows of one step over paged caches: new tokens of each sequence,
    packed, and where their keys and values go (one page table for every
    layer's cache)."""
    batch: serve.PagedBatch
    node_token: torch.Tensor   # int32 [rows]: token id of each row
    last_rows: torch.Tensor    # int32 [batch]: each sequence's last row
    window: int = SLIDING_WINDOW
    sinks: int = 0

    @property
    def rows(self) -> int:
        return self.batch.rows


def routes_view(b: "Buffers", moe: MoeWeights) -> torch.Tensor:
    """The routes [rows][2] (u8) the last MoE block wrote into b.ws."""
    off = moe.layout(b.rows).routes
    return b.ws[off:off + 2 * b.rows].view(b.rows, 2)


@dataclass
class Buffers:
    """Activations of one prefill at a row count, allocated once."""
    rows: int
    x: torch.Tensor          # residual stream / MoE output [rows][H]
    carry: torch.Tensor      # attention residual [rows][H]
    normed: torch.Tensor     # [rows][H]
    q: torch.Tensor          # [rows][QD]
    k: torch.Tensor          # [rows][KD]
    v: torch.Tensor
    att: torch.Tensor        # attention output [rows][QD]
    post: torch.Tensor       # MoE input [rows][H]
    ws: torch.Tensor         # MoE workspace (shared by the layers)
    xs: Optional[torch.Tensor] = None   # split-bf16 projections: x_hi, x_lo of one input

    def split(self, src: torch.Tensor, stream) -> torch.Tensor:
        """src [rows][n] fp32 -> its bf16 hi / lo split in xs (grown on demand)."""
        n = src.numel()
        if self.xs is None or self.xs.numel() < 2 * n:
            self.xs = torch.empty(2 * n, dtype=torch.int16, device=src.device)
        _call(capi.lib().aps_linear_tc_split(_p(src), self.rows, src.shape[1], _p(self.xs), stream))
        return self.xs

    @staticmethod
    def allocate(rows: int, H: int, moe: MoeWeights, device) -> "Buffers":
        e = lambda *s: torch.empty(s, dtype=torch.float32, device=device)
        ws = torch.empty(max(moe.layout(rows).total_bytes, 1), dtype=torch.uint8, device=device)
        return Buffers(rows, e(rows, H), e(rows, H), e(rows, H), e(rows, QD), e(rows, KD), e(rows, KD),
                       e(rows, QD), e(rows, H), ws)


class DecoderLayer:
    """PhiDecoderLayer over the C ABI (reference include/layer.h:77-95).

    tc_terms: None for the fp32 projections (the reference's default build);
    3 or 4 for the split-bf16 Linear on the q/k/v/o projections (the
    reference's USE_TC / USE_TC_ALL tensor-core path, src/layer.cu:16-27,
    src/tensor.cu:514-584), whose weights are packed here once."""

    def __init__(self, w: LayerWeights, tc_terms: Optional[int] = None):
        self.w = w
        self.H = w.in_w.numel()
        self.tc_terms = tc_terms
        self.tc = {}
        if tc_terms is not None:
            from .attention import linear_tc_prepare
            self.tc = {nm: linear_tc_prepare(wt) for nm, (wt, _) in w.proj.items()}

    def _project(self, b: Buffers, src: torch.Tensor, names, stream) -> None:
        """The projections of one input: fp32 chains, or the split products
        (x split once for all of them)."""
        L, T, K = capi.lib(), b.rows, src.shape[1]
        if self.tc:
            # every output of the input in one launch (their column blocks share the grid)
            xs = b.split(src, stream)
            cnt = len(names)
            vp = ctypes.c_void_p * cnt
            _call(L.aps_linear_tc_multi(_p(xs), T, K, cnt, vp(*[_p(self.tc[nm]) for nm, _, _ in names]),
                                        vp(*[_p(self.w.proj[nm][1]) for nm, _, _ in names]),
                                        (ctypes.c_int32 * cnt)(*[n for _, _, n in names]), int(self.tc_terms == 4),
                                        vp(*[_p(dst) for _, dst, _ in names]), stream))
        else:
            # few rows: every output of the input in one grid (q, k and v of
            # 37 rows 27 us against 46 us as two launches, of 613 rows 126
            # against 170).  Past 1,024 rows each grid fills the chip by
            # itself and q alone, then k and v together, balance better
            # (2,048 rows 361 us against 368, 10,240 rows 1775 against 1861)
            # (the shared grid takes 16-byte aligned arrays, aps_linear any)
            alone = lambda nm, dst, n: (n >= 2048 and T > 1024) or any(
                t is not None and t.data_ptr() % 16 for t in (src, dst) + tuple(self.w.proj[nm]))
            wide = [x for x in names if alone(*x)]
            narrow = [x for x in names if not alone(*x)]
            for nm, dst, n in wide:
                _call(L.aps_linear(_p(src), _p(self.w.proj[nm][0]), _p(self.w.proj[nm][1]), T, K, n, _p(dst),
                                   stream))
            if narrow:
                cnt = len(narrow)
                vp = ctypes.c_void_p * cnt
                _call(L.aps_linear_multi(_p(src), T, K, cnt, vp(*[_p(self.w.proj[nm][0]) for nm, _, _ in narrow]),
                                         vp(*[_p(self.w.proj[nm][1]) for nm, _, _ in narrow]),
                                         (ctypes.c_int32 * cnt)(*[n for _, _, n in narrow]),
                                         vp(*[_p(dst) for _, dst, _ in narrow]), stream))

    def attention(self, b: Buffers, plan: RowPlan, stream) -> None:
        """normed -> att (projections, RoPE, tree attention)."""
        L, T, H, w = capi.lib(), b.rows, self.H, self.w
        self._project(b, b.normed, (("q_proj", b.q, QD), ("k_proj", b.k, KD), ("v_proj", b.v, KD)), stream)
        c, s = _device_table(b.q.device, plan.max_len, HEAD_DIM, ROPE_THETA)
        _call(L.aps_rope_tree(_p(b.q), _p(b.k), _p(plan.pos), T, NUM_ATTENTION_HEADS, NUM_KV_HEADS, HEAD_DIM,
                              _p(c), _p(s), c.shape[0], stream))
        _call(L.aps_attention_tree(_p(b.q), _p(b.k), _p(b.v), _p(b.att), _p(plan.pos), _p(plan.anc), plan.max_len,
                                   T, NUM_ATTENTION_HEADS, NUM_KV_HEADS, HEAD_DIM, SLIDING_WINDOW, stream))

    def attention_cached(self, b: Buffers, plan: CachedRows, cache: serve.PagedKvCache, stream) -> None:
        """normed -> att over the paged cache: projections, q and k rotated as
        k and v go into the cache, attention over what is there.  All of it on
        `stream`, the current one or not."""
        self._project(b, b.normed, (("q_proj", b.q, QD), ("k_proj", b.k, KD), ("v_proj", b.v, KD)), stream)
        p = plan.batch
        c, s = _device_table(b.q.device, p.max_kv_len, HEAD_DIM, ROPE_THETA)
        with serve.on_stream(stream, b.q.device):
            serve.kv_append_gpu(cache, b.k, b.v, p.positions, p.slots, c, s, q=b.q, q_out=b.q)
            serve.attention_paged_gpu(b.q, cache, p.q_offsets, p.kv_lens, p.page_table, p.max_q_len, p.max_kv_len,
                                      q_heads=NUM_ATTENTION_HEADS, window=plan.window, sinks=plan.sinks, out=b.att)

    def forward_carry(self, b: Buffers, plan, has_carry: bool, stream, cache: Optional[serve.PagedKvCache] = None
                      ) -> None:
        """In place on b: on entry the layer input is b.x (+ b.carry when
        has_carry); on exit b.x is the MoE output and b.carry the attention
        residual.  plan: a RowPlan, or with this layer's cache CachedRows."""
        L, T, H, w = capi.lib(), b.rows, self.H, self.w
        if has_carry:
            _call(L.aps_add_layer_norm(_p(b.x), _p(b.carry), _p(w.in_w), _p(w.in_b), T, H, ctypes.c_float(NORM_EPS),
                                       _p(b.normed), stream))
        else:
            _call(L.aps_layer_norm(_p(b.x), _p(w.in_w), _p(w.in_b), T, H, ctypes.c_float(NORM_EPS), _p(b.normed),
                                   stream))
        if cache is None:
            self.attention(b, plan, stream)
        else:
            self.attention_cached(b, plan, cache, stream)
        # attn = att W_o^T + b_o into carry, then carry += x and post = LN(carry)
        self._project(b, b.att, (("o_proj", b.carry, H),), stream)
        _call(L.aps_add_layer_norm(_p(b.carry), _p(b.x), _p(w.post_w), _p(w.post_b), T, H, ctypes.c_float(NORM_EPS),
                                   _p(b.post), stream))
        _call(L.aps_moe_forward(w.moe.handle, _p(b.post), capi.DTYPE_F32, _p(w.gate), T, _p(b.x), capi.DTYPE_F32,
                                _p(b.ws), b.ws.numel(), stream))


class Model:
    """PhiTinyMoEModel's prefill (reference include/model.h:7-27,
    src/model.cu:45-159) over any number of layers."""

    def __init__(self, embeddings: torch.Tensor, norm_w: torch.Tensor, norm_b: torch.Tensor,
                 lm_head_w: torch.Tensor, lm_head_b: Optional[torch.Tensor], layers: List[LayerWeights],
                 tc: str = "off"):
        """tc: "off" (fp32 projections, the reference's default build), "tc"
        (the split-bf16 Linear, three products, for the LM head and layer
        31's attention projections: the reference's USE_TC) or "all" (four
        products, the LM head and every layer's attention projections:
        USE_TC_ALL)."""
        if tc not in ("off", "tc", "all"):
            raise ValueError("tc is 'off', 'tc' or 'all'")
        self.emb, self.norm_w, self.norm_b = embeddings, norm_w, norm_b
        self.head_w, self.head_b = lm_head_w, lm_head_b
        terms = None if tc == "off" else (4 if tc == "all" else 3)
        self.layers = [DecoderLayer(w, terms if (tc == "all" or (tc == "tc" and i == 31)) else None)
                       for i, w in enumerate(layers)]
        self.head_terms = terms
        self.head_tc = None
        if terms is not None:
            from .attention import linear_tc_prepare
            self.head_tc = linear_tc_prepare(lm_head_w)
        self.H = embeddings.shape[1]
        self._bufs: Dict[int, Buffers] = {}

    def buffers(self, rows: int) -> Buffers:
        b = self._bufs.get(rows)
        if b is None:
            b = Buffers.allocate(rows, self.H, self.layers[0].w.moe, self.emb.device)
            self._bufs[rows] = b
        return b

    def prefill(self, plan, on_layer=None, caches: Optional[Sequence[serve.PagedKvCache]] = None,
                buffers: Optional[Buffers] = None) -> torch.Tensor:
        """logits [batch][vocab] of each prompt's last token; launches only
        (the outputs come from torch's caching allocator).  on_layer(i, b),
        when given, runs after layer i's launches (for example to copy its
        routes out of the shared workspace on the same stream).  With caches
        (one a layer) plan is CachedRows: its tokens join the sequences that
        the caches hold.  buffers: the activations' place, of plan.rows rows;
        the model's own, kept for each row count, unless given."""
        L, dev = capi.lib(), self.emb.device
        stream = ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)
        b = self.buffers(plan.rows) if buffers is None else buffers
        T, H = plan.rows, self.H
        if b.rows != T:
            raise ValueError("prefill: buffers of other rows")
        _call(L.aps_gather_rows(_p(self.emb), self.emb.shape[0], H, _p(plan.node_token), T, _p(b.x), stream))
        for i, layer in enumerate(self.layers):
            layer.forward_carry(b, plan, i > 0, stream, caches[i] if caches is not None else None)
            if on_layer is not None:
                on_layer(i, b)
        if self.layers:
            _call(L.aps_add_layer_norm(_p(b.x), _p(b.carry), _p(self.norm_w), _p(self.norm_b), T, H,
                                       ctypes.c_float(NORM_EPS), _p(b.normed), stream))
        else:
            _call(L.aps_layer_norm(_p(b.x), _p(self.norm_w), _p(self.norm_b), T, H, ctypes.c_float(NORM_EPS),
                                   _p(b.normed), stream))
        batch = plan.last_rows.shape[0]
        rows_out = torch.empty((batch, H), dtype=torch.float32, device=dev)
        _call(L.aps_gather_rows(_p(b.normed), T, H, _p(plan.last_rows), batch, _p(rows_out), stream))
        V = self.head_w.shape[0]
        logits = torch.empty((batch, V), dtype=torch.float32, device=dev)
        if self.head_tc is not None:
            xs = torch.empty(2 * batch * H, dtype=torch.int16, device=dev)
            _call(L.aps_linear_tc_split(_p(rows_out), batch, H, _p(xs), stream))
            _call(L.aps_linear_tc(_p(xs), batch, H, _p(self.head_tc), _p(self.head_b), V, int(self.head_terms == 4),
                                  _p(logits), stream))
        else:
            _call(L.aps_linear(_p(rows_out), _p(self.head_w), _p(self.head_b), batch, H, V, _p(logits), stream))
        return logits

    def generate(self, prompts: Sequence[Sequence[int]]) -> torch.Tensor:
        return self.prefill(RowPlan.from_prompts(prompts, self.emb.device))

    def generate_decode(self, prompts: Sequence[Sequence[int]], max_new_tokens: int, kv_dtype=torch.float32,
                        page_size: int = 16, window: int = SLIDING_WINDOW, sinks: int = 0,
                        repetition: float = 1.0, frequency: float = 0.0, presence: float = 0.0,
                        bias: Optional[Dict[int, float]] = None, mask: Optional[torch.Tensor] = None,
                        eos: int = EOS_TOKEN_ID) -> Tuple[List[List[int]], torch.Tensor]:
        """Greedy decoding of a prompt batch on paged caches (kv_dtype:
        torch.float32, torch.bfloat16 or "mxfp4"): each token is computed once,
        where the reference's generate_decode runs the whole prefix again for
        each (src/model.cu:163-204).  Returns the new ids of each prompt, up to
        and with eos, and the logits [batch][max_new_tokens][vocab] they were
        chosen from: after the penalties, the biases {id: value} and the mask
        ([1] or [batch] rows of int32 words, bit t % 32 of word t / 32 allows
        token t).  Of equal logits the lowest id wins; NaN never does beside
        a number, and of none but NaN and -inf id 0.  One host wait, at the
        end.  Caches and activations are the call's own, from torch's caching
        allocator: calls may run side by side on other streams."""
        if len(prompts) == 0:
            raise RuntimeError("generate_decode received an empty input batch")
        if max_new_tokens < 1:
            raise ValueError("max_new_tokens must be positive")
        dev, n_seq = self.emb.device, len(prompts)
        V = self.head_w.shape[0]
        lens = [len(p) for p in prompts]
        flat = np.concatenate([np.asarray(p, np.int64).reshape(-1) for p in prompts])
        if min(lens) == 0:
            raise ValueError("empty input")
        if max(lens) + max_new_tokens - 1 > prefix.MAX_POSITION_EMBEDDINGS:
            raise ValueError("sequence is too long")
        if flat.min() < 0 or flat.max() >= self.emb.shape[0]:
            raise ValueError("token out of vocabulary")
        if not repetition > 0.0:
            raise ValueError("repetition must be positive")
        if page_size not in (16, 32, 64, 128, 256):
            raise ValueError("page_size is 16, 32, 64, 128 or 256")
        if mask is not None and (mask.dim() != 2 or mask.shape[0] not in (1, n_seq)):
            raise ValueError("mask: one row of words, or one a prompt")
        # pages for the whole answer, consecutive for each sequence
        need = [-(-(n + max_new_tokens - 1) // page_size) for n in lens]
        first = np.cumsum([0] + need)
        pages = [range(first[b], first[b + 1]) for b in range(n_seq)]
        caches = [serve.PagedKvCache.allocate(int(first[-1]), page_size, NUM_KV_HEADS, HEAD_DIM, kv_dtype, dev)
                  for _ in self.layers]
        plan = serve.PagedBatch(lens, lens, pages, page_size, dev, num_pages=int(first[-1]))
        last = np.cumsum(lens) - 1
        i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
        rows = CachedRows(plan, i32(flat), i32(last), window, sinks)
        # one new token a sequence from here on: the same arrays, advanced on the device
        step = serve.PagedBatch([1] * n_seq, [n + max_new_tokens - 1 for n in lens], pages, page_size, dev)
        kv_lens, seq = i32(lens), torch.arange(n_seq, device=dev)
        rules = {}
        history = None
        if repetition != 1.0 or frequency != 0.0 or presence != 0.0:
            history = torch.full((n_seq, max(lens) + max_new_tokens), -1, dtype=torch.int32, device=dev)
            for b, p in enumerate(prompts):
                history[b, :lens[b]] = i32(p)
            full = lambda v: torch.full((n_seq,), v, dtype=torch.float32, device=dev)  # noqa: E731
            rules.update(history=history, prompt_lens=i32(lens), repetition=full(repetition),
                         frequency=full(frequency), presence=full(presence))
        if bias:
            rules.update(bias_ids=i32([list(bias)] * n_seq), bias_lens=i32([len(bias)] * n_seq),
                         bias_values=torch.tensor([list(bias.values())] * n_seq, dtype=torch.float32, device=dev))
        if mask is not None:
            rules.update(mask=mask.to(dev).contiguous())
            if mask.shape[0] == 1:
                rules.update(mask_index=torch.zeros(n_seq, dtype=torch.int32, device=dev))
        out = torch.empty((n_seq, max_new_tokens, V), dtype=torch.float32, device=dev)
        ids = torch.empty((n_seq, max_new_tokens), dtype=torch.int32, device=dev)
        bufs = None
        for t in range(max_new_tokens):
            if bufs is None or bufs.rows != rows.rows:
                bufs = Buffers.allocate(rows.rows, self.H, self.layers[0].w.moe, dev)
            logits = self.prefill(rows, caches=caches, buffers=bufs)
            if rules:
                if history is not None:
                    rules["history_lens"] = kv_lens
                serve.logits_process_gpu(logits, out=logits, **rules)
            out[:, t] = logits
            # argmax leaves open which of equal logits it takes, and takes a NaN
            x = torch.where(logits.isnan(), -math.inf, logits)
            token = torch.where(x == x.amax(1, keepdim=True), torch.arange(V, device=dev), V).amin(1).to(torch.int32)
            ids[:, t] = token
            if t + 1 == max_new_tokens:
                break
            if history is not None:
                history[seq, kv_lens.long()] = token
            step.positions = kv_lens.clone()
            kv_lens = kv_lens + 1
            at = step.positions.long()
            page = step.page_table[seq, at // page_size].long()
            step.slots, step.kv_lens = page * page_size + at % page_size, kv_lens
            rows = CachedRows(step, token, seq.to(torch.int32), window, sinks)
        done = []
        for row in ids.cpu().tolist():
            done.append(row[:row.index(eos) + 1] if eos in row else row)
        return done, out
