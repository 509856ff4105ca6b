"""Serving operators on arrays that share memory, on the GPU."""
import numpy as np
import pytest
import torch

from aps2026_amd import attention, serve

pytestmark = pytest.mark.gpu


def test_append_between_the_rows_of_one_buffer(gpu_device):
    """q, k, v and the rotated queries as slices of one wider row, and a row that
    is shifted into its neighbours."""
    dev, rows, dim = gpu_device, 11, 64
    cos, sin = (torch.from_numpy(a).to(dev) for a in attention.rope_table(rows, dim))
    pos = torch.arange(rows, dtype=torch.int32, device=dev)
    slots = torch.arange(rows, device=dev)
    x = torch.from_numpy(np.random.default_rng(0).standard_normal((rows, 6 * dim), dtype=np.float32)).to(dev)
    q, k, v, q_out = x.split([2 * dim, dim, dim, 2 * dim], 1)
    cache = serve.PagedKvCache.allocate(1, 16, 1, dim, torch.float32, dev)
    want = serve.kv_append_gpu(cache, k, v, pos, slots, cos, sin, q=q)
    held = cache.k.clone(), cache.v.clone()
    cache.k.zero_(), cache.v.zero_()
    assert serve.kv_append_gpu(cache, k, v, pos, slots, cos, sin, q=q, q_out=q_out) is q_out
    assert torch.equal(q_out, want) and torch.equal(cache.k, held[0]) and torch.equal(cache.v, held[1])
    for to in (x[:, 1:2 * dim + 1], x[:, 2 * dim:4 * dim], x[:, dim:3 * dim]):
        with pytest.raises(ValueError, match="q_out overlaps"):
            serve.kv_append_gpu(cache, k, v, pos, slots, cos, sin, q=q, q_out=to)


def test_logits_beside_their_rows(gpu_device):
    """Logits and their results as halves of one buffer's rows; a shifted slice."""
    dev = gpu_device
    x = torch.randn(7, 2 * 45, device=dev)
    mask = torch.full((7, 2), 0x5A5A5A5A, dtype=torch.int32, device=dev)
    want = serve.logits_process_gpu(x[:, :45].contiguous(), mask=mask)
    out = x[:, 45:]
    assert serve.logits_process_gpu(x[:, :45], mask=mask, out=out) is out and torch.equal(out, want)
    with pytest.raises(ValueError, match="overlap"):
        serve.logits_process_gpu(x[:, :45], mask=mask, out=x[:, 1:46])


def test_one_row_of_a_wider_buffer(gpu_device):
    """A single token's queries and logits, taken from rows of odd width."""
    dev = gpu_device
    cache = serve.PagedKvCache.allocate(2, 16, 1, 64, torch.bfloat16, dev)
    cache.k.normal_(), cache.v.normal_()
    plan = serve.PagedBatch([1], [20], [[1, 0]], 16, dev)
    wide = torch.randn(3, 2 * 64 + 1, dtype=torch.bfloat16, device=dev)
    args = (cache, plan.q_offsets, plan.kv_lens, plan.page_table, 1, 20)
    want = serve.attention_paged_gpu(wide[:1, :128].contiguous(), *args, q_heads=2, window=64)
    assert torch.equal(serve.attention_paged_gpu(wide[:1, :128], *args, q_heads=2, window=64), want)
    with pytest.raises(ValueError, match="stride"):
        serve.attention_paged_gpu(wide[:2, :128], *args, q_heads=2, window=64)
    x = torch.randn(3, 91, device=dev)
    y = x[:1, :90]
    bias = dict(bias_ids=torch.tensor([[5]], dtype=torch.int32, device=dev), bias_values=torch.ones(1, 1, device=dev),
                bias_lens=torch.ones(1, dtype=torch.int32, device=dev))
    want = serve.logits_process_gpu(y.contiguous(), **bias)
    assert torch.equal(serve.logits_process_gpu(y, out=y, **bias), want) and torch.equal(x[:1, :90], want)
