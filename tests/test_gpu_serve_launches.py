"""Calls of the paged cache's and the logits' operators (include/aps_serve.h) past
what one launch's grid holds: 2^32 threads."""
import ctypes

import torch

from aps2026_amd import capi, serve
from tests.test_gpu_decode_launches import BF16, _free_memory, assert_repeats, note, pytestmark, repeated  # noqa: F401

I32 = torch.int32


def test_logits_of_many_rows(gpu_device):
    rows, n, v = (1 << 24) + 21, 1021, 12
    note(f"logits of {rows} rows")
    dev = gpu_device
    ids = lambda *s: torch.randint(0, v, s, dtype=I32, device=dev)  # noqa: E731
    rules = dict(history=ids(n, 3), history_lens=torch.randint(0, 4, (n,), dtype=I32, device=dev),
                 prompt_lens=torch.ones(n, dtype=I32, device=dev), repetition=1 + torch.rand(n, device=dev),
                 frequency=torch.rand(n, device=dev), presence=torch.rand(n, device=dev), bias_ids=ids(n, 2),
                 bias_values=torch.randn(n, 2, device=dev), bias_lens=torch.randint(0, 3, (n,), dtype=I32, device=dev),
                 mask=torch.randint(1, 1 << v, (n, 1), dtype=I32, device=dev))
    x = torch.randn(n, v, device=dev).to(BF16)
    many = {name: repeated(t, rows) for name, t in rules.items()}
    assert_repeats(serve.logits_process_gpu(repeated(x, rows), **many), serve.logits_process_gpu(x, **rules))
    # each row its mask by an index
    many["mask_index"], many["mask"] = repeated(torch.arange(n, dtype=I32, device=dev), rows), rules["mask"]
    assert_repeats(serve.logits_process_gpu(repeated(x, rows), **many), serve.logits_process_gpu(x, **rules))


def test_cache_of_many_rows(gpu_device):
    """One head of 64 values a row; k and v from the same rows, most of them into no slot."""
    rows, n, pages = (1 << 29) + 5, 1019, 4
    note(f"cache of {rows} rows")
    dev = gpu_device
    cache = serve.PagedKvCache.allocate(pages, 16, 1, 64, BF16, dev)
    few = torch.randn(n, 64, device=dev).to(BF16)
    x = repeated(few, rows)
    at = torch.tensor([0, 1, (1 << 29) - 33, (1 << 29) - 32, (1 << 29) - 1, 1 << 29, rows - 1], device=dev)   # (a launch ends at 2^29 - 32)
    slots = torch.full((rows,), -1, dtype=torch.int64, device=dev)
    slots[at] = torch.arange(len(at), device=dev)
    positions = torch.full((rows,), -1, dtype=I32, device=dev)
    serve.kv_append_gpu(cache, x, x, positions, slots, torch.zeros(1, 32, device=dev), torch.zeros(1, 32, device=dev))
    for held in (cache.k, cache.v):
        assert torch.equal(held.view(-1, 64)[:len(at)], few[at % n])
        assert not bool(held.view(-1, 64)[len(at):].any())
    del positions
    # back, the cache's first rows again and again
    few_slots = torch.arange(len(at), device=dev)
    slots.copy_(torch.arange(rows, device=dev).remainder_(len(at)))
    rc = capi.lib().aps_kv_gather(cache._ref, slots.data_ptr(), rows, x.data_ptr(), None, capi.DTYPE_BF16,
                                  ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0
    assert_repeats(x, serve.kv_gather_gpu(cache, few_slots, BF16)[0])
