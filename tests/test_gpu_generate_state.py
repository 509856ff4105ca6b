"""What decoding on paged caches keeps and shares between calls."""
import ctypes
import gc
import threading

import pytest
import torch

from aps2026_amd import decoder, serve
from tests.device_weights import random_model_weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(gpu_device):
    W = random_model_weights(gpu_device, H=512, F=64, E=4, V=256, layers=2, seed=9)
    layers = [decoder.layer_from_tensors(W, i, torch.float32) for i in range(2)]
    return decoder.Model(W["model.embed_tokens.weight"], W["model.norm.weight"], W["model.norm.bias"],
                         W["lm_head.weight"], W["lm_head.bias"], layers)


def test_memory_does_not_grow_with_the_prompts_seen(model, gpu_device):
    """Prompts of other totals leave nothing behind."""
    def used(total):
        model.generate_decode([[1] * total, [2, 3]], 3)
        gc.collect()
        torch.cuda.synchronize()
        return torch.cuda.memory_allocated(gpu_device)

    first = used(500)
    kept = set(model._bufs)
    assert [used(n) for n in (400, 333, 100, 499)] == [first] * 4
    assert set(model._bufs) == kept


def test_buffers_of_other_rows_are_refused(model, gpu_device):
    b = decoder.Buffers.allocate(4, model.H, model.layers[0].w.moe, gpu_device)
    plan = decoder.RowPlan.packed([[1, 2, 3]], gpu_device)
    with pytest.raises(ValueError, match="buffers of other rows"):
        model.prefill(plan, buffers=b)


def test_calls_on_two_streams_at_once(model, gpu_device):
    """Two batches of equal size, decoded at the same time from two threads,
    each on its own stream, are what they are one after the other."""
    batches = [[[5, 9, 9, 200, 31], list(range(40)), [7]], [[11, 12], [13] * 25, list(range(90, 120))]]
    want = [model.generate_decode(p, 12, eos=-1) for p in batches]
    torch.cuda.synchronize()
    got, failed = [None, None], []

    def decode(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream(gpu_device)):
                got[i] = [model.generate_decode(batches[i], 12, eos=-1) for _ in range(4)]
        except Exception as e:   # noqa: BLE001 (shown by the assertion below)
            failed.append(e)

    threads = [threading.Thread(target=decode, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    torch.cuda.synchronize()
    for i in range(2):
        for ids, logits in got[i]:
            assert ids == want[i][0] and torch.equal(logits, want[i][1])


@pytest.mark.parametrize("as_int", [True, False])
def test_a_layer_runs_on_the_stream_it_is_given(model, gpu_device, as_int):
    """A side stream that is busy, and the default stream from within another:
    the layer's attention waits for its projections there."""
    dev, layer = gpu_device, model.layers[0]
    plan = serve.PagedBatch([21], [21], [[1, 0]], 16, dev, num_pages=2)
    rows = decoder.CachedRows(plan, torch.zeros(21, dtype=torch.int32, device=dev),
                              torch.zeros(1, dtype=torch.int32, device=dev))
    x = torch.randn(21, model.H, generator=torch.Generator(dev).manual_seed(4), device=dev)

    def run(stream, within):
        cache = serve.PagedKvCache.allocate(2, 16, 4, 128, torch.float32, dev)
        b = decoder.Buffers.allocate(21, model.H, layer.w.moe, dev)
        b.normed.copy_(x)
        for t in (b.q, b.k, b.v, b.att):
            t.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(within), torch.cuda.stream(stream):
            torch.cuda._sleep(20_000_000)              # about 10 ms before the projections
        with torch.cuda.stream(within):
            handle = stream.cuda_stream
            layer.attention_cached(b, rows, cache, handle if as_int else ctypes.c_void_p(handle))
        torch.cuda.synchronize()
        return b.att.clone(), cache.k.clone(), cache.v.clone()

    default, side = torch.cuda.default_stream(dev), torch.cuda.Stream(dev)
    want = run(default, default)
    assert bool(want[0].abs().sum() > 0)
    for stream, within in ((side, default), (default, side), (side, side)):
        assert all(torch.equal(a, b) for a, b in zip(run(stream, within), want))


def test_a_logit_that_is_nan_is_not_chosen(model, gpu_device):
    """One token's logit is NaN in every step: the choice is the largest of the
    others; of nothing but NaN it is token 0."""
    ids, logits = model.generate_decode([[5, 9, 200], [7]], 3, eos=-1)
    keep = model.head_w.clone()
    try:
        model.head_w[ids[0][0]] = float("nan")
        got, with_nan = model.generate_decode([[5, 9, 200], [7]], 3, eos=-1)
        assert bool(with_nan[:, :, ids[0][0]].isnan().all())
        best = torch.where(with_nan.isnan(), -float("inf"), with_nan).amax(2)
        assert got[0][0] != ids[0][0]
        for b in range(2):
            for t in range(3):
                assert with_nan[b, t, got[b][t]] == best[b, t]
        second = logits[:, 0].clone()
        second[:, ids[0][0]] = -float("inf")
        assert [row[0] for row in got] == second.argmax(1).tolist()
        model.head_w.fill_(float("nan"))
        assert model.generate_decode([[5], [7, 8]], 2, eos=-1)[0] == [[0, 0], [0, 0]]
    finally:
        model.head_w.copy_(keep)
