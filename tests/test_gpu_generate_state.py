"""What decoding on paged caches keeps and shares between calls."""
import gc
import threading

import pytest
import torch

from aps2026_amd import decoder
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
