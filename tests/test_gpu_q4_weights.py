"""Weights as they come to the 4-bit layers (serve.quantise_q4_gpu,
decoder.Model(tc="q4")): off 16 bytes, and what the model keeps of them."""
import gc
import weakref

import pytest
import torch

from aps2026_amd import decoder, serve
from tests.device_weights import random_model_weights

pytestmark = pytest.mark.gpu

H, V, LAYERS = 512, 259, 2
PROMPTS = [[5, 9, 9, 200, 31], [7]]


def off16(t):
    """t at an address that is no multiple of 16 bytes."""
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    buf[1:].copy_(t.reshape(-1))
    return buf[1:].view(t.shape)


def same(a, b):
    return torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales) and torch.equal(a.zeros, b.zeros)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantise_q4_off_16_bytes(gpu_device, dtype):
    print(f"[gpu-case] quantise_q4 off 16 bytes {dtype}", flush=True)
    w = torch.randn(40, 384, device=gpu_device).to(dtype)
    odd = off16(w)
    assert odd.data_ptr() % 16 and same(serve.quantise_q4_gpu(odd, 64), serve.quantise_q4_gpu(w, 64))
    assert torch.equal(odd, w)


def build(dev, change=lambda t: t, tc="q4"):
    W = random_model_weights(dev, H=H, F=64, E=4, V=V, layers=LAYERS, seed=9)
    layers = [decoder.layer_from_tensors(W, i, torch.float32) for i in range(LAYERS)]
    for lw in layers:
        lw.proj = {n: tuple(change(t) for t in p) for n, p in lw.proj.items()}
    head = change(W["lm_head.weight"])
    return decoder.Model(W["model.embed_tokens.weight"], W["model.norm.weight"], W["model.norm.bias"], head,
                         W["lm_head.bias"], layers, tc=tc), head, layers


def test_model_of_weights_off_16_bytes(gpu_device):
    print("[gpu-case] model off 16 bytes", flush=True)
    (odd, *_), (plain, *_) = build(gpu_device, off16), build(gpu_device)
    assert torch.equal(odd.generate(PROMPTS), plain.generate(PROMPTS))


def test_model_keeps_no_weights_but_in_4_bits(gpu_device):
    """What the caller drops is freed: the head's and the projections' fp32 values."""
    print("[gpu-case] model keeps none", flush=True)
    model, head, layers = build(gpu_device)
    want = model.generate(PROMPTS)
    refs = [weakref.ref(head)] + [weakref.ref(w) for lw in layers for w, _ in lw.proj.values()]
    assert all(r() is not None for r in refs)
    del head, layers
    gc.collect()
    assert [r() for r in refs] == [None] * (1 + 4 * LAYERS)
    assert torch.equal(model.generate(PROMPTS), want)
    assert [r.logprobs.shape[0] for r in model.score(PROMPTS)] == [4, 0]
    assert model.generate_decode(PROMPTS, 2, eos=-1)[1].shape == (2, 2, V)


def test_weights_of_another_stream_may_be_freed(gpu_device):
    """Freed as soon as the model is there, their memory goes to no other tensor while it is read."""
    print("[gpu-case] model on another stream", flush=True)
    want = build(gpu_device)[0].generate(PROMPTS)
    torch.cuda.synchronize()
    W, head, layers = build(gpu_device, tc="off")
    args = (W.emb, W.norm_w, W.norm_b)
    bias = W.head_b
    del W
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(int(2e7))      # the quantising waits behind it
        model = decoder.Model(*args, head, bias, layers, tc="q4")
    sizes = [head.shape] + [w.shape for lw in layers for w, _ in lw.proj.values()]
    del head, layers
    gc.collect()
    over = [torch.full(tuple(s), float("nan"), device=gpu_device) for s in sizes]   # on the weights' own stream
    torch.cuda.synchronize()
    assert over and torch.equal(model.generate(PROMPTS), want)
