"""Weights as they come to the 4-bit layers (serve.quantise_q4_gpu,
decoder.Model(tc="q4")): off 16 bytes, and what the model keeps of them."""
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
