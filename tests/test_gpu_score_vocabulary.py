"""Model.score where the head gives fewer logits than there are embeddings."""
import pytest
import torch

from aps2026_amd import decoder
from tests.device_weights import random_model_weights

pytestmark = pytest.mark.gpu


def test_a_token_without_a_logit_is_refused(gpu_device):
    """It has no probability: 0, that of a padding id, would be that of certainty."""
    print("[gpu-case] score of a narrower head", flush=True)
    W = random_model_weights(gpu_device, H=256, F=64, E=4, V=120, layers=1, seed=3)
    layers = [decoder.layer_from_tensors(W, 0, torch.float32)]
    model = decoder.Model(W["model.embed_tokens.weight"], W["model.norm.weight"], W["model.norm.bias"],
                          W["lm_head.weight"][:100].contiguous(), W["lm_head.bias"][:100].contiguous(), layers)
    for prompts in ([[1, 100]], [[5, 6], [3, 119, 2]]):
        with pytest.raises(ValueError, match="vocabulary"):
            model.score(prompts)
    got = model.score([[119, 99, 4], [110]])      # the first of a prompt is read, not scored
    assert [r.logprobs.shape[0] for r in got] == [2, 0] and bool((got[0].logprobs < 0).all())
