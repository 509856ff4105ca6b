"""A decoder whose projections and LM head are in 4 bits (decoder.Model(tc="q4")),
and what a decoder says about tokens: generate_decode's log probabilities and
Model.score."""
import numpy as np
import pytest
import torch

from aps2026_amd import decoder, serve
from tests import decode_oracle as oracle
from tests.device_weights import random_model_weights

pytestmark = pytest.mark.gpu

LAYERS, H, V = 2, 512, 259
PROMPTS = [[5, 9, 9, 200, 31], list(range(40)), [7]]
# Two layers of fp32 products of at most 2048 steps, eight one after another on
# the way through a layer: 2 * 8 * 2048 * 2^-24, if every rounding went one way.
FP32 = 2 * 8 * 2048 * 2.0 ** -24


def build(dev, tc="off", change=lambda name, t: t):
    W = random_model_weights(dev, H=H, F=64, E=4, V=V, layers=LAYERS, seed=9)
    W = {n: change(n, t) for n, t in W.items()}
    layers = [decoder.layer_from_tensors(W, i, torch.float32) for i in range(LAYERS)]
    return decoder.Model(W["model.embed_tokens.weight"], W["model.norm.weight"], W["model.norm.bias"],
                         W["lm_head.weight"], W["lm_head.bias"], layers, tc=tc)


def near(a, b, tol):
    return bool(((a - b).norm(dim=-1) <= tol * b.norm(dim=-1)).all())


def f64(t):
    return t.detach().cpu().double().numpy()


@pytest.fixture(scope="module")
def model(gpu_device):
    return build(gpu_device)


def test_model_in_4_bits(gpu_device, model):
    """The same model on the values that the codes stand for, its products in fp32."""
    def values(name, t):
        if not (name.endswith("_proj.weight") or name == "lm_head.weight"):
            return t
        w = serve.quantise_q4_gpu(t.contiguous(), decoder.Q4_GROUP)
        v = oracle.q4_values(w.codes.cpu().numpy(), f64(w.scales), w.zeros.cpu().numpy())
        return torch.from_numpy(v.astype(np.float32)).to(t)   # a code of 4 bits times a scale of 8: exact

    q4, want = build(gpu_device, "q4"), build(gpu_device, change=values)
    assert near(q4.generate(PROMPTS), want.generate(PROMPTS), FP32)
    ids, logits = q4.generate_decode(PROMPTS, 5, eos=-1)
    want_ids, want_logits = want.generate_decode(PROMPTS, 5, eos=-1)
    assert ids == want_ids and near(logits, want_logits, FP32)
    assert not near(logits, model.generate_decode(PROMPTS, 5, eos=-1)[1], FP32)
    with pytest.raises(ValueError, match="tc is"):
        build(gpu_device, "q5")


def test_generate_decode_with_logprobs(gpu_device, model):
    kw = dict(repetition=1.3, bias={3: 2.0, 9: -4.0}, eos=-1)
    ids, logits = model.generate_decode(PROMPTS, 4, **kw)
    ids2, logits2, r = model.generate_decode(PROMPTS, 4, logprobs=6, **kw)
    assert ids2 == ids and torch.equal(logits2, logits)
    assert r.logprobs.shape == r.entropy.shape == (3, 4) and r.top_ids.shape == r.top_logprobs.shape == (3, 4, 6)
    want = oracle.logprobs(f64(logits).reshape(-1, V), np.array(ids).reshape(-1, 1), 6)
    oracle.assert_within(f64(r.logprobs).reshape(-1, 1), want["logprobs"], want["logprobs_tol"])
    oracle.assert_within(f64(r.entropy).reshape(-1), want["entropy"], want["entropy_tol"])
    assert np.array_equal(r.top_ids.cpu().numpy().reshape(-1, 6), want["top_ids"])
    assert r.top_ids[..., 0].tolist() == ids           # greedy: the likeliest, of equal logits the lowest id
    assert torch.equal(r.top_logprobs[..., 0], r.logprobs)
    none = model.generate_decode(PROMPTS, 2, logprobs=0, **kw)[2]
    assert none.top_ids.shape == (3, 2, 0) and torch.equal(none.logprobs, r.logprobs[:, :2])
    for bad in (-1, 65):
        with pytest.raises(ValueError, match="logprobs"):
            model.generate_decode(PROMPTS, 2, logprobs=bad, **kw)


@pytest.mark.parametrize("tc", ["off", "q4"])
def test_score(gpu_device, model, tc):
    m = model if tc == "off" else build(gpu_device, "q4")
    got = m.score(PROMPTS, top=4)
    assert [r.logprobs.shape[0] for r in got] == [4, 39, 0]
    for p, r in zip(PROMPTS[:2], got):
        for i in (0, len(p) // 2, len(p) - 2):
            x = f64(m.prefill(decoder.RowPlan.packed([p[:i + 1]], gpu_device)))
            want = oracle.logprobs(x, np.array([[p[i + 1]]]), 4)
            # logits near each other by FP32 of their norm, and so is what follows from them
            far = 4 * FP32 * np.linalg.norm(x)
            assert abs(float(r.logprobs[i]) - want["logprobs"][0, 0]) <= far + want["logprobs_tol"][0, 0]
            assert abs(float(r.entropy[i]) - want["entropy"][0]) <= far * (1 + np.abs(x).max()) + want["entropy_tol"][0]
            assert np.abs(f64(r.top_logprobs[i]) - want["top_logprobs"][0]).max() <= far + want["top_logprobs_tol"].max()
    assert m.score([[3]])[0].logprobs.shape == (0,)
    for bad, error in (([], RuntimeError), ([[1], []], ValueError), ([[V]], ValueError), ([[-1, 2]], ValueError)):
        with pytest.raises(error):
            m.score(bad)
    with pytest.raises(ValueError, match="top"):
        m.score(PROMPTS, top=65)


def test_step_in_4_bits_on_another_stream(gpu_device):
    """Two decodes side by side give what each gives alone."""
    m = build(gpu_device, "q4")
    want = [m.generate_decode([p], 4, eos=-1, logprobs=3) for p in PROMPTS[:2]]
    side, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for p, st in zip(PROMPTS[:2], side):
        with torch.cuda.stream(st):
            got.append(m.generate_decode([p], 4, eos=-1, logprobs=3))
    torch.cuda.synchronize()
    for (ids, x, r), (wids, wx, wr) in zip(got, want):
        assert ids == wids and torch.equal(x, wx) and all(torch.equal(a, b) for a, b in zip(r, wr))
