"""More operators of the serving path, as cases that can be timed and compared.

What a decode step of a model with weights in 4 bits needs around the paged
cache, from its projections to what it says about the token it chose:

  rope      rotate q and k by their positions: the pairs of a head as halves or
            as neighbours, the whole head or its first dimensions, frequencies
            scaled for long contexts; forth and back
  linear    y = x W^T + b with W in 4 bits: codes 0..15, a scale and (or not) a
            zero for each group of neighbouring inputs
  logprobs  log probabilities of given tokens under rows of logits, the entropy
            of the row and its likeliest tokens

Shapes of the model that the repository runs: hidden 4096, 16 query and 4
key/value heads of 128, vocabulary 32064; others are generic.

A weight is codes [out][in / 2] (two to a byte, the even input in the low
half), scales [out][in / group] in fp32 or bf16 and zeros [out][in / group] as
bytes (none: 8): w = (code - zero) scale.

Nothing here depends on the number of cases; sizes go by the case alone and
values by the seed.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

HIDDEN, HEADS, KV_HEADS, DIM, VOCAB, THETA = 4096, 16, 4, 128, 32064, 10000.0
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2}
DEV = "cuda"


def _rope(rows, dtype="f32", q_heads=HEADS, kv_heads=KV_HEADS, dim=DIM, rotary=DIM, layout="half", scaling="none",
          factor=1.0, context=4096, run=1, fused=False, inverse=False):
    """run: tokens of one sequence that follow each other."""
    return {"family": "rope", "rows": rows, "dtype": dtype, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "rotary": rotary, "layout": layout, "scaling": scaling, "factor": factor, "context": context, "run": run,
            "fused": fused, "inverse": inverse}


def _linear(rows, n_in, n_out, dtype="f32", group=128, scales="bf16", zeros=True, bias=False):
    return {"family": "linear", "rows": rows, "in": n_in, "out": n_out, "dtype": dtype, "group": group,
            "scales": scales, "zeros": zeros, "bias": bias}


def _logprobs(rows, vocab=VOCAB, dtype="f32", tokens=1, top=5, masked=False, pad=0):
    """tokens: given ids of each row; pad: columns behind the vocabulary."""
    return {"family": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "tokens": tokens, "top": top,
            "masked": masked, "pad": pad}


def listed():
    return [
        # A decode step of one sequence: latency.
        {"name": "rope_one", **_rope(1)},
        # 16 prompts of 512 tokens; q and k are slices of one row, half of each head turns, neighbours are pairs.
        {"name": "rope_prompts", **_rope(16 * 512, "bf16", rotary=64, layout="pairs", run=512, fused=True)},
        # One long text past the length that the model was trained on.
        {"name": "rope_long", **_rope(65536, "bf16", scaling="parts", factor=16.0, context=65536, run=65536)},
        # The query projection of one token.
        {"name": "q4_one", **_linear(1, HIDDEN, HEADS * DIM, bias=True)},
        # The LM head for one token, groups of 64.
        {"name": "q4_head", **_linear(1, HIDDEN, VOCAB, "bf16", group=64)},
        # Five rows of a narrow model: sizes that fill no tile.
        {"name": "q4_ragged", **_linear(5, 1440, 1001, group=32, scales="f32", zeros=False, bias=True)},
        # A serving batch through the LM head.
        {"name": "q4_batch", **_linear(16, HIDDEN, VOCAB)},
        # A large batch through a wide layer.
        {"name": "q4_wide", **_linear(64, 8192, 8192, "bf16")},
        # A chunk of a prompt through the output projection.
        {"name": "q4_chunk", **_linear(256, HEADS * DIM, HIDDEN, "bf16", zeros=False, bias=True)},
        # The token that was chosen for one prompt, with alternatives: latency.
        {"name": "logprobs_one", **_logprobs(1, top=20)},
        # Every token of a set of prompts scored.
        {"name": "logprobs_prompts", **_logprobs(4096, dtype="f32", top=1)},
        # A serving batch under a grammar, some candidates a row, a padded vocabulary of another model.
        {"name": "logprobs_batch", **_logprobs(250, vocab=100003, dtype="bf16", tokens=4, top=20, masked=True, pad=5)},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    family = rng.choice(["rope", "linear", "linear", "logprobs"])
    dtype = rng.choice(["f32", "bf16"])
    if family == "rope":
        q_heads, kv_heads = rng.choice([(16, 4), (16, 4), (8, 8), (32, 8), (24, 2), (10, 2)])
        dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
        rotary = rng.choice([dim, dim, dim // 2, dim // 4, 2 * rng.randint(1, dim // 2)])
        most = 65536 * (HEADS + KV_HEADS) * DIM // ((q_heads + kv_heads) * dim) // BYTES[dtype]
        rows = rng.choice([_log_int(rng, 1, 256), _log_int(rng, 1, most)])
        scaling = rng.choice(["none", "linear", "base", "parts"]) if rotary > 2 else "none"
        return _rope(rows, dtype, q_heads, kv_heads, dim, rotary, rng.choice(["half", "pairs"]), scaling,
                     1.0 if scaling == "none" else rng.uniform(1.5, 32.0), _log_int(rng, 64, 1 << 20),
                     rng.choice([1, _log_int(rng, 1, rows)]), rng.random() < 0.5, rng.random() < 0.3)
    if family == "linear":
        group = rng.choice([32, 64, 128, 128])
        rows = rng.choice([1, rng.randint(1, 16), _log_int(rng, 1, 64), _log_int(rng, 1, 256)])
        n_in = group * _log_int(rng, 1, 16384 // group)
        most = min(VOCAB, HIDDEN * VOCAB // n_in, 64 * 8192 * 8192 // (rows * n_in))
        n_out = _log_int(rng, min(64, most), most)
        return _linear(rows, n_in, n_out, dtype, group, rng.choice(["bf16", "f32"]), rng.random() < 0.6,
                       rng.random() < 0.5)
    vocab = rng.choice([VOCAB, _log_int(rng, 500, 160000)])
    rows = rng.choice([_log_int(rng, 1, 64), _log_int(rng, 1, max(1, 4096 * VOCAB // vocab * 2 // BYTES[dtype] // 2))])
    return _logprobs(rows, vocab, dtype, rng.choice([1, 1, 1, rng.randint(2, 16)]), rng.choice([0, 1, 5, 20, 50]),
                     rng.random() < 0.3, rng.choice([0, 0, rng.randint(1, 100)]))


def _frequencies(case):
    """Angles per position [rotary / 2] in 64 bits, and the factor on cos and sin."""
    d, factor = case["rotary"], case["factor"]
    i = np.arange(d // 2)
    if case["scaling"] == "base":      # a larger base: the slowest pair turns `factor` times slower
        return (THETA * factor ** (d / (d - 2))) ** (-2.0 * i / d), 1.0
    freq = THETA ** (-2.0 * i / d)
    if case["scaling"] == "linear":
        return freq / factor, 1.0
    if case["scaling"] == "parts":     # pairs with over 32 turns in the trained length stay, those below one are slowed
        keep = np.clip((4096 * freq / (2 * math.pi) - 1) / (32 - 1), 0.0, 1.0)
        return freq * (keep + (1 - keep) / factor), 1.0 + 0.1 * math.log(factor)
    return freq, 1.0


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=g, device=DEV)  # noqa: E731
    rand = lambda *shape: torch.rand(shape, generator=g, device=DEV)  # noqa: E731
    dtype, rows = TYPES[case["dtype"]], case["rows"]
    s = {"case": case}
    if case["family"] == "rope":
        freq, s["amplitude"] = _frequencies(case)
        s["freq"] = torch.from_numpy(freq).to(DEV)
        run = case["run"]
        first = np.random.default_rng(seed).integers(0, max(1, case["context"] - run + 1), -(-rows // run))
        at = np.arange(rows)
        s["positions"] = torch.from_numpy((first[at // run] + at % run).astype(np.int32)).to(DEV)
        q, k = case["q_heads"] * case["dim"], case["kv_heads"] * case["dim"]
        if case["fused"]:  # q, k and v of a token side by side, as one projection writes them
            s["q"], s["k"], _ = randn(rows, q + 2 * k).to(dtype).split([q, k, k], 1)
        else:
            s["q"], s["k"] = randn(rows, q).to(dtype), randn(rows, k).to(dtype)
    elif case["family"] == "linear":
        n, k, groups = case["out"], case["in"], case["in"] // case["group"]
        code = (8 + 2.6 * randn(n, k)).round_().clamp_(0, 15).to(torch.uint8)
        s["codes"] = code[:, 0::2] | code[:, 1::2] << 4
        del code
        s["scales"] = (0.01 * (0.5 + rand(n, groups))).to(TYPES[case["scales"]])
        s["zeros"] = (8 + 1.5 * randn(n, groups)).round_().clamp_(0, 15).to(torch.uint8) if case["zeros"] else None
        s["bias"] = 0.1 * randn(n) if case["bias"] else None
        s["x"] = randn(rows, k).to(dtype)
    else:
        vocab = case["vocab"]
        # a few likely tokens over a broad rest
        x = 2 * randn(rows, vocab + case["pad"]) + 9 * rand(rows, vocab + case["pad"]) ** 24
        if case["masked"]:  # a grammar lets some of the tokens through, in some rows but a handful
            keep = torch.where(torch.arange(rows, device=DEV)[:, None] % 2 == 0, 20.0 / vocab, 0.7)
            x.masked_fill_(rand(rows, vocab + case["pad"]) > keep, -math.inf)
            x[:, 0] = 0.0
        s["logits"] = x.to(dtype)[:, :vocab]
        s["tokens"] = (vocab * rand(rows, case["tokens"])).int().clamp(max=vocab - 1)
    return s


# ---- one pass ---------------------------------------------------------------

def run(s):
    return {"rope": _run_rope, "linear": _run_linear, "logprobs": _run_logprobs}[s["case"]["family"]](s)


def _run_rope(s):
    case = s["case"]
    dim, half = case["dim"], case["rotary"] // 2
    if own:
        from aps2026_amd import serve
        return serve.rope_gpu(s["q"], s["k"], s["positions"], s["freq"], head_dim=dim, layout=case["layout"],
                              amplitude=s["amplitude"], inverse=case["inverse"])
    angle = s["positions"].double()[:, None, None] * s["freq"]
    c, sn = angle.cos() * s["amplitude"], angle.sin() * s["amplitude"]
    if case["inverse"]:
        sn = -sn

    def turn(x):
        x = x.unflatten(1, (-1, dim))
        a = x[..., :2 * half].double()
        x0, x1 = (a[..., :half], a[..., half:]) if case["layout"] == "half" else (a[..., 0::2], a[..., 1::2])
        y0, y1 = x0 * c - x1 * sn, x0 * sn + x1 * c
        y = torch.cat((y0, y1), -1) if case["layout"] == "half" else torch.stack((y0, y1), -1).flatten(-2)
        return torch.cat((y.to(x.dtype), x[..., 2 * half:]), -1).flatten(1)

    return turn(s["q"]), turn(s["k"])


def _run_linear(s):
    if own:
        from aps2026_amd import serve
        return serve.linear_q4_gpu(s["x"], serve.Q4Weight(s["codes"], s["scales"], s["zeros"]), bias=s["bias"])
    group = s["case"]["group"]
    code = torch.stack((s["codes"] & 15, s["codes"] >> 4), -1).flatten(-2).float().unflatten(1, (-1, group))
    code -= 8.0 if s["zeros"] is None else s["zeros"].float()[..., None]
    y = torch.matmul(s["x"].float(), (code * s["scales"].float()[..., None]).flatten(1).T)
    return (y if s["bias"] is None else y + s["bias"]).to(s["x"].dtype)


def _run_logprobs(s):
    case = s["case"]
    if own:
        from aps2026_amd import serve
        r = serve.token_logprobs_gpu(s["logits"], s["tokens"], top=case["top"])
        return {"logprobs": r.logprobs, "entropy": r.entropy, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs}
    x = s["logits"].float()
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    norm = top + total.log()
    rest = torch.where(e > 0, e * (top - x), 0.0)
    # order of the likeliest: by value, then by the lower index
    bits = (x + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32 | (0x7FFFFFFF - torch.arange(x.shape[1], device=DEV))
    ids = 0x7FFFFFFF - (torch.topk(key, case["top"], dim=1).values & 0x7FFFFFFF)
    return {"logprobs": x.gather(1, s["tokens"].long()) - norm, "entropy": (total.log() + rest.sum(1, keepdim=True) / total)[:, 0],
            "top_ids": ids.int(), "top_logprobs": x.gather(1, ids) - norm}


# ---- what a pass cannot do without -------------------------------------------

def work(case):
    rows, size = case["rows"], BYTES[case["dtype"]]
    if case["family"] == "rope":
        heads = case["q_heads"] + case["kv_heads"]
        return {"bytes": rows * (2 * heads * case["dim"] * size + 4) + 4 * case["rotary"],
                "flops": rows * 3 * heads * case["rotary"]}
    if case["family"] == "linear":
        n, k, groups = case["out"], case["in"], case["in"] // case["group"]
        held = n * k // 2 + n * groups * (BYTES[case["scales"]] + case["zeros"]) + 4 * n * case["bias"]
        return {"bytes": held + rows * (n + k) * size, "flops": 2 * rows * n * k}
    n = rows * case["vocab"]
    return {"bytes": n * size + rows * (8 * case["tokens"] + 8 * case["top"] + 4), "flops": 5 * n}


# ---- the definition in 64 bits -------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "linear": _exact_linear, "logprobs": _exact_logprobs}[case["family"]](case, s)


def _exact_rope(case, s):
    half, turns = case["rotary"] // 2, s["positions"].double()[:, None] * (s["freq"] / (2 * math.pi))
    by = torch.polar(torch.full_like(turns, s["amplitude"]), 2 * math.pi * (turns - turns.round()))[:, None]
    by = by.conj() if case["inverse"] else by

    def turned(x):
        out = x.double().reshape(case["rows"], -1, case["dim"])
        first = slice(0, half) if case["layout"] == "half" else slice(0, 2 * half, 2)
        second = slice(half, 2 * half) if case["layout"] == "half" else slice(1, 2 * half, 2)
        z = torch.complex(out[..., first].contiguous(), out[..., second].contiguous()) * by
        out[..., first], out[..., second] = z.real, z.imag
        return out.flatten(1)

    return turned(s["q"]), turned(s["k"])


def _exact_linear(case, s):
    # sum over groups of scale (x . code - zero sum x)
    rows, n, group = case["rows"], case["out"], case["group"]
    x = s["x"].double().reshape(rows, -1, group)
    y = torch.zeros(rows, n, dtype=torch.float64, device=DEV)
    for at in range(case["in"] // group):
        held = s["codes"][:, at * group // 2:(at + 1) * group // 2]
        dot = x[:, at, 0::2] @ (held % 16).double().T + x[:, at, 1::2] @ (held // 16).double().T
        zero = s["zeros"][:, at].double() if s["zeros"] is not None else torch.full((n,), 8.0, dtype=torch.float64, device=DEV)
        y += (dot - x[:, at].sum(1, keepdim=True) * zero) * s["scales"][:, at].double()
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_logprobs(case, s):
    out = {"logprobs": [], "entropy": [], "top_logprobs": []}
    for at in range(0, case["rows"], 256):
        p = torch.log_softmax(s["logits"][at:at + 256].double(), 1)
        out["logprobs"].append(p.gather(1, s["tokens"][at:at + 256].long()))
        out["entropy"].append(-(p.exp() * p.clamp(min=-1e300)).sum(1))
        out["top_logprobs"].append(p.sort(1, descending=True).values[:, :case["top"]])
    return {"top_ids": None, **{name: torch.cat(v) for name, v in out.items()}}
