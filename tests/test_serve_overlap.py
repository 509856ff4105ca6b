"""Outputs of the serving operators that overlap other arrays of a call are
refused, and slices of one wider row, which only lie between each other, are
not.  No call here reaches the device: where the arrays are apart, a later check
refuses a misaligned one."""
import ctypes

import numpy as np
import pytest

from aps2026_amd import capi

P = 1 << 20   # an address that is never read
BF16, ARG = capi.DTYPE_BF16, capi.APS_ERR_ARG


def cache(k=P << 10, v=P << 11, **kw):
    d = dict(k_scale=None, v_scale=None, num_pages=8, page_size=16, kv_heads=1, head_dim=64, dtype=BF16)
    d.update(kw)
    return ctypes.byref(capi.KvCacheDesc(k, v, *[d[n] for n, _ in capi.KvCacheDesc._fields_[2:]]))


def append(rows, q, qs, q_out, os, k, ks, v, vs, q_heads=2, c=None):
    """True if refused for an overlap (slots off their alignment end any other call)."""
    rc = capi.lib().aps_kv_append(c if c is not None else cache(), k, ks, v, vs, q, qs, q_out, os, BF16, rows, q_heads,
                                  P, P + 4, P, P, 4, None)
    assert rc == ARG
    message = capi.last_error()
    assert ("overlap" in message) != ("aligned" in message)
    return "overlap" in message


def test_append():
    far = 1 << 40
    row = 256                                             # q 128, k 64, v 64 values of 2 bytes
    fused = dict(q=P, qs=row, k=P + 256, ks=row, v=P + 384, vs=row)
    assert not append(9, q_out=far, os=128, **fused)
    assert not append(9, q_out=P, os=row, **fused)        # in place
    assert append(9, q_out=P + 2, os=row, **fused)        # shifted by a value
    assert append(9, q_out=P + 2 * row, os=row, **fused)  # by a row
    assert append(9, q_out=P + 256, os=row, **fused)      # over k
    assert append(9, q_out=P - 4 * row, os=row, **fused)
    assert not append(9, q_out=P - 2 * 9 * row, os=row, **fused)
    assert not append(9, q_out=P - 2 * 9 * row + 256, os=row, **fused)   # its last row ends where q begins
    assert append(9, q_out=P - 2 * 9 * row + 258, os=row, **fused)
    assert not append(9, q_out=P + 2 * 9 * row, os=row, **fused)
    assert not append(9, q_out=P + 512, os=2 * row, q=P, qs=2 * row, k=P + 256, ks=2 * row, v=P + 384, vs=2 * row)
    assert append(9, q_out=P + 130, os=128, **fused)      # other strides
    assert append(1, q_out=P + 254, os=row, **fused)
    assert not append(1, q_out=P + 512, os=row, **fused)


def test_append_over_the_cache():
    held = 8 * 16 * 64
    apart = dict(q=P, qs=128, k=P << 1, ks=64, v=P << 2, vs=64)
    for at, size, kw in ((P << 10, 2 * held, {}), (P << 11, 2 * held, {}),
                         (P << 10, held // 2, dict(dtype=capi.KV_MXFP4, k_scale=P << 12, v_scale=P << 13))):
        for to, hit in ((at, True), (at + size - 2, True), (at + size, False), (at - 5 * 256, False),
                        (at - 5 * 256 + 2, True)):
            assert append(5, q_out=to, os=128, c=cache(**kw), **apart) is hit


@pytest.mark.parametrize("seed", range(4))
def test_append_as_sets_of_bytes(seed):
    """Random rows and strides against the bytes themselves."""
    rng = np.random.default_rng(seed)
    found = set()
    for _ in range(1500):
        rows, base = int(rng.integers(1, 7)), P
        widths = {"q": 128, "q_out": 128, "k": 64, "v": 64}
        stride = {n: w + int(rng.integers(0, 400)) for n, w in widths.items()}
        if rng.random() < 0.7:
            stride = {n: max(stride.values()) for n in widths}
        at = {n: base + 2 * int(rng.integers(0, 2600)) for n in widths}
        if at["q"] == at["q_out"] and stride["q"] != stride["q_out"]:
            continue
        span = {n: {b for r in range(rows) for b in range(at[n] + 2 * r * stride[n], at[n] + 2 * (r * stride[n] + w))}
                for n, w in widths.items()}
        want = any(span["q_out"] & span[n] for n in ("k", "v"))
        want |= at["q"] != at["q_out"] and bool(span["q_out"] & span["q"])
        got = append(rows, at["q"], stride["q"], at["q_out"], stride["q_out"], at["k"], stride["k"], at["v"], stride["v"])
        assert got is want, (rows, at, stride)
        found.add(want)
    assert found == {True, False}


def test_gather():
    held = 8 * 16 * 64 * 2
    size = 5 * 64 * 4

    def gather(k_out, v_out):
        assert capi.lib().aps_kv_gather(cache(), P + 4, 5, k_out, v_out, capi.DTYPE_F32, None) == ARG
        message = capi.last_error()
        assert ("overlap" in message) != ("aligned" in message)
        return "overlap" in message

    assert not gather(P, 2 * P) and not gather(P, None) and not gather(None, P) and not gather(P, P + size)
    assert gather(P, P) and gather(P, P + size - 16) and gather(P + size - 16, P)
    for at in (P << 10, P << 11):
        assert gather(at, None) and gather(P, at + held - 16) and gather(at - size + 16, P)
        assert not gather(at + held, None) and not gather(P, at - size)


def logits(rows, x, xs, out, os, vocab=100):
    """True if refused for an overlap (a misaligned list of lengths ends any other call)."""
    r = capi.LogitsRules(history=P, history_lens=P + 2, history_stride=4)
    assert capi.lib().aps_logits_process(x, xs, BF16, rows, vocab, ctypes.byref(r), out, os, None) == ARG
    message = capi.last_error()
    assert ("overlap" in message) != ("aligned" in message)
    return "overlap" in message


def test_logits():
    assert not logits(6, P, 100, P, 100) and not logits(6, P, 130, P, 130)           # in place
    assert logits(6, P, 100, P + 2, 100) and logits(6, P + 2, 100, P, 100)           # shifted by a logit
    assert logits(6, P, 130, P + 260, 130)                                           # by a row
    assert not logits(6, P, 230, P + 200, 230) and logits(6, P, 230, P + 198, 230)   # beside each other in a row
    assert not logits(6, P, 100, P + 1200, 100) and logits(6, P, 100, P + 1198, 100)
    assert logits(1, P, 100, P + 198, 100) and not logits(1, P, 100, P + 200, 100)
    assert logits(6, P, 100, P + 600, 300) and not logits(6, P, 100, P + 1200, 300)  # other strides


def test_logits_as_sets_of_bytes():
    rng = np.random.default_rng(5)
    found = set()
    for _ in range(2000):
        rows, vocab = int(rng.integers(1, 7)), 40
        xs, os = (vocab + int(rng.integers(0, 90)) for _ in range(2))
        if rng.random() < 0.7:
            os = xs
        x, out = (P + 2 * int(rng.integers(0, 900)) for _ in range(2))
        if x == out:
            continue
        spans = [{b for r in range(rows) for b in range(at + 2 * r * st, at + 2 * (r * st + vocab))}
                 for at, st in ((x, xs), (out, os))]
        want = bool(spans[0] & spans[1])
        assert logits(rows, x, xs, out, os, vocab) is want, (rows, x - P, xs, out - P, os)
        found.add(want)
    assert found == {True, False}
