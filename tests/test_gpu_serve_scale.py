"""Attention at scales of either sign and none, on both kernels."""
import math

import numpy as np
import pytest
import torch

from tests import serve_oracle as oracle
from tests.test_gpu_serve import BF16, F32, Case, f64, held, note

pytestmark = pytest.mark.gpu

TYPES = [(F32, "f32"), (F32, "bf16"), (F32, "mxfp4"), (BF16, "bf16"), (BF16, "mxfp4")]


def spoil(c, b, j):
    """Makes the value of position j of sequence b one that is not finite; returns what puts 1 there."""
    page, off = c.table[b, j // c.page], j % c.page
    if c.cache.v_scale is not None:
        c.cache.v_scale[page, :, off] = 255
        return lambda: c.cache.v_scale[page, :, off].fill_(127)
    c.cache.v[page, :, off] = float("inf")
    return lambda: c.cache.v[page, :, off].fill_(1.0)


def exact(c, window, sinks, scale):
    """(outputs, bound): the magnitude of the scores' products is that of |scale|."""
    want, mag, prod, seen = oracle.attention(
        f64(c.q).reshape(c.rows, c.qh, c.dim), *held(c.cache), c.offs, c.kv_lens, c.table, c.page, c.qh, window, sinks,
        scale, c.pages)
    bound = oracle.attention_bound(want, mag, np.abs(prod), seen, c.dim, c.qt, 24 if c.qt is F32 else 8)
    assert (bound > 0).all()
    return want, bound


@pytest.mark.parametrize("qt,kind", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("scale", [-0.5, 0.0, 3.0])
@pytest.mark.parametrize("q_lens,kv_lens", [([2, 1], [40, 70]), ([40, 33], [90, 200]), ([45, 1, 2], [300, 90, 130])])
def test_scales(gpu_device, qt, kind, dim, scale, q_lens, kv_lens):
    """Rows of one tile, blocks of many and both at once; no key, or one with a
    value that is not finite, which the last token of the first sequence alone
    sees: the rows beside it are computed again at that scale too."""
    note(f"scale {scale} {qt} {kind} {dim} {q_lens}")
    c = Case(gpu_device, qt, kind, 4, 2, dim, 16, q_lens, kv_lens, seed=41)
    for window, sinks in ((1 << 30, 0), (50, 3)):
        want, bound = exact(c, window, sinks, scale)
        got = f64(c.run(window, sinks, scale=scale)).reshape(want.shape)
        worst = (np.abs(got - want) / bound).max()
        note(f"  worst {worst:.3f} of the bound")
        assert worst <= 1.0
    last = c.offs[1] - 1
    mend = spoil(c, 0, kv_lens[0] - 1)
    got = f64(c.run(50, 3, scale=scale)).reshape(c.rows, 4, dim)
    mend()
    want, bound = exact(c, 50, 3, scale)
    assert not np.isfinite(got[last]).any()
    rest = np.arange(c.rows) != last
    assert (np.abs(got - want) <= bound)[rest].all()


@pytest.mark.parametrize("q_lens,kv_lens", [([2, 1], [40, 70]), ([40, 33], [90, 200])])
def test_outputs_of_another_scale_fail(gpu_device, q_lens, kv_lens):
    """The bound tells outputs of another scale, and none at all, from the right ones."""
    c = Case(gpu_device, F32, "bf16", 4, 2, 64, 16, q_lens, kv_lens, seed=4)
    want, bound = exact(c, 50, 3, -0.5)
    for got in (c.run(50, 3, scale=0.5), torch.zeros_like(c.q), c.run(50, 3, scale=-0.5) + 1e-2):
        assert (np.abs(f64(got).reshape(want.shape) - want) > bound).mean() > 0.5
    assert math.isfinite(bound.max())


@pytest.mark.parametrize("qt,kind", TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("q_lens,kv_lens", [([2, 1], [40, 70]), ([40, 33], [90, 200])])
def test_queries_that_are_not_finite_at_no_scale(gpu_device, qt, kind, value, q_lens, kv_lens):
    """0 times NaN or an infinity is NaN, also where every score is 0."""
    note(f"no scale {qt} {kind} {value} {q_lens}")
    c = Case(gpu_device, qt, kind, 4, 2, 64, 16, q_lens, kv_lens, seed=5)
    want, bound = exact(c, 50, 3, 0.0)
    c.q[1, 64 + 7] = value                     # row 1, head 1
    got = f64(c.run(50, 3, scale=0.0)).reshape(want.shape)
    assert np.isnan(got[1, 1]).all()
    rest = np.ones(want.shape[:2], bool)
    rest[1, 1] = False
    assert (np.abs(got - want) <= bound)[rest].all()
