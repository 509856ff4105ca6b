"""The limits on attention's distances (tests/serve_limits.py), on the CPU: they
pass the numbers of bits that the kernels state, and fail one term (8 bits of a
weight or a query) fewer."""
import ctypes
import math

import numpy as np
import pytest
import torch

from aps2026_amd import capi
from tests import serve_limits as limits
from tests import serve_oracle as oracle

SHAPES = [([1] * 6, [300, 513, 97, 800, 250, 411]), ([5, 2], [400, 333]), ([60], [200]), ([2, 1, 2], [1300, 900, 700])]


def batch(q_lens, kv_lens, dim, query_type, seed=3, page=16):
    rng = np.random.default_rng(seed)
    draw = lambda t, *shape: torch.from_numpy(rng.standard_normal(shape, dtype=np.float32)).to(t).double().numpy()  # noqa: E731
    counts = [-(-n // page) for n in kv_lens]
    first = np.cumsum([0] + counts)
    table = np.full((len(kv_lens), max(counts)), -1)
    for b, n in enumerate(counts):
        table[b, :n] = np.arange(first[b], first[b + 1])
    k, v = (draw(torch.bfloat16, first[-1], 1, page, dim) for _ in range(2))
    return (draw(query_type, sum(q_lens), 4, dim), k, v, np.concatenate([[0], np.cumsum(q_lens)]), kv_lens, table, page,
            4, 1 << 30, 0, 1 / math.sqrt(dim))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_lens,kv_lens", SHAPES)
@pytest.mark.parametrize("query_type,bits,fewer", [(torch.float32, (24, 24), [(24, 16), (16, 24)]),
                                                   (torch.bfloat16, (24, 16), [(24, 8)]),
                                                   (torch.bfloat16, (24, 8), [(24, 7)])])
def test_limits_tell_the_bits(dim, q_lens, kv_lens, query_type, bits, fewer):
    args = batch(q_lens, kv_lens, dim, query_type)
    want = oracle.attention(*args, num_pages=args[1].shape[0])[0]

    def distance(query_bits, weight_bits):
        out = torch.from_numpy(limits.attention(*args, query_bits, weight_bits)).to(query_type)
        return limits.distance(out.double().numpy(), want, query_type)

    assert distance(60, 60) < 1e-7                     # the two definitions agree
    assert distance(*bits) < limits.LIMIT[bits[1]]
    for less in fewer:
        assert distance(*less) > limits.LIMIT[bits[1]]


@pytest.mark.parametrize("scale", [2.4e38, -2.4e38, 3.4e38, float("inf"), float("-inf"), float("nan")])
def test_scales_without_a_base_2_form_are_refused(scale):
    """Scores are scaled by scale log2 e, which passes fp32's range from 2.36e38."""
    p = 1 << 20                                # no array is read
    cache = capi.KvCacheDesc(p, p, None, None, 8, 16, 4, 128, capi.DTYPE_BF16)
    # out lies over q, so that a call whose scale is taken is refused as well
    rc = capi.lib().aps_attention_paged(ctypes.byref(cache), p, 2048, capi.DTYPE_BF16, 4, 16, p, p, p, 4, 2, 1, 64, 64, 0,
                                        scale, p, None, 0, None)
    assert rc == capi.APS_ERR_ARG and "scale" in capi.last_error()


@pytest.mark.parametrize("kv_heads,max_q", [(2048, 1),    # 2^31 workgroups for 2^20 steps
                                            (1024, 40)])  # and for the short sequences beside chunks
def test_more_workgroups_than_a_launch_has_are_refused(kv_heads, max_q):
    """Before the first launch of the call: nothing is written."""
    p, L = 1 << 20, capi.lib()
    cache = capi.KvCacheDesc(p, p, None, None, 8, 16, kv_heads, 64, capi.DTYPE_BF16)
    sizes = (1 << 20, kv_heads)
    # out lies over q, so that a call whose sizes are taken is refused as well
    rc = L.aps_attention_paged(ctypes.byref(cache), p, kv_heads * 64, capi.DTYPE_BF16, *sizes, p, p, p, 4, 1 << 20, max_q,
                               64, 64, 0, 0.1, p, None, 0, None)
    assert rc == capi.APS_ERR_SHAPE and "workgroups" in capi.last_error()
    assert L.aps_attention_paged_workspace_size(ctypes.byref(cache), *sizes, 1 << 20, max_q, 64, 64, 0) == 0
