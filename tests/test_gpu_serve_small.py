"""The smallest values that a 4-bit cache can be given."""
import numpy as np
import pytest
import torch

from aps2026_amd import serve
from tests import serve_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
def test_blocks_of_values_below_the_normal_ones(gpu_device, dim):
    """Subnormal values against the oracle's codes and scales, byte for byte, and
    read back as what those stand for."""
    dev, rows = gpu_device, 16
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((rows, dim)) * np.exp2(rng.integers(-152, -118, (rows, 1)))).astype(np.float32)
    x[0], x[1, ::2], x[2] = 2.0 ** -127, 2.0 ** -149, -(2.0 ** -128)
    t = torch.from_numpy(x).to(dev)
    cache = serve.PagedKvCache.allocate(1, 16, 1, dim, "mxfp4", dev)
    table = torch.zeros(1, dim // 2, device=dev)
    slots = torch.arange(rows, device=dev)
    serve.kv_append_gpu(cache, t, t, torch.full((rows,), -1, dtype=torch.int32, device=dev), slots, table, table)
    codes, scales = oracle.mx_encode(x)
    for have, scale, got in zip((cache.k, cache.v), (cache.k_scale, cache.v_scale), serve.kv_gather_gpu(cache, slots)):
        assert np.array_equal(scale.cpu().numpy().reshape(rows, -1), scales)
        assert np.array_equal(have.cpu().numpy().reshape(rows, -1), codes)
        assert np.array_equal(got.cpu().numpy().astype(np.float64), oracle.mx_values(codes, scales))
