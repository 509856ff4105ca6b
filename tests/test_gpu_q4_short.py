"""4-bit linear layers with fewer inputs than the 256 of a wave's turn
(include/aps_decode.h): an output takes its own scales and no others."""
import math

import numpy as np
import pytest
import torch

from aps2026_amd import serve
from tests import decode_oracle as oracle

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def f64(t):
    return t.detach().cpu().double().numpy()


def fill_lds_with_nan(dev):
    """Leaves NaN in most of every CU's LDS: 16 rows of x of 8 KB each lie there."""
    w = serve.Q4Weight(torch.zeros(8192, 2048, dtype=torch.uint8, device=dev), torch.ones(8192, 32, device=dev))
    serve.linear_q4_gpu(torch.full((16, 4096), math.nan, dtype=torch.bfloat16, device=dev), w)


SHORT = [(32, 32), (64, 32), (96, 32), (224, 32), (64, 64), (192, 64), (128, 128)]   # inputs, group
# one launch, narrow and not; many rows by 16 x 16 tiles and by larger ones; waves that share x
ROWS = [("f32", 1, 37), ("f32", 5, 300), ("bf16", 3, 37), ("bf16", 12, 4200), ("f32", 7, 33), ("f32", 40, 70),
        ("bf16", 20, 8200), ("bf16", 70, 8300), ("f32", 9, 16400)]


@pytest.mark.parametrize("k,group", SHORT)
@pytest.mark.parametrize("dtype,rows,n", ROWS)
@pytest.mark.parametrize("scales,zeros", [("f32", True), ("bf16", False)])
def test_scales_of_other_outputs_do_not_matter(gpu_device, k, group, dtype, rows, n, scales, zeros):
    print(f"[gpu-case] short {dtype} {rows} x {k} -> {n} group {group} {scales}", flush=True)
    dev, rng = gpu_device, np.random.default_rng(n + k)
    per = k // group
    codes = rng.integers(0, 256, (n, k // 2), dtype=np.uint8)
    s = torch.from_numpy(rng.uniform(0.005, 0.02, (n, per)).astype(np.float32)).to(dev, TYPES[scales])
    z = torch.from_numpy(rng.integers(0, 16, (n, per), dtype=np.uint8)).to(dev) if zeros else None
    x = torch.from_numpy(rng.standard_normal((rows, k)).astype(np.float32)).to(dev, TYPES[dtype])
    code = torch.from_numpy(codes).to(dev)
    fill_lds_with_nan(dev)
    plain = serve.linear_q4_gpu(x, serve.Q4Weight(code, s, z))
    want, bound = oracle.linear_q4(f64(x), codes, f64(s), z.cpu().numpy() if zeros else None, None)
    if dtype == "bf16":
        bound = bound + oracle.HALF_STEP["bf16"] * (np.abs(want) + bound)
    oracle.assert_within(f64(plain), want, bound)
    for value in (math.nan, math.inf):
        bad = s.clone()
        at = [3, n // 2, n - 1]
        bad[at, 0] = value
        fill_lds_with_nan(dev)
        got = serve.linear_q4_gpu(x, serve.Q4Weight(code, bad, z))
        keep = torch.ones(n, dtype=torch.bool, device=dev)
        keep[at] = False
        assert torch.equal(got[:, keep], plain[:, keep])
        assert not bool(got[:, at].isfinite().any())


def test_a_quantised_row_that_is_not_finite_stays_alone(gpu_device):
    w = torch.randn(20, 64, device=gpu_device)
    clean = serve.quantise_q4_gpu(w, 32)
    w[11, 40] = math.nan
    dirty, x = serve.quantise_q4_gpu(w, 32), torch.randn(6, 64, device=gpu_device)
    for rows in (1, 6):
        a, b = serve.linear_q4_gpu(x[:rows], clean), serve.linear_q4_gpu(x[:rows], dirty)
        assert bool(b[:, 11].isnan().all())
        keep = torch.arange(20, device=gpu_device) != 11
        assert torch.equal(a[:, keep], b[:, keep])
