"""How many bits the attention kernels keep, against limits that one term fewer
fails (tests/serve_limits.py)."""
import math

import pytest
import torch

from tests import serve_limits as limits
from tests import serve_oracle as oracle
from tests.test_gpu_serve import BF16, F32, Case, f64, held, note
from tests.test_serve_limits import SHAPES

pytestmark = pytest.mark.gpu


def distances(c, window, sinks, parts, **kw):
    """The distance of each part (a list of sequences) of one call's outputs."""
    got = f64(c.run(window, sinks, **kw)).reshape(c.rows, c.qh, c.dim)
    want = oracle.attention(f64(c.q).reshape(c.rows, c.qh, c.dim), *held(c.cache), c.offs, c.kv_lens, c.table, c.page,
                            c.qh, window, sinks, 1 / math.sqrt(c.dim), c.pages)[0]
    out = []
    for part in parts:
        rows = [r for b in part for r in range(c.offs[b], c.offs[b + 1])]
        out.append(limits.distance(got[rows], want[rows], c.qt))
    note("  distances " + " ".join(f"{x:.2e}" for x in out))
    return out


@pytest.mark.parametrize("kind", ["bf16", "mxfp4"])
@pytest.mark.parametrize("q_lens,kv_lens,most", [
    ([90, 1, 90, 90] + [1] * 5, [400, 900, 90, 300, 130, 350, 800, 411, 202], 1),    # three prompts beside steps
    ([1, 70, 8, 70], [700, 70, 300, 350], 8),                                        # up to 8 tokens: 32 rows
    ([64, 64, 3], [64, 500, 1900], 3),                                               # keys of the steps are split
    ([64, 8, 64], [300, 400, 500], 8),                                               # the most rows that leave room for it
])
def test_steps_beside_prompts_keep_their_bits(gpu_device, kind, q_lens, kv_lens, most):
    """Weights of a sequence of up to 32 rows keep 16 bits whatever stands beside
    it; those of longer ones 8."""
    note(f"steps beside prompts {kind} {q_lens}")
    c = Case(gpu_device, BF16, kind, 8, 2, 128, 16, q_lens, kv_lens, seed=17)
    short = [b for b, n in enumerate(q_lens) if n <= most]
    few, many = distances(c, 1 << 30, 0, [short, [b for b in range(len(q_lens)) if b not in short]])
    assert few < limits.LIMIT[16]
    assert many < limits.LIMIT[8]
    c.check(c.run(1 << 30, 0), 1 << 30, 0)
    c.check(c.run(50, 3), 50, 3)


def test_rows_of_short_sequences_beside_prompts(gpu_device):
    """Their parts stand by sequence and token: rows before, between and behind
    the sequences are left alone, and more tokens than max_q_len too."""
    note("rows of short sequences beside prompts")
    c = Case(gpu_device, BF16, "bf16", 4, 1, 128, 16, [60, 0, 1, 60, 2, 0, 7], [1300, 50, 1900, 90, 1500, 0, 1700],
             extra_rows=6, seed=3)
    n = int(c.offs[-1])
    c.offs += 2
    out = torch.full((c.rows, 4 * 128), 3.0, dtype=BF16, device=gpu_device)
    c.run(1 << 30, 0, out=out)
    assert bool((out[:2] == 3.0).all()) and bool((out[2 + n:] == 3.0).all())
    c.q, c.offs, c.rows = c.q[2:2 + n].contiguous(), c.offs - 2, n
    c.check(out[2:2 + n], 1 << 30, 0)
    cut = torch.full((n, 4 * 128), 5.0, dtype=BF16, device=gpu_device)
    c.run(1 << 30, 0, out=cut, max_q_len=59)
    keep = [r for b in range(7) for r in range(c.offs[b], min(c.offs[b + 1], c.offs[b] + 59))]
    left = [r for r in range(n) if r not in keep]
    assert len(left) == 2 and bool((cut[left] == 5.0).all())
    c.check(torch.where(torch.isin(torch.arange(n, device=gpu_device), torch.tensor(keep, device=gpu_device))[:, None],
                        cut, out[2:2 + n]), 1 << 30, 0)


@pytest.mark.parametrize("qt,kind", [(F32, "f32"), (F32, "bf16"), (F32, "mxfp4"), (BF16, "bf16"), (BF16, "mxfp4")])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_lens,kv_lens", SHAPES + [([90, 33], [700, 1500])])
def test_bits_of_every_form(gpu_device, qt, kind, dim, q_lens, kv_lens):
    """Terms beside each other in the columns (4 rows, of bf16 queries 8), tiles of
    16 rows, blocks of 128 rows and keys that are split: 24 bits of fp32 queries
    and their weights, 16 of bf16 queries' weights and past 32 rows 8."""
    note(f"bits {qt} {kind} {dim} {q_lens}")
    c = Case(gpu_device, qt, kind, 4, 1, dim, 16, q_lens, kv_lens, seed=23)
    bits = 24 if qt is F32 else 16 if max(q_lens) <= 8 else 8
    assert distances(c, 1 << 30, 0, [range(len(q_lens))])[0] < limits.LIMIT[bits]
