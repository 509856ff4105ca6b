"""Row gathers, elementwise operations and row quantisation (include/aps_moe.h) past
what one launch's grid holds: 2^32 threads."""
import ctypes

import torch

from aps2026_amd import capi
from tests.test_gpu_decode_launches import BF16, F32, _free_memory, assert_repeats, note, pytestmark, repeated  # noqa: F401


def call(name, *args):
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    rc = getattr(capi.lib(), name)(*[ctypes.c_void_p(a.data_ptr()) if torch.is_tensor(a) else a for a in args], stream)
    assert rc == 0, capi.last_error()


def test_gather_of_many_rows(gpu_device):
    count = (1 << 24) + 9
    note(f"gather of {count} rows")
    x = torch.randn(1013, 4, device=gpu_device)
    at = torch.randperm(1013, device=gpu_device).to(torch.int32)
    for width in (4, 3):                       # in 16 bytes, and a value at a time
        few = x[:, :width].contiguous()
        out = torch.empty(count, width, device=gpu_device)
        call("aps_gather_rows", few, 1013, width, repeated(at, count), count, out)
        assert_repeats(out, few[at.long()])


def test_elementwise_of_many_values(gpu_device):
    """Arrays off 16 bytes, where a thread has one value."""
    n, h = (1 << 32) + 12, 4
    note(f"elementwise of {n} values")
    a, b = (torch.empty(n + 1, device=gpu_device)[1:] for _ in range(2))
    bias = torch.arange(1, h + 1, dtype=F32, device=gpu_device)
    rows = lambda t: t.view(-1, h)  # noqa: E731
    for t, scale in ((a, 1.0), (b, 3.0)):
        t.fill_(7.0)
        call("aps_zero", t, n)
        call("aps_add_bias_inplace", t, scale * bias, n, h)
        assert_repeats(rows(t), scale * bias[None])
    call("aps_add_inplace", a, b, n)
    assert_repeats(rows(a), 4 * bias[None])
    few = torch.empty(h + 1, device=gpu_device)[1:]
    call("aps_silu_mul", (4 * bias).contiguous(), (3 * bias).contiguous(), few, h)
    out = torch.empty(n + 1, device=gpu_device)[1:]
    call("aps_silu_mul", a, b, out, n)
    assert_repeats(rows(out), few[None])


def test_quantise_rows_of_many_rows(gpu_device):
    rows = (1 << 26) + 3
    note(f"quantise_rows_e4m3 of {rows} rows")
    few = torch.randn(1009, 16, device=gpu_device).to(BF16)

    def quantised(x):
        out, scale = torch.empty(len(x), 16, dtype=torch.uint8, device=gpu_device), torch.empty(len(x), 1, device=gpu_device)
        call("aps_quantise_rows_e4m3", x, 16, 16, out, 16, scale, len(x))
        return out, scale

    for got, want in zip(quantised(repeated(few, rows)), quantised(few)):
        assert_repeats(got, want)
