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
