"""What the serving path keeps between calls, on the CPU."""
import gc
import weakref

import torch

from aps2026_amd import attention


def test_outgrown_rotation_tables_stay():
    """A call that is longer than the ones before takes a larger table; the
    smaller ones may still be read, by another stream or a recorded graph."""
    dev, theta = torch.device("cpu"), 4321.0
    first = attention._device_table(dev, 9, 64, theta)
    want = [t.clone() for t in first]
    held = [weakref.ref(t) for t in first]
    del first
    sizes = set()
    for n in range(9, 400):
        c, s = attention._device_table(dev, n, 64, theta)
        assert c.shape == s.shape and c.shape[0] >= n
        sizes.add(c.shape[0])
    gc.collect()
    assert all(r() is not None for r in held)
    assert len(sizes) <= 7                                  # doubled, not grown by every call
    assert torch.equal(c[:9], want[0]) and torch.equal(s[:9], want[1])
    assert all(torch.equal(r(), w) for r, w in zip(held, want))
    attention._tables.pop((dev, 64, theta))
