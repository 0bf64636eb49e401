"""CPU: what the Python calls of the paged cache refuse before the library is
reached, and what importing the package costs."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_another_current_device_is_refused(monkeypatch):
    """The C entries launch on the current device: a cache elsewhere raises."""
    import torch
    from zlift_b200 import paged
    cache = object.__new__(paged.KVCache)                    # (the device number of CPU tensors is -1)
    cache.heads, cache.dim, cache.device, cache.type = 2, 8, -1, paged.BF16
    cache.softmax_scale = 1.0
    x = torch.zeros(3, 2, 8, dtype=torch.bfloat16)
    q = torch.zeros(3, 4, 8, dtype=torch.bfloat16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)      # noqa: E731
    table = torch.zeros(1, 2, dtype=torch.int32)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(ValueError, match="current device"):
        paged.kv_write(cache, x, x, i32(0, 1, 2))
    with pytest.raises(ValueError, match="current device"):
        paged.kv_read(cache, x, x, table, i32(0, 3))
    with pytest.raises(ValueError, match="current device"):
        paged.paged_attention(cache, q, q.clone(), None, table, i32(0, 3), i32(5), 3)


def test_the_package_imports_without_torch():
    """`import *` and the calls on plain pointers need no torch; the paged
    calls are there by name where it is."""
    code = ("import sys; sys.modules['torch'] = None\n"
            "from zlift_b200 import *\n"
            "assert Handle and flash_forward and load and 'kv_write' not in globals()\n")
    subprocess.run([sys.executable, "-c", code], cwd=ROOT, check=True)
    import zlift_b200
    from zlift_b200 import KVCache, kv_read, kv_write, paged, paged_attention
    assert zlift_b200.KVCache is KVCache is paged.KVCache
    assert (kv_write, kv_read, paged_attention) == (paged.kv_write, paged.kv_read, paged.paged_attention)
