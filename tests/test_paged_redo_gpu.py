"""Rows that a hidden key has spoilt are computed again, on the GPU: however
long that takes, no other part of the kernel may run out of time over it, and
rows that are NaN by right are not among them."""
import math

import pytest

from tests.test_paged_gpu import Case
from tests.test_paged_ranges_gpu import exact

pytestmark = pytest.mark.gpu


def close(o, lse, want, rows):
    wo, wl, to, tl = want
    return bool(((o[rows].double() - wo[rows]).abs() <= to[rows]).all()) and \
        bool(((lse[:, rows].double() - wl[:, rows]).abs() <= tl[:, rows]).all())


@pytest.mark.parametrize("held", ["same", "int8"])
def test_redone_rows_keep_nobody_waiting(cuda, held):
    """NaN in the newest token's V, a long context, and a limit on waits far
    below the time that the spoilt rows take."""
    import torch
    from zlift_b200 import blas, load, paged
    c = Case("bf16", held, new=(100, 40), ctx=(20000, 90), heads=8, kv_heads=2, dim=128, page=64, seed=3)
    want = exact(c)
    v = c.v_in.clone()
    v[19999] = math.nan
    assert paged.kv_write(c.cache, c.k_in, v, c.slots) == 0
    torch.cuda.synchronize()
    lib = load()
    default = lib.zlift_get_wait_limit_ns()
    try:
        assert lib.zlift_set_wait_limit_ns(10_000_000) == 0          # 10 ms
        o, lse = c.run()
        torch.cuda.synchronize()
        assert blas.device_error() == 0
    finally:
        assert lib.zlift_set_wait_limit_ns(default) == 0
    assert torch.isnan(o[99].float()).all()
    rows = [i for i in range(140) if i != 99]
    assert close(o, lse, want, rows)


@pytest.mark.parametrize("elem,held", [("bf16", "same"), ("f16", "same"), ("bf16", "int8"), ("f16", "fp8")])
@pytest.mark.parametrize("new", [1, 5, 150])
@pytest.mark.parametrize("which", ["k", "v", "kv"])
def test_a_sequence_that_is_nan_by_right(cuda, elem, held, new, which):
    """A cached token of NaN: every query of its sequence sees it, the other
    sequence's none."""
    import torch
    from zlift_b200 import blas, paged
    c = Case(elem, held, new=(new, new), ctx=(new + 700, new + 300), heads=8, kv_heads=2, dim=128, seed=7)
    want = exact(c)
    k, v = c.k_in.clone(), c.v_in.clone()
    if "k" in which:
        k[11, :, 5] = math.nan
    if "v" in which:
        v[11, :, 5] = math.nan
    assert paged.kv_write(c.cache, k, v, c.slots) == 0
    o, lse = c.run()
    torch.cuda.synchronize()
    assert blas.device_error() == 0
    assert close(o, lse, want, list(range(new, 2 * new)))
    if "k" in which:
        assert torch.isnan(o[:new].float()).all() and torch.isnan(lse[:, :new]).all()
    else:
        assert torch.isnan(o[:new, :, 5].float()).all()
        if held == "same":                                   # the other columns are as they were
            wo, wl, to, tl = want
            cols = [i for i in range(128) if i != 5]
            assert ((o[:new][:, :, cols].double() - wo[:new][:, :, cols]).abs() <= to[:new][:, :, cols]).all()
        else:
            assert torch.isnan(o[:new].float()).all()
        assert ((lse[:, :new].double() - want[1][:, :new]).abs() <= want[3][:, :new]).all()
