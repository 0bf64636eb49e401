"""Paged attention under a wait limit that ordinary waits may exceed, on the
GPU: a call either gives the right answer or reports error 1, and ends by
itself either way; with the default limit and a fresh workspace the next one
is right."""
import pytest

from tests.test_paged_gpu import Case
from tests.test_paged_ranges_gpu import check, exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("held", ["same", "int8"])
@pytest.mark.parametrize("new,ctx,page", [(1, 9000, 16), (5, 3000, 64), (300, 5000, 24), (700, 700, 16)])
def test_a_limit_that_may_run_out(cuda, held, new, ctx, page):
    import torch
    from zlift_b200 import blas, load, paged
    lib = load()
    c = Case("bf16", held, new=(new, new), ctx=(ctx, new + 3), heads=8, kv_heads=2, dim=128, page=page, seed=1)
    o, lse, o_tol, _ = exact(c)
    default = lib.zlift_get_wait_limit_ns()
    made = {}
    try:
        assert lib.zlift_set_wait_limit_ns(1) == 0
        for _ in range(5):
            made["ws"] = torch.zeros(64 << 20, dtype=torch.uint8, device=cuda)
            got, _ = c.run(workspace=made["ws"])
            torch.cuda.synchronize()
            error = blas.device_error()
            assert error in (0, 1)
            if error == 0:
                assert ((got.double() - o).abs() <= o_tol).all()
    finally:
        assert lib.zlift_set_wait_limit_ns(default) == 0
    check(c)
