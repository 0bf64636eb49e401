"""A work line whose steps are several key blocks, on the GPU."""
import pytest

from tests.test_paged_gpu import Case
from tests.test_paged_ranges_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("held", ["same", "int8"])
def test_a_table_wider_than_the_line(cuda, held):
    """The few-row kernel on a long chunk, with a page table that could hold 2^33
    steps: the answer does not change with the step."""
    import torch
    c = Case("bf16", held, new=(1500,), ctx=(1600,), heads=16, kv_heads=2, dim=128, seed=1)
    wide = torch.full((1, 3_200_000), -7, dtype=torch.int32, device=cuda)
    wide[:, :c.table.shape[1]] = c.table
    check(c, max_q=1)
    c.table = wide
    check(c, max_q=1)
    check(c)
