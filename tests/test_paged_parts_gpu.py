"""Long contexts whose parts are joined from all over the GPU: a lost or
misplaced part of O has to show.

Each of the 128 columns of V is one in its own 128th of the keys and zero
elsewhere, so that a column of O is the weight of that part and nothing else,
and the bound (a fraction of sum p |v|, column by column) is some 0.8% of it in
bf16: 16 keys of 60000 are 3.4%.  That they are seen is tested on the CPU, with
the keys left out of the definition.
"""
import types

import pytest

from tests.test_paged_gpu import Case
from tests.test_paged_ranges_gpu import check, exact, rewrite


def one_part_a_column(ctx, kv_heads, device=None):
    import torch
    part = torch.arange(ctx, device=device) * 128 // ctx
    return torch.nn.functional.one_hot(part, 128).float()[:, None].expand(ctx, kv_heads, 128)


@pytest.mark.parametrize("elem,held", [("bf16", "same"), ("f16", "same"), ("bf16", "int8")])
def test_the_bound_sees_sixteen_lost_keys(elem, held):
    import torch
    g = torch.Generator().manual_seed(1)
    n = 20000
    c = types.SimpleNamespace(elem=elem, held=held, heads=2, kv_heads=1, dim=128, new=[2], ctx=[n], total_q=2,
                              dev=torch.device("cpu"), q=torch.randn(2, 2, 128, generator=g))
    k, v = torch.randn(n, 1, 128, generator=g).double(), one_part_a_column(n, 1).double()
    c.held64 = lambda which: k if which == "k" else v
    o, _, o_tol, _ = exact(c)
    for at in (0, 5008, n // 2 - 8, n - 18):
        left = v.clone()
        left[at:at + 16] = 0                                 # their O is lost, their weight is not
        c.held64 = lambda which: k if which == "k" else left
        short = exact(c)[0]
        assert ((short - o).abs() > 1.5 * o_tol).flatten(1).any(1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("elem,held", [("bf16", "same"), ("f16", "same"), ("bf16", "int8"), ("f16", "fp8")])
@pytest.mark.parametrize("new,ctx,heads,kv_heads", [
    ((1,), (60000,), 4, 1), ((3,), (60000,), 8, 1), ((33,), (60000,), 4, 1), ((1, 6, 1), (20000, 7000, 50), 8, 2),
    ((40, 1, 200), (20000, 333, 9000), 8, 2), ((300,), (30011,), 16, 2)])
def test_no_part_is_lost(cuda, elem, held, new, ctx, heads, kv_heads):
    import torch
    c = Case(elem, held, new=new, ctx=ctx, heads=heads, kv_heads=kv_heads, dim=128, page=64, seed=sum(new))
    rewrite(c, v=torch.cat([one_part_a_column(n, kv_heads, cuda) for n in ctx]))
    check(c)
