"""Paged attention over V rows of very unlike sizes, on the GPU, against the
definition in 64 bits.

An 8-bit row's scale may be anything, so the rows of one tile may differ by
any factor: a row that the mask hides, or one whose weight is zero, must not
cost the others their bits.

The bound, of every output element: with u the unit roundoff of the output's
type (2^-8 bf16, of 8 significant bits; 2^-11 fp16, of 11), w that of the
weights (the same, and fp16's over an 8-bit cache), and d a bound on the
error of a score,

    u |o| + (w + 2 d + (n / 16 + 8) 2^-23) sum p |v| + f

in which d = (dim + 8) 2^-24 scale max(|q| . |k|) + 4e-6 (1 + max |score|)
enters numerator and denominator, n / 16 products are added in fp32, and f is
what fp16 weights lose below 2^-14: 2^-25 sum |v| over a 16-bit cache (the
largest weight is 1 at least); over an 8-bit one, where the weights carry the
V scales, at most u max |o| over the row.  Outputs in fp16 have 2^-25 besides.
"""
import math

import pytest

from tests.test_paged_gpu import UNIT, Case

pytestmark = pytest.mark.gpu


def exact(c, causal=True):
    """O, LSE and the bounds of both, in 64 bits."""
    import torch
    scale = 1 / math.sqrt(c.dim)
    o = torch.zeros(c.total_q, c.heads, c.dim, dtype=torch.float64, device=c.dev)
    lse = torch.full((c.heads, c.total_q), -math.inf, dtype=torch.float64, device=c.dev)
    o_tol, l_tol = torch.zeros_like(o), torch.zeros_like(lse)
    keys, vals = c.held64("k"), c.held64("v")
    group = c.heads // c.kv_heads
    u = UNIT[c.elem]
    w = u if c.held == "same" else 2.0 ** -11
    k0 = q0 = 0
    for n, ctx in zip(c.new, c.ctx):
        hidden = torch.zeros(n, ctx, dtype=torch.bool, device=c.dev)
        if causal:
            reach = torch.arange(n, device=c.dev)[:, None] + ctx - n
            hidden = torch.arange(ctx, device=c.dev)[None, :] > reach
        for h in range(c.heads):
            kk, vv = keys[k0:k0 + ctx, h // group], vals[k0:k0 + ctx, h // group]
            qq = c.q[q0:q0 + n, h].double()
            rows = slice(q0, q0 + n)
            z = (qq @ kk.T * scale).masked_fill(hidden, -math.inf)
            p = torch.softmax(z, -1)
            lse[h, rows] = torch.logsumexp(z, -1)
            o[rows, h] = p @ vv
            dots = (qq.abs() @ kk.abs().T * scale).masked_fill(hidden, 0.0).amax(-1)
            top = z.abs().masked_fill(hidden, 0.0).amax(-1)
            d = (c.dim + 8) * 2.0 ** -24 * dots + 4e-6 * (1 + top)
            l_tol[h, rows] = d + 4e-6 * (1 + lse[h, rows].abs())
            rel = w + 2 * d + (ctx / 16 + 8) * 2.0 ** -23
            o_tol[rows, h] = u * o[rows, h].abs() + rel[:, None] * (p @ vv.abs())
            if c.held != "same":
                o_tol[rows, h] += u * o[rows, h].abs().amax(-1, keepdim=True)
            elif c.elem == "f16":
                o_tol[rows, h] += 2.0 ** -25 * ((~hidden).double() @ vv.abs())
            if c.elem == "f16":
                o_tol[rows, h] += 2.0 ** -25                 # O itself below 2^-14
        k0 += ctx
        q0 += n
    return o, lse, o_tol, l_tol


def check(c, causal=True, **kw):
    import torch
    from zlift_b200 import blas
    got, lse = c.run(causal, **kw)
    torch.cuda.synchronize()
    assert blas.device_error() == 0
    o, el, o_tol, l_tol = exact(c, causal)
    assert torch.isfinite(got.float()).all()
    over = ((got.double() - o).abs() / o_tol.clamp_min(1e-300)).max().item()
    assert over <= 1, f"O is at {over:.3g} times its bound"
    off = ((lse.double() - el).abs() / l_tol).max().item()
    assert off <= 1, f"LSE is at {off:.3g} times its bound"


def rewrite(c, k=None, v=None):
    from zlift_b200 import paged
    c.k_in = c.k_in if k is None else k.to(c.k_in.dtype)
    c.v_in = c.v_in if v is None else v.to(c.v_in.dtype)
    assert paged.kv_write(c.cache, c.k_in, c.v_in, c.slots) == 0


@pytest.mark.parametrize("held", ["same", "int8", "fp8"])
@pytest.mark.parametrize("new", [2, 6, 100])
@pytest.mark.parametrize("size", [1e4, 1e9, 1e30])
def test_a_large_hidden_row_costs_nothing(cuda, held, new, size):
    """The newest token's V is far above the others': only its own query sees it."""
    c = Case("bf16", held, new=(new, 3), ctx=(new + 50, 700), heads=8, kv_heads=2, dim=128, seed=new)
    v = c.v_in.float()
    v[new + 50 - 1] *= size
    v[-1] *= size
    rewrite(c, v=v)
    check(c)


@pytest.mark.parametrize("held", ["int8", "fp8"])
@pytest.mark.parametrize("new", [3, 130])
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 8, 2), (64, 4, 4)])
def test_rows_that_grow_along_the_chunk(cuda, held, new, dim, heads, kv_heads):
    """Every new token's V is above all before it, up to 1e25 in all."""
    import torch
    c = Case("bf16", held, new=(new,), ctx=(new + 300,), heads=heads, kv_heads=kv_heads, dim=dim,
             seed=new)
    grow = torch.ones(new + 300, device=cuda)
    grow[300:] = 10.0 ** torch.linspace(0, 25, new, device=cuda)
    rewrite(c, v=c.v_in.float() * grow[:, None, None])
    check(c)


@pytest.mark.parametrize("held", ["same", "int8", "fp8"])
@pytest.mark.parametrize("elem,size", [("bf16", 1e5), ("bf16", 1e20), ("f16", 6e4)])
@pytest.mark.parametrize("new,ctx", [(1, 40), (1, 5000), (4, 300), (90, 600)])
def test_a_large_row_of_zero_weight_costs_nothing(cuda, held, elem, size, new, ctx):
    """One cached V row far above the others, whose key no query gives any weight."""
    import torch
    c = Case(elem, held, new=(new,), ctx=(ctx,), heads=8, kv_heads=2, dim=128, seed=ctx)
    k, v = c.k_in.float(), c.v_in.float()
    ones = torch.ones(128, device=cuda)
    c.q = (c.q.float() * 0.1 + 4.0 * ones).to(c.q.dtype)
    at = ctx // 3
    k[at] = -9.0 * ones                                      # a score of about -400
    v = v * (1.0 if elem == "bf16" else 1e-3)
    v[at] = size * torch.sign(v[at])
    rewrite(c, k, v)
    check(c)


@pytest.mark.parametrize("held", ["int8", "fp8"])
@pytest.mark.parametrize("new", [1, 4, 70])
@pytest.mark.parametrize("size", [1e-28, 1e-20, 1e-9, 1e9, 1e20, 1e30])
def test_rows_of_any_size(cuda, held, new, size):
    """All V rows tiny, or all of them huge."""
    c = Case("bf16", held, new=(new,), ctx=(new + 200,), heads=8, kv_heads=2, dim=128, seed=3,
             spread=0.4)
    rewrite(c, v=c.v_in.float() * size)
    check(c)


@pytest.mark.parametrize("held", ["int8", "fp8"])
@pytest.mark.parametrize("new", [1, 40])
def test_a_sink_of_small_value(cuda, held, new):
    """Most of the weight on one token whose V is 1000 times below the others',
    which share the rest: both parts count."""
    import torch
    c = Case("bf16", held, new=(new,), ctx=(20000,), heads=4, kv_heads=1, dim=128, page=64, seed=5)
    k, v = c.k_in.float() * 0.1, c.v_in.float()
    ones = torch.ones(128, device=cuda)
    c.q = (c.q.float() * 0.1 + 1.0 * ones).to(c.q.dtype)
    k[0] = 0.9 * ones                                        # a weight of e^10
    v[0] *= 1e-3
    rewrite(c, k, v)
    check(c)
