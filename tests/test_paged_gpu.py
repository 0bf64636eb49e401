"""The paged K/V cache and the attention over it, on the GPU, against the
definition in 64 bits.

Write and read are compared bit for bit: the quotients and products of the
quantisation are rounded once to fp32, which 64-bit arithmetic followed by
one cast reproduces (24-bit operands: products are exact in 53 bits, and a
quotient rounded to 53 and then to 24 bits is the one rounded to 24).

Attention.  With u the unit roundoff of the 16-bit type (2^-8 bf16, 2^-11
fp16), every output is within u |o| (its own rounding) + u A (weights rounded
to the type before the product with V; they sum to one) + 2e-5 A (fp32
accumulation and exponentials) of the exact value, A the largest |v| of the
sequence and head.  LSE: the fp32 dot products are within
(dim + 8) 2^-24 scale max(|q| . |k|), the rest within 4e-6 (1 + |lse|).
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TOP = {"int8": 127.0, "fp8": 448.0}


def kinds():
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "int8": torch.int8,
            "fp8": torch.float8_e4m3fn}


def quantise64(x, held):
    """Codes (as float64) and fp32 scales of rows [..., dim], in 64 bits."""
    import torch
    x = x.double()
    amax = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    full = (amax >= 2.0 ** -100) & ~bad
    one = torch.ones_like(amax)
    scale = torch.where(full, amax / TOP[held], torch.where(bad, one * math.nan, one * 0)).float()
    mul = torch.where(full, TOP[held] / torch.where(full, amax, one), one * 0).float()
    v = (torch.where(full[..., None], x, 0.0) * mul.double()[..., None]).float().double()
    if held == "int8":
        return torch.round(v), scale
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -30))).clamp_min(-6.0)
    step = torch.exp2(e - 3)
    return torch.round(v / step) * step, scale


class Case:
    """A cache filled through kv_write, with sequences of given lengths."""

    def __init__(self, elem="bf16", held="same", new=(1,), ctx=(5,), heads=4, kv_heads=2, dim=64,
                 page=16, layout="nhd", seed=0, junk=True, big=0, spread=0.0):
        import torch
        from zlift_b200 import paged
        self.elem, self.held, self.heads, self.kv_heads, self.dim = elem, held, heads, kv_heads, dim
        self.new, self.ctx, self.page = list(new), list(ctx), page
        dev = torch.device("cuda")
        self.dev = dev
        g = torch.Generator(device=dev).manual_seed(seed)
        kind = kinds()[elem]
        hkind = kind if held == "same" else kinds()[held]
        per = [-(-c // page) for c in self.ctx]
        pages = sum(per) + 2 + big
        width = max(1, max(per)) + 1
        table = np.full((len(per), width), -7, np.int32)     # unused entries: never followed
        order = np.random.RandomState(seed).permutation(pages)
        if big:                                              # use the far end of a large cache
            order = np.sort(order)[::-1].copy()
        at = 0
        for i, n in enumerate(per):
            table[i, :n] = order[at: at + n]
            at += n
        self.table = torch.from_numpy(table).to(dev)

        # a cache full of junk: NaN everywhere that nothing is written
        def blank(scale_too):
            if layout == "nhd":
                t = torch.empty(2, pages, page, kv_heads, dim, dtype=hkind, device=dev)
                k, v = t[0], t[1]
            elif layout == "hnd":
                t = torch.empty(2, pages, kv_heads, page, dim, dtype=hkind, device=dev)
                k, v = t[0].transpose(1, 2), t[1].transpose(1, 2)
            elif layout == "pair":                           # K and V of a page side by side
                t = torch.empty(pages, 2, page, kv_heads, dim, dtype=hkind, device=dev)
                k, v = t[:, 0], t[:, 1]
            else:                                            # rows that no vector load may take
                t = torch.empty(2, pages, page, kv_heads, dim + 1, dtype=hkind, device=dev)
                k, v = t[0, ..., 1:], t[1, ..., 1:]
            if not big:
                raw = t.view(torch.uint8)
                raw.fill_(0xff if junk else 0)               # NaN in f16, bf16 and e4m3
                if held == "int8" and junk:
                    raw.fill_(0x80)
            return k, v

        k, v = blank(True)
        ks = vs = None
        if held != "same":
            ks, vs = (torch.full((pages, kv_heads, page), math.nan if junk else 0.0, device=dev)
                      for _ in range(2))
        self.cache = paged.KVCache(k, v, ks, vs)
        total = sum(self.ctx)

        def rand(*shape):
            x = torch.randn(*shape, generator=g, device=dev)
            return (x * torch.exp(spread * torch.randn(*shape[:-1], 1, generator=g, device=dev))).to(kind)

        self.k_in, self.v_in = rand(total, kv_heads, dim), rand(total, kv_heads, dim)
        slots = []
        for i, c in enumerate(self.ctx):
            pos = np.arange(c)
            slots.append(table[i, pos // page].astype(np.int64) * page + pos % page)
        self.slots = torch.from_numpy(np.concatenate(slots + [np.zeros(0, np.int64)])
                                      .astype(np.int32)).to(dev)
        if total:
            assert paged.kv_write(self.cache, self.k_in, self.v_in, self.slots) == 0
        self.cu = torch.tensor(np.concatenate([[0], np.cumsum(self.new)]), dtype=torch.int32,
                               device=dev)
        self.lens = torch.tensor(self.ctx, dtype=torch.int32, device=dev)
        self.total_q = sum(self.new)
        self.q = rand(self.total_q, heads, dim)

    def held64(self, which):
        """The values that the cache stands for, [tokens, kv_heads, dim]."""
        x = self.k_in if which == "k" else self.v_in
        if self.held == "same":
            return x.double()
        codes, scale = quantise64(x, self.held)
        return codes * scale.double()[..., None]

    def exact(self, causal=True, scale=None):
        import torch
        scale = 1 / math.sqrt(self.dim) if scale is None else scale
        o = torch.zeros(self.total_q, self.heads, self.dim, dtype=torch.float64, device=self.dev)
        lse = torch.full((self.heads, self.total_q), -math.inf, dtype=torch.float64, device=self.dev)
        o_tol, l_tol = torch.zeros_like(o), torch.zeros_like(lse)
        keys, vals = self.held64("k"), self.held64("v")
        group = self.heads // self.kv_heads
        k0 = q0 = 0
        u = UNIT[self.elem]
        for n, c in zip(self.new, self.ctx):
            for h in range(self.heads):
                kk, vv = keys[k0:k0 + c, h // group], vals[k0:k0 + c, h // group]
                qq = self.q[q0:q0 + n, h].double()
                for i in range(n):
                    seen = max(0, min(c, c - n + i + 1)) if causal else c
                    if not seen:
                        continue
                    z = kk[:seen] @ qq[i] * scale
                    lse[h, q0 + i] = torch.logsumexp(z, 0)
                    o[q0 + i, h] = torch.softmax(z, 0) @ vv[:seen]
                    big = vv[:seen].abs().max()
                    o_tol[q0 + i, h] = u * o[q0 + i, h].abs() + (u + 2e-5) * big
                    dots = (kk[:seen].abs() @ qq[i].abs()).max() * abs(scale)
                    l_tol[h, q0 + i] = (self.dim + 8) * 2.0 ** -24 * dots + \
                        4e-6 * (1 + lse[h, q0 + i].abs())
            k0 += c
            q0 += n
        return o, lse, o_tol, l_tol

    def run(self, causal=True, scale=None, max_q=None, stream=None, o=None, lse=True, q=None, **kw):
        import torch
        from zlift_b200 import paged
        made = o is None
        o = torch.full_like(self.q, 7.0) if made else o
        ls = torch.full((self.heads, self.total_q), 7.0, device=self.dev) if lse is True else lse
        if made and stream is not None:                      # filled on this stream, used on that
            torch.cuda.current_stream().synchronize()
        rc = paged.paged_attention(self.cache, self.q if q is None else q, o, ls, self.table, self.cu,
                                   self.lens, max(self.new) if max_q is None else max_q,
                                   causal=causal, scale=scale, stream=stream, **kw)
        assert rc == 0
        return o, ls

    def check(self, causal=True, scale=None, **kw):
        import torch
        from zlift_b200 import blas
        o, lse = self.run(causal, scale, **kw)
        torch.cuda.synchronize()
        assert blas.device_error() == 0
        eo, el, to, tl = self.exact(causal, scale)
        assert torch.isfinite(o.float()).all()
        over = ((o.double() - eo).abs() - to).max().item() if o.numel() else 0.0
        assert over <= 0, f"O is {over:.3g} past its bound"
        if lse is not None and lse.numel():
            fin = torch.isfinite(el)
            assert torch.equal(torch.isfinite(lse), fin) and (lse[~fin] == -math.inf).all()
            off = ((lse.double() - el).abs() - tl)[fin]
            assert off.numel() == 0 or off.max().item() <= 0, f"LSE is {off.max():.3g} past its bound"
        return o, lse


# ---- write and read ----------------------------------------------------------

@pytest.mark.parametrize("held", ["same", "int8", "fp8"])
@pytest.mark.parametrize("elem", ["bf16", "f16"])
@pytest.mark.parametrize("dim,heads,page,layout", [
    (128, 8, 16, "nhd"), (64, 3, 7, "hnd"), (256, 1, 32, "pair"), (32, 2, 1, "nhd"),
    (96, 2, 16, "nhd"), (40, 5, 3, "odd"), (1, 1, 16, "nhd")])
def test_write_read_round_trip(cuda, elem, held, dim, heads, page, layout):
    """What is read back is exactly code * scale of the definition, rounded
    once to the output's type; nothing outside the written slots changes."""
    import torch
    from zlift_b200 import blas, paged
    c = Case(elem, held, new=(1, 1, 1), ctx=(37, 1, 16), heads=heads, kv_heads=heads, dim=dim,
             page=page, layout=layout, seed=dim + page, spread=1.0)
    outs = [kinds()[elem]]
    if held != "same":
        outs = [torch.bfloat16, torch.float16, torch.float32]
    cu = torch.tensor([0, 37, 38, 54], dtype=torch.int32, device=cuda)
    for kind in outs:
        k, v = (torch.full((56, heads, dim), 3.0, dtype=kind, device=cuda) for _ in range(2))
        assert paged.kv_read(c.cache, k, v, c.table, cu) == 0
        for got, which in ((k, "k"), (v, "v")):
            want = c.held64(which).float().to(kind)
            assert torch.equal(got[:54], want)
            assert (got[54:] == 3.0).all()                   # past cu[batch]: left alone
    # unused slots keep their junk
    used = torch.zeros(c.cache.k.shape[0] * page, dtype=torch.bool, device=cuda)
    used[c.slots.long()] = True
    raw = (c.cache.k.float() if held != "int8" else c.cache.k).reshape(-1, heads, dim)[~used]
    assert (raw == -128).all() if held == "int8" else torch.isnan(raw).all()
    assert blas.device_error() == 0


def test_read_window_and_empty_sequences(cuda):
    """starts select a window; sequences without tokens in it are passed over."""
    import torch
    from zlift_b200 import paged
    c = Case("bf16", "fp8", new=(1,) * 4, ctx=(40, 3, 25, 9), kv_heads=2, dim=128, seed=3)
    cu = torch.tensor([0, 5, 5, 12, 13], dtype=torch.int32, device=cuda)
    starts = torch.tensor([30, 1, 17, 8], dtype=torch.int32, device=cuda)
    k, v = (torch.empty(13, 2, 128, device=cuda) for _ in range(2))
    assert paged.kv_read(c.cache, k, v, c.table, cu, starts=starts) == 0
    pick = list(range(30, 35)) + list(range(43 + 17, 43 + 24)) + [40 + 3 + 25 + 8]
    assert torch.equal(k, c.held64("k").float()[pick])
    assert torch.equal(v, c.held64("v").float()[pick])


@pytest.mark.parametrize("held", ["int8", "fp8"])
@pytest.mark.parametrize("dim", [128, 24])
def test_write_edges(cuda, held, dim):
    """Zero rows, rows below 2^-100, and rows with a NaN or an infinity."""
    import torch
    from zlift_b200 import paged
    c = Case("bf16", held, new=(1,), ctx=(0,), kv_heads=1, heads=1, dim=dim, junk=False)
    x = torch.zeros(6, 1, dim, dtype=torch.bfloat16, device=cuda)
    x[1, 0, 3] = 2.0 ** -101
    x[2, 0, 5] = 2.0 ** -100
    x[3, 0, :] = 1.0
    x[3, 0, 1] = math.nan
    x[4, 0, 0] = -math.inf
    x[5, 0, :] = 3.0e38
    slots = torch.tensor([0, 1, 2, 3, 4, 5], dtype=torch.int32, device=cuda)
    table = torch.tensor([[0]], dtype=torch.int32, device=cuda)
    cu = torch.tensor([0, 6], dtype=torch.int32, device=cuda)
    assert paged.kv_write(c.cache, x, -x, slots) == 0
    k, v = (torch.empty(6, 1, dim, device=cuda) for _ in range(2))
    assert paged.kv_read(c.cache, k, v, table, cu) == 0
    codes, scale = quantise64(x, held)
    want = (codes * scale.double()[..., None]).float()
    assert torch.equal(k[[0, 1, 2, 5]], want[[0, 1, 2, 5]])
    assert torch.equal(v[[0, 1, 2, 5]], -want[[0, 1, 2, 5]])
    assert (k[:2] == 0).all() and k[2, 0, 5] != 0
    assert torch.isnan(k[3:5]).all() and torch.isnan(v[3:5]).all()


def test_write_skips_padding_and_refuses_slots_outside(cuda):
    import torch
    from zlift_b200 import blas, paged
    for dim in (128, 24):
        c = Case("bf16", "same", new=(1,), ctx=(0,), kv_heads=1, heads=1, dim=dim, junk=False)
        cap = c.cache.k.shape[0] * 16
        x = torch.ones(3, 1, dim, dtype=torch.bfloat16, device=cuda)
        slots = torch.tensor([-1, 4, -(2 ** 31)], dtype=torch.int32, device=cuda)
        assert paged.kv_write(c.cache, x, x, slots) == 0
        assert blas.device_error() == 0
        assert c.cache.k.float().sum() == dim and (c.cache.k[0, 4] == 1).all()
        slots = torch.tensor([cap, 5, 2 ** 31 - 1], dtype=torch.int32, device=cuda)
        assert paged.kv_write(c.cache, x, x, slots) == 0
        assert blas.device_error() == 2 and blas.device_error() == 0
        assert c.cache.k.float().sum() == 2 * dim


def test_read_refuses_pages_outside(cuda):
    import torch
    from zlift_b200 import blas, paged
    for dim in (128, 24):
        c = Case("f16", "same", new=(1,), ctx=(40,), kv_heads=1, heads=1, dim=dim)
        t = c.table.clone()
        t[0, 1] = c.cache.k.shape[0]
        k, v = (torch.empty(50, 1, dim, dtype=torch.float16, device=cuda) for _ in range(2))
        cu = torch.tensor([0, 40], dtype=torch.int32, device=cuda)
        assert paged.kv_read(c.cache, k, v, t, cu) == 0
        assert blas.device_error() == 2
        assert torch.equal(k[:16], c.k_in[:16]) and torch.equal(k[32:40], c.k_in[32:40])
        assert (k[16:32] == 0).all()


# ---- attention -----------------------------------------------------------------

@pytest.mark.parametrize("held", ["same", "int8", "fp8"])
@pytest.mark.parametrize("elem", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [
    (8, 2, 128, 16), (4, 4, 64, 32), (6, 2, 64, 24), (8, 1, 128, 128), (5, 1, 128, 8),
    (32, 2, 64, 64)])
def test_decode(cuda, elem, held, heads, kv_heads, dim, page):
    """One token a sequence, contexts from one token on."""
    c = Case(elem, held, new=(1,) * 6, ctx=(1, 2, 17, 130, 515, 64), heads=heads,
             kv_heads=kv_heads, dim=dim, page=page, seed=heads + dim, spread=0.4)
    c.check()


@pytest.mark.parametrize("held", ["same", "int8", "fp8"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [
    (8, 2, 128, 16), (4, 4, 64, 32), (3, 1, 64, 8), (7, 1, 128, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_few_tokens(cuda, held, heads, kv_heads, dim, page, causal):
    """Drafted tokens: ragged chunks of a few tokens, some sequences without any."""
    c = Case("bf16", held, new=(5, 0, 2, 8, 1), ctx=(5, 33, 300, 129, 700), heads=heads,
             kv_heads=kv_heads, dim=dim, page=page, seed=heads, spread=0.4)
    c.check(causal=causal)


@pytest.mark.parametrize("elem,held", [("bf16", "same"), ("f16", "same"), ("bf16", "int8"),
                                       ("f16", "int8"), ("bf16", "fp8"), ("f16", "fp8")])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [
    (8, 2, 128, 16), (4, 4, 64, 32), (6, 2, 128, 24), (8, 1, 64, 256)])
@pytest.mark.parametrize("causal", [True, False])
def test_chunk(cuda, elem, held, heads, kv_heads, dim, page, causal):
    """Chunks that span several query and key tiles, with and without context."""
    c = Case(elem, held, new=(150, 1, 67, 0), ctx=(150, 260, 407, 12), heads=heads,
             kv_heads=kv_heads, dim=dim, page=page, seed=heads + page, spread=0.4)
    c.check(causal=causal)


@pytest.mark.parametrize("held", ["same", "fp8"])
@pytest.mark.parametrize("new", [1, 3, 70])
def test_rows_that_see_nothing(cuda, held, new):
    """seq_k below the chunk (the first rows see no key) and empty contexts:
    O = 0, LSE = -inf."""
    for causal in (True, False):
        c = Case("bf16", held, new=(new, new, new), ctx=(0, 1, max(1, new // 2)), heads=8,
                 kv_heads=2, dim=128)
        o, lse = c.check(causal=causal)
        assert (o[:new] == 0).all() and (lse[:, :new] == -math.inf).all()


@pytest.mark.parametrize("held", ["same", "int8", "fp8"])
@pytest.mark.parametrize("new", [1, 4, 90])
def test_hint_does_not_change_results(cuda, held, new):
    """max_q picks a kernel; every kernel gives the same answer within the bounds."""
    c = Case("bf16", held, new=(new, 1, new), ctx=(new + 3, 200, 333), heads=8, kv_heads=2, dim=128,
             seed=new, spread=0.4)
    for hint in (0, 1, 4, 8, 64, 5000):
        c.check(max_q=hint)


@pytest.mark.parametrize("dim,heads,kv_heads,page,layout", [
    (96, 4, 2, 16, "nhd"), (80, 2, 2, 5, "odd"), (128, 4, 2, 1, "nhd"), (256, 2, 1, 16, "nhd"),
    (64, 4, 2, 20, "odd"), (128, 4, 1, 20, "hnd"), (1, 1, 1, 3, "nhd"), (128, 256, 1, 16, "nhd")])
@pytest.mark.parametrize("held", ["same", "int8"])
def test_layouts_outside_the_tensor_cores(cuda, dim, heads, kv_heads, page, layout, held):
    c = Case("f16", held, new=(1, 9, 3), ctx=(70, 40, 3), heads=heads, kv_heads=kv_heads, dim=dim,
             page=page, layout=layout, seed=dim, spread=0.4)
    c.check()


@pytest.mark.parametrize("layout", ["nhd", "hnd", "pair"])
@pytest.mark.parametrize("held", ["same", "int8", "fp8"])
@pytest.mark.parametrize("new", [1, 6, 140])
def test_strides(cuda, layout, held, new):
    """Cache layouts, queries out of a fused QKV tensor, an output with gaps."""
    import torch
    c = Case("bf16", held, new=(new, new), ctx=(new + 100, new), heads=8, kv_heads=2, dim=128,
             layout=layout, seed=new)
    qkv = torch.zeros(c.total_q, 12, 128, dtype=torch.bfloat16, device=cuda)
    qkv[:, :8] = c.q
    o = torch.full((8, c.total_q + 1, 160), 5.0, dtype=torch.bfloat16, device=cuda)
    c.check(q=qkv[:, :8], o=o[:, :-1, :128].transpose(0, 1))
    assert (o[:, -1] == 5).all() and (o[:, :, 128:] == 5).all()


@pytest.mark.parametrize("held", ["same", "int8", "fp8"])
@pytest.mark.parametrize("new", [1, 5, 80])
def test_large_scores_and_growing_maximum(cuda, held, new):
    """Scores of hundreds that grow along the keys: the running maximum moves
    at every step, and early weights underflow to zero."""
    import torch
    from zlift_b200 import paged
    c = Case("bf16", held, new=(new,), ctx=(new + 400,), heads=4, kv_heads=2, dim=128, seed=2)
    ramp = torch.linspace(0.05, 8.0, c.k_in.shape[0], device=cuda)[:, None, None]
    direction = torch.ones(128, device=cuda)
    c.k_in = (ramp * direction + 0.1 * c.k_in.float()).to(torch.bfloat16)
    c.q = (0.7 * direction + 0.1 * c.q.float()).to(torch.bfloat16)
    assert paged.kv_write(c.cache, c.k_in, c.v_in, c.slots) == 0
    c.check()
    c.q = -c.q                                               # and a falling one
    c.check()


@pytest.mark.parametrize("held", ["same", "int8", "fp8"])
@pytest.mark.parametrize("new", [2, 6, 100])
def test_masked_keys_have_no_effect(cuda, held, new):
    """NaN and infinities in keys and values that the mask hides from a query
    leave it exactly as finite ones do; queries that see them get NaN."""
    import torch
    from zlift_b200 import paged
    c = Case("bf16", held, new=(new, 3), ctx=(new + 50, 60), heads=8, kv_heads=2, dim=128, seed=5)
    clean, clse = c.run()
    clean, clse = clean.clone(), clse.clone()
    first = new - 1                                          # the last token of sequence 0 only
    at = new + 50 - 1
    for kbad, vbad in ((math.nan, 1.0), (1.0, math.nan), (1.0, math.inf), (math.nan, -math.inf)):
        k, v = c.k_in.clone(), c.v_in.clone()
        k[at, :, 7] = k[at, :, 7] * kbad if kbad != 1.0 else k[at, :, 7]
        v[at, :, 9] = vbad if vbad != 1.0 else v[at, :, 9]
        assert paged.kv_write(c.cache, k, v, c.slots) == 0
        o, lse = c.run()
        keep = torch.ones(c.total_q, dtype=torch.bool, device=cuda)
        keep[first] = False
        u = UNIT["bf16"]
        assert torch.isfinite(o[keep].float()).all()
        assert ((o[keep].float() - clean[keep].float()).abs()
                <= 2 * (u + 2e-5) * c.v_in.float().abs().max()).all()
        assert (lse[:, keep] - clse[:, keep]).abs().max() <= 1e-5
        bad = ~torch.isfinite(o[first].float())
        if math.isnan(kbad):
            assert bad.all() and torch.isnan(lse[:, first]).all()
        else:
            assert bad[:, 9].all()


@pytest.mark.parametrize("held", ["same", "int8"])
@pytest.mark.parametrize("new", [1, 4, 100])
def test_pages_outside_count_as_absent(cuda, held, new):
    """Pages outside the cache are not followed: error 2, and the other keys'
    attention is that of a sequence without them."""
    import torch
    from zlift_b200 import blas
    c = Case("bf16", held, new=(new,), ctx=(new + 200,), heads=8, kv_heads=2, dim=128, seed=1)
    c.table[0, 1] = c.cache.k.shape[0] + 3
    c.table[0, 4] = -1
    o, lse = c.run(causal=False)
    torch.cuda.synchronize()
    assert blas.device_error() == 2 and blas.device_error() == 0
    left = [j for j in range(new + 200) if j // 16 not in (1, 4)]
    c.k_in, c.v_in, c.ctx = c.k_in[left], c.v_in[left], [len(left)]
    eo, el, to, tl = c.exact(causal=False)
    assert ((o.double() - eo).abs() <= to).all() and ((lse.double() - el).abs() <= tl).all()


@pytest.mark.parametrize("new", [1, 40])
def test_lengths_outside_are_clamped(cuda, new):
    """cu_q past total_q and lengths past the page table stay in bounds."""
    import torch
    from zlift_b200 import blas
    c = Case("bf16", "same", new=(new, new), ctx=(new + 20, new + 9), heads=4, kv_heads=2, dim=128)
    good = c.table.clone()
    c.table = torch.where(good < 0, torch.zeros_like(good), good)
    c.cu[2] = c.total_q + 1000
    c.lens[1] = 2 ** 30
    o, _ = c.run()
    torch.cuda.synchronize()
    assert blas.device_error() == 2
    eo, _, to, _ = c.exact()
    assert ((o.double() - eo).abs() <= to)[:new].all()


@pytest.mark.parametrize("held", ["same", "int8", "fp8"])
@pytest.mark.parametrize("new", [1, 5, 200])
def test_repeatable(cuda, held, new):
    """The same call gives the same bits, whatever ran in between on the workspace."""
    import torch
    c = Case("bf16", held, new=(new,) * 3, ctx=(new + 900, new + 5, new + 333), heads=8, kv_heads=2,
             dim=128, seed=9)
    d = Case("f16", "same", new=(3, 30), ctx=(2000, 40), heads=16, kv_heads=4, dim=64, seed=10)
    o, lse = c.run()
    for _ in range(3):
        d.run()
        o2, lse2 = c.run()
        assert torch.equal(o, o2) and torch.equal(lse, lse2)
    d.check()


def test_other_stream_and_graph(cuda):
    """Runs on the stream that it is given, and replays from a graph with new
    lengths in place."""
    import torch
    from zlift_b200 import paged
    c = Case("bf16", "same", new=(1, 1), ctx=(300, 211), heads=8, kv_heads=2, dim=128, seed=4)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        o, lse = c.run(stream=s)                             # makes the workspace too
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            assert paged.kv_write(c.cache, c.k_in, c.v_in, c.slots, stream=s) == 0
            assert paged.paged_attention(c.cache, c.q, o, lse, c.table, c.cu, c.lens, 1, stream=s) == 0
        for lens in ([300, 211], [299, 1], [17, 200]):
            c.lens.copy_(torch.tensor(lens))
            o.fill_(7)
            graph.replay()
            s.synchronize()
            full = c.ctx
            k, v = c.k_in, c.v_in
            c.ctx = lens
            c.k_in = torch.cat([k[:lens[0]], k[300:300 + lens[1]]])
            c.v_in = torch.cat([v[:lens[0]], v[300:300 + lens[1]]])
            eo, el, to, tl = c.exact()
            c.k_in, c.v_in, c.ctx = k, v, full
            assert ((o.double() - eo).abs() <= to).all() and ((lse.double() - el).abs() <= tl).all()
    s.synchronize()


@pytest.mark.parametrize("held", ["same", "int8"])
def test_offsets_past_32_bits(cuda, held):
    """A cache of more than 2^32 elements, used at its far end."""
    pages = (1 << 32) // (2 * 16 * 128) + 64
    for new in (1, 70):
        c = Case("bf16", held, new=(new,), ctx=(new + 90,), heads=4, kv_heads=2, dim=128, big=pages,
                 junk=False, seed=1)
        assert int(c.table[0, 0]) * 16 * 2 * 128 > (1 << 32) - (1 << 20)
        c.check()


def test_scale_and_no_lse(cuda):
    c = Case("bf16", "same", new=(2, 90), ctx=(100, 130), heads=4, kv_heads=1, dim=64, seed=8)
    c.check(scale=0.37)
    c.check(scale=-0.2)
    c.check(scale=0.0)
    c.check(lse=None)


@pytest.mark.parametrize("batch", [33, 200])
def test_many_sequences(cuda, batch):
    """More sequences than a warp has lanes, of very unlike lengths."""
    r = np.random.RandomState(batch)
    new = [int(x) for x in r.randint(0, 4, batch)]
    ctx = [int(x) for x in r.choice([1, 3, 40, 500], batch)]
    c = Case("bf16", "same", new=new, ctx=[max(a, b) for a, b in zip(new, ctx)], heads=4, kv_heads=2,
             dim=64, seed=batch)
    c.check()
    c.check(max_q=100)


def test_long_context(cuda):
    """Contexts that are split over many blocks, among short ones."""
    for held in ("same", "int8", "fp8"):
        for new in (1, 6, 40):
            c = Case("bf16", held, new=(new, 1, new), ctx=(20000, 50, 7000), heads=8, kv_heads=2,
                     dim=128, page=64, seed=6)
            c.check()


def test_written_through_a_chunked_prefill(cuda):
    """Prefill in chunks gives what one chunk gives: each chunk is written,
    then attends over everything before it."""
    import torch
    from zlift_b200 import paged
    c = Case("bf16", "same", new=(300,), ctx=(300,), heads=8, kv_heads=2, dim=128, seed=12)
    whole, wlse = c.check()
    o, lse = torch.empty_like(whole), torch.empty_like(wlse)
    for a, b in ((0, 128), (128, 129), (129, 140), (140, 300)):
        cu = torch.tensor([0, b - a], dtype=torch.int32, device=cuda)
        lens = torch.tensor([b], dtype=torch.int32, device=cuda)
        part = torch.empty(8, b - a, device=cuda)
        assert paged.kv_write(c.cache, c.k_in[a:b], c.v_in[a:b], c.slots[a:b]) == 0
        assert paged.paged_attention(c.cache, c.q[a:b], o[a:b], part, c.table, cu, lens, b - a) == 0
        lse[:, a:b] = part
    eo, el, to, tl = c.exact()
    assert ((o.double() - eo).abs() <= to).all() and ((lse.double() - el).abs() <= tl).all()


def test_small_workspace_is_declined_or_enough(cuda):
    """A workspace of the size asked for serves the call; a smaller one is
    declined before anything is launched."""
    import torch
    from zlift_b200 import paged
    c = Case("bf16", "same", new=(1, 1), ctx=(3000, 5), heads=8, kv_heads=2, dim=128)
    need = paged.attention_workspace(c.cache, 8, 2, 1, 2)
    want, _ = c.run()
    ws = torch.zeros(max(need, 16), dtype=torch.uint8, device=cuda)
    o, _ = c.run(workspace=ws)
    assert torch.equal(o, want)
    if need > 16:
        o = torch.full_like(c.q, 7.0)
        assert paged.paged_attention(c.cache, c.q, o, None, c.table, c.cu, c.lens, 1,
                                     workspace=ws[:need - 1]) == 1
        torch.cuda.synchronize()
        assert (o == 7).all()


@pytest.mark.parametrize("held", ["int8", "fp8", "bf16"])
def test_example_runs(cuda, held):
    """examples/paged_serving.py: projections, cache and attention together,
    against the contiguous forward on the same tokens."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                        "paged_serving.py")
    spec = importlib.util.spec_from_file_location("paged_serving", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.main(held)


@pytest.mark.parametrize("held", ["same", "int8", "fp8"])
@pytest.mark.parametrize("elem", ["bf16", "f16"])
@pytest.mark.parametrize("new", [1, 70])
def test_one_key_returns_its_value(cuda, elem, held, new):
    """A query that sees one key gets that key's V: every code from the largest
    to the subnormal ones, at any scale, within the two roundings (weight times
    scale, and output) of each value itself."""
    import torch
    from zlift_b200 import paged
    for size in (1e-3, 1.0, 30.0):
        c = Case(elem, held, new=(new,), ctx=(new,), heads=4, kv_heads=2, dim=128, seed=int(size) + new)
        v = c.v_in.float()
        v[0] = size * torch.exp2(-torch.arange(128, device=cuda) / 6.0) * torch.sign(v[0])
        c.v_in = v.to(c.v_in.dtype)
        assert paged.kv_write(c.cache, c.k_in, c.v_in, c.slots) == 0
        o, _ = c.run()
        want = c.held64("v")[0].repeat_interleave(2, 0)
        # (fp16 holds nothing below 2^-24)
        bound = (2.01 * UNIT[elem]) * want.abs() + (2.0 ** -24 if elem == "f16" else 0.0)
        assert ((o[0].double() - want).abs() <= bound).all()


@pytest.mark.parametrize("new,heads,kv_heads", [(1, 4, 1), (3, 8, 1), (33, 4, 1)])
@pytest.mark.parametrize("held", ["same", "fp8"])
def test_one_unit_over_the_whole_gpu(cuda, held, new, heads, kv_heads):
    """One sequence and one KV head: every worker has a part of one unit."""
    c = Case("bf16", held, new=(new,), ctx=(60000,), heads=heads, kv_heads=kv_heads, dim=128, page=64,
             seed=new)
    c.check()


def test_calls_on_two_streams_keep_apart(cuda):
    """Each stream has a workspace of its own."""
    import torch
    c = Case("bf16", "same", new=(1, 2), ctx=(3000, 500), heads=8, kv_heads=2, dim=128, seed=1)
    d = Case("bf16", "int8", new=(40,), ctx=(2500,), heads=8, kv_heads=2, dim=128, seed=2)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    c.run(stream=s1)
    d.run(stream=s2)
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        outs.append((c, c.run(stream=s1)))
        outs.append((d, d.run(stream=s2)))
    torch.cuda.synchronize()
    for case, (o, lse) in outs:
        eo, el, to, tl = case.exact()
        assert ((o.double() - eo).abs() <= to).all() and ((lse.double() - el).abs() <= tl).all()


def test_a_capture_makes_no_workspace(cuda):
    """A stream without a workspace says so under capture, where memory would
    be the graph's."""
    import torch
    c = Case("bf16", "same", new=(1,), ctx=(300,), heads=8, kv_heads=2, dim=128)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    from zlift_b200 import paged
    paged._workspaces.pop((c.cache.device, s.cuda_stream), None)
    o, lse = torch.full_like(c.q, 7.0), torch.empty(8, 1, device=cuda)
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=s):
        with pytest.raises(RuntimeError):
            c.run(stream=s, o=o, lse=lse)
    torch.cuda.synchronize()
    c.check(stream=s)
