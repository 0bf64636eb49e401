"""What the paged key/value cache operators are measured on.

Three operators of a serving step, which share one cache of fixed-size pages:

  write   new tokens' K and V into their slots, quantised to 8 bits per
          (token, head) where the cache holds 8 bits.  A write pass ends with
          reading the same tokens back, so that what it returns is the values
          the cache now stands for;
  read    the tokens of a batch of sequences out of the cache into packed
          16-bit K and V;
  attend  attention of each sequence's newest tokens (a chunk, a few drafted
          tokens or a single one) over all of its cached tokens.

Where ``own`` is false ``run`` computes them with elementary torch operations
in 32 bits, where it is true with the package's entry points.

The formulas.  A slot is page * page_size + offset.  An 8-bit row x of one
token and head has the scale s = amax / top (amax = max |x|, top = 127 for
int8 and 448 for e4m3) and the codes round(x * (top / amax)), ties to even,
both in 32 bits; it stands for code * s.  Attention of query i of a sequence
with m new and n cached tokens runs over the keys j <= i + n - m (all of them
when not causal): o = softmax(scale * q.K^T) V, lse = log sum exp of the
scaled scores; query head h uses key head h // (heads / kv_heads).
"""
import math

import numpy as np
import torch

own = False

TOP = {"int8": 127.0, "fp8": 448.0}
HELD = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
KIND = {"bf16": torch.bfloat16, "f16": torch.float16}


def _case(name, op, elem, held, batch, new, ctx, ragged, heads, kv_heads, dim, page, causal=True):
    c = dict(op=op, elem=elem, held=held, batch=batch, new=new, ctx=ctx, ragged=ragged,
             heads=heads, kv_heads=kv_heads, dim=dim, page=page, causal=causal)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # one decoding step of a mid-sized batch: a token for each sequence
        _case("write_step_int8", "write", "bf16", "int8", 64, 1, 4096, True, 32, 8, 128, 16),
        # prompts of a batch entering the cache, 8 KV heads
        _case("write_prompts_fp8", "write", "bf16", "fp8", 8, 4096, 4096, False, 32, 8, 128, 64),
        # a ragged chunk of half-precision tokens into an unquantised cache, narrow heads
        _case("write_chunk_f16", "write", "f16", "same", 5, 701, 3000, True, 16, 16, 64, 32),
        # one long sequence dequantised for a consumer that wants it contiguous
        _case("read_long_int8", "read", "bf16", "int8", 1, 1, 131072, False, 32, 8, 128, 64),
        # a small ragged batch moved out of a 16-bit cache
        _case("read_ragged_f16", "read", "f16", "same", 7, 1, 1153, True, 16, 4, 64, 16),
        # the smallest call: one sequence, a short context, one token
        _case("decode_one", "attend", "bf16", "same", 1, 1, 515, False, 8, 2, 128, 16),
        # the ordinary decoding step: a ragged batch with grouped heads
        _case("decode_batch", "attend", "bf16", "same", 64, 1, 4096, True, 32, 8, 128, 16),
        # long contexts in an 8-bit cache, where the cache's bytes are the cost
        _case("decode_long_int8", "attend", "bf16", "int8", 16, 1, 32768, True, 32, 8, 128, 64),
        # every head with keys of its own, narrow heads, half precision
        _case("decode_mha_fp8", "attend", "f16", "fp8", 24, 1, 2047, True, 16, 16, 64, 32),
        # a few drafted tokens a sequence, scored together
        _case("draft_fp8", "attend", "bf16", "fp8", 32, 5, 4096, True, 32, 8, 128, 32),
        # a chunk of one long prompt over what is already cached
        _case("chunk_long", "attend", "bf16", "same", 1, 512, 32768, False, 32, 8, 128, 64),
        # chunks of several prompts, the compute-bound end, 8-bit cache
        _case("chunk_batch_int8", "attend", "bf16", "int8", 4, 2048, 4096, True, 32, 8, 128, 16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "attend"])
    elem = rng.choice(["bf16", "f16"])
    held = rng.choice(["same", "int8", "fp8"])
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
    group = rng.choice([1, 2, 3, 4, 6, 8])
    if kv_heads * group > 40:
        group = 2
    page = rng.choice([8, 16, 24, 32, 64, 128, 256])
    ragged = rng.random() < 0.7
    room = 64 * 4096 * 8                       # (tokens x kv_heads) of the largest caches
    if op == "attend":
        kind = rng.choice(["one", "few", "chunk"])
        new = 1 if kind == "one" else rng.randint(2, 16) if kind == "few" else _log(rng, 17, 2048)
        ctx = max(new, _log(rng, 64, 32768))
        batch = _log(rng, 1, 96)
        # as much work as the largest listed cases at most
        while batch > 1 and (batch * ctx * kv_heads > room
                             or batch * new * ctx * kv_heads * group > 4 * 2048 * 4096 * 32):
            batch //= 2
        while new > 1 and batch * new * ctx * kv_heads * group > 4 * 2048 * 4096 * 32:
            new //= 2
        causal = rng.random() < 0.8
    else:
        ctx = _log(rng, 16, 32768)
        batch = _log(rng, 1, 96)
        while batch > 1 and batch * ctx * kv_heads > room // 4:
            batch //= 2
        new = _log(rng, 1, ctx) if op == "write" else 1
        causal = True
    return _case(None, op, elem, held, batch, new, ctx, ragged, kv_heads * group, kv_heads, dim,
                 page, causal)


def _lengths(case):
    """(new tokens, cached tokens in all) of each sequence: part of the case, not of the seed."""
    b, new, ctx = case["batch"], case["new"], case["ctx"]
    if not case["ragged"]:
        return np.full(b, new), np.full(b, ctx)
    r = np.random.RandomState((b * 1000003 + new * 10007 + ctx * 31 + case["page"]) % (1 << 31))
    n = r.randint((new + 1) // 2, new + 1, b)
    k = np.maximum(n, r.randint(max(1, ctx // 4), ctx + 1, b))
    n[0], k[0] = new, ctx
    return n, k


def _held(case):
    return KIND[case["elem"]] if case["held"] == "same" else HELD[case["held"]]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    n, k = _lengths(case)
    b, hk, d, ps = case["batch"], case["kv_heads"], case["dim"], case["page"]
    kind = KIND[case["elem"]]
    per = -(-k // ps)                                    # pages of each sequence
    pages = int(per.sum()) + 3                           # a few free ones, as a pool has
    table = np.zeros((b, int(per.max())), np.int32)
    order = np.random.RandomState(int(seed) % (1 << 31)).permutation(pages).astype(np.int32)
    at = 0
    for i in range(b):                                   # pages are handed out in no order
        table[i, : per[i]] = order[at: at + per[i]]
        at += per[i]

    def rand(*shape):
        # rows of unlike size, as heads and tokens have
        x = torch.randn(*shape, generator=g, device=dev)
        return x * torch.exp(0.4 * torch.randn(*shape[:-1], 1, generator=g, device=dev))

    def cut(lens):
        return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=dev)

    s = {"case": case, "table": torch.from_numpy(table).to(dev)}
    shape = (pages, ps, hk, d)
    for name in ("k", "v"):
        s[name + "_scale"] = None
        if case["op"] == "write":
            s[name] = torch.zeros(shape, device=dev, dtype=torch.uint8).view(torch.int8).to(_held(case))
            if case["held"] != "same":
                s[name + "_scale"] = torch.zeros(pages, hk, ps, device=dev)
        elif case["held"] == "same":
            s[name] = rand(*shape).to(kind)
        else:
            codes, scale = _quantise(rand(*shape).to(kind).float(), case["held"])
            s[name], s[name + "_scale"] = codes, scale.transpose(1, 2).contiguous()
    total_new, total = int(n.sum()), int(k.sum())
    if case["op"] == "write":
        pos = np.concatenate([np.arange(k[i] - n[i], k[i]) for i in range(b)])
        row = np.repeat(np.arange(b), n)
        s["slots"] = torch.from_numpy((table[row, pos // ps].astype(np.int64) * ps + pos % ps).astype(np.int32)).to(dev)
        s["starts"] = torch.from_numpy((k - n).astype(np.int32)).to(dev)
        s["cu"] = cut(n)
        s["new_k"], s["new_v"] = (rand(total_new, hk, d).to(kind) for _ in range(2))
        s["k_out"], s["v_out"] = torch.empty_like(s["new_k"]), torch.empty_like(s["new_k"])
    elif case["op"] == "read":
        s["starts"], s["cu"] = None, cut(k)
        s["k_out"], s["v_out"] = (torch.empty(total, hk, d, dtype=kind, device=dev) for _ in range(2))
    else:
        s["q"] = rand(total_new, case["heads"], d).to(kind)
        s["o"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(case["heads"], total_new, device=dev)
        s["cu"], s["max_new"] = cut(n), int(n.max())
        s["lens"] = torch.from_numpy(k.astype(np.int32)).to(dev)
        s["max_len"] = int(k.max())
    return s


def _quantise(x, held):
    """Codes and scales of 32-bit rows [..., d]."""
    amax = x.abs().amax(-1)
    top = torch.full_like(amax, TOP[held])
    full = amax > 0
    scale = torch.where(full, amax / top, torch.zeros_like(amax))
    v = x * torch.where(full, top / amax, torch.zeros_like(amax)).unsqueeze(-1)
    codes = torch.round(v).to(torch.int8) if held == "int8" else v.to(torch.float8_e4m3fn)
    return codes, scale


def _rows(s, name, page, offset):
    """Cached rows at (page, offset) as 32-bit values [..., heads, dim]."""
    c = s[name]
    if s[name + "_scale"] is None:
        return c[page, offset].float()
    codes = c.view(torch.int8)[page, offset].view(c.dtype).float()
    return codes * s[name + "_scale"][page, :, offset].unsqueeze(-1)


def _plain_write(s):
    ps = s["case"]["page"]
    slot = s["slots"].long()
    page, offset = slot // ps, slot % ps
    for name in ("k", "v"):
        x = s["new_" + name]
        if s[name + "_scale"] is None:
            s[name][page, offset] = x
        else:
            codes, scale = _quantise(x.float(), s["case"]["held"])
            s[name].view(torch.int8)[page, offset] = codes.view(torch.int8)
            s[name + "_scale"][page, :, offset] = scale


def _plain_read(s):
    ps, cu = s["case"]["page"], s["cu"].long()
    i = torch.arange(s["k_out"].shape[0], device=cu.device)
    seq = torch.searchsorted(cu, i, right=True) - 1
    pos = i - cu[seq]
    if s["starts"] is not None:
        pos = pos + s["starts"].long()[seq]
    page = s["table"].long()[seq, pos // ps]
    return tuple(_rows(s, name, page, pos % ps).to(s["k_out"].dtype) for name in ("k", "v"))


def _plain_attend(s):
    c = s["case"]
    ps, hk, group = c["page"], c["kv_heads"], c["heads"] // c["kv_heads"]
    dev = s["q"].device
    cu, lens = s["cu"].long(), s["lens"].long()
    new = cu[1:] - cu[:-1]
    # keys and values of every sequence, padded to the longest
    j = torch.arange(s["max_len"], device=dev)
    there = j[None, :] < lens[:, None]
    page = torch.where(there, s["table"].long()[:, j // ps], 0)
    keys, vals = (_rows(s, name, page, (j % ps).expand_as(page)) for name in ("k", "v"))
    vals = torch.where(there[:, :, None, None], vals, 0.0)
    # queries, padded the same way: [batch, kv head, group, query, dim]
    i = torch.arange(s["max_new"], device=dev)
    live = i[None, :] < new[:, None]
    q = s["q"][torch.where(live, cu[:-1, None] + i[None, :], 0)].float()
    q = q.unflatten(2, (hk, group)).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(q.flatten(2, 3), keys.permute(0, 2, 3, 1)) * (1 / math.sqrt(c["dim"]))
    scores = scores.unflatten(2, (group, -1))
    seen = there[:, None, :].expand(-1, len(i), -1)
    if c["causal"]:
        seen = seen & (j[None, None, :] <= i[None, :, None] + (lens - new)[:, None, None])
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    p = torch.exp(scores - top)
    del scores
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), vals.permute(0, 2, 1, 3)).unflatten(2, (group, -1))
    o = o / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total)).squeeze(-1)
    # back to packed rows
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[live].to(s["q"].dtype)
    lse = lse.permute(0, 3, 1, 2).flatten(2, 3)[live].t().contiguous()
    return o, lse


def _check(rc):
    if rc:
        raise RuntimeError("the call was declined or failed: %d" % rc)


def run(state):
    s = state
    op = s["case"]["op"]
    if not own:
        if op == "attend":
            o, lse = _plain_attend(s)
            return {"o": o, "lse": lse}
        if op == "write":
            _plain_write(s)
        k, v = _plain_read(s)
        return {"k": k, "v": v}
    from zlift_b200 import paged
    if "cache" not in s:                       # a serving program keeps it beside its pages
        s["cache"] = paged.KVCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if op == "attend":
        _check(paged.paged_attention(s["cache"], s["q"], s["o"], s["lse"], s["table"], s["cu"],
                                     s["lens"], max_q=s["max_new"], causal=s["case"]["causal"]))
        return {"o": s["o"], "lse": s["lse"]}
    if op == "write":
        _check(paged.kv_write(s["cache"], s["new_k"], s["new_v"], s["slots"]))
    _check(paged.kv_read(s["cache"], s["k_out"], s["v_out"], s["table"], s["cu"],
                         starts=s["starts"]))
    return {"k": s["k_out"], "v": s["v_out"]}


def work(case):
    n, k = (x.astype(np.int64) for x in _lengths(case))
    hk, h, d = case["kv_heads"], case["heads"], case["dim"]
    cell = 2 * d if case["held"] == "same" else d + 4    # a cached row, with its scale
    if case["op"] == "write":       # in, into the cache, and the values returned
        return {"bytes": int(n.sum()) * 2 * hk * (2 * d + cell + 2 * d), "flops": 0}
    if case["op"] == "read":
        return {"bytes": int(k.sum()) * 2 * hk * (cell + 2 * d), "flops": 0}
    if case["causal"]:              # query i sees k - n + i + 1 keys
        pairs = int((n * (k - n) + n * (n + 1) // 2).sum())
    else:
        pairs = int((n * k).sum())
    moved = int(k.sum()) * 2 * hk * cell + int(n.sum()) * h * (4 * d + 4)
    return {"bytes": moved, "flops": 4 * d * h * pairs}


def exact(case, seed):
    """The definition in 64 bits, one sequence and one key head at a time."""
    s = prepare(case, seed)
    n, k = _lengths(case)
    ps, hk, d = case["page"], case["kv_heads"], case["dim"]
    flat = {}

    def rounded(x):                                       # an 8-bit cache's value of rows x
        x = x.double()
        amax = x.abs().amax(-1, keepdim=True)
        scale = amax / TOP[case["held"]]
        y = torch.where(amax > 0, x / torch.where(amax > 0, scale, 1.0), 0.0)
        if case["held"] == "int8":
            return torch.round(y) * scale
        # e4m3: three mantissa bits, the smallest exponent is -6
        e = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -30))).clamp_min(-6.0)
        step = torch.exp2(e - 3)
        return torch.round(y / step) * step * scale

    if case["op"] == "write":
        return {w: s["new_" + w].double() if case["held"] == "same" else rounded(s["new_" + w])
                for w in ("k", "v")}
    for w in ("k", "v"):
        flat[w] = s[w].flatten(0, 1)
        if s[w + "_scale"] is not None:
            flat[w + "s"] = s[w + "_scale"].permute(0, 2, 1).flatten(0, 1)

    def cached(w, i, head):
        pos = torch.arange(int(k[i]), device=s["table"].device)
        slot = s["table"][i].long()[pos // ps] * ps + pos % ps
        x = flat[w][:, head].double()[slot]
        return x if w + "s" not in flat else x * flat[w + "s"][:, head].double()[slot][:, None]

    if case["op"] == "read":
        return {w: torch.cat([torch.stack([cached(w, i, h) for h in range(hk)], 1)
                              for i in range(case["batch"])]) for w in ("k", "v")}
    group = case["heads"] // hk
    o = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.empty(s["lse"].shape, dtype=torch.float64, device=s["q"].device)
    at = np.concatenate([[0], np.cumsum(n)])
    for i in range(case["batch"]):
        rows = slice(int(at[i]), int(at[i + 1]))
        reach = torch.arange(int(n[i]), device=o.device)[:, None] + int(k[i] - n[i])
        hidden = torch.arange(int(k[i]), device=o.device)[None, :] > reach
        for head in range(hk):
            keys, vals = cached("k", i, head), cached("v", i, head)
            for h in range(head * group, (head + 1) * group):
                z = s["q"][rows, h].double() @ keys.T / math.sqrt(d)
                if case["causal"]:
                    z = z.masked_fill(hidden, -math.inf)
                lse[h, rows] = torch.logsumexp(z, -1)
                o[rows, h] = torch.softmax(z, -1) @ vals
    return {"o": o, "lse": lse}
