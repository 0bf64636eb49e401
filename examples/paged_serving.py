"""One attention layer served from a paged 8-bit cache, through the public calls.

Prompts of unlike lengths enter in chunks, then every sequence decodes a token
at a time and, at the end, scores a few drafted tokens together:

  QKV and output projections   cublasGemmEx (blas.Handle.gemm_ex)
  K and V into the cache       paged.kv_write (quantising)
  attention over the pages     paged.paged_attention
  a sequence read back         paged.kv_read

and the last step is checked against attention over the same tokens in one
piece: flash_forward on the K and V that kv_read returns.

Run: python examples/paged_serving.py [int8|fp8|bf16]
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import zlift_b200  # noqa: E402
from zlift_b200 import blas, paged  # noqa: E402

HEADS, KV_HEADS, DIM, PAGE = 8, 2, 128, 16
WIDTH = HEADS * DIM


class Layer:
    def __init__(self, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: (torch.randn(*s, generator=g, device="cuda") / math.sqrt(s[-1])).bfloat16()  # noqa: E731
        self.qkv = rand((HEADS + 2 * KV_HEADS) * DIM, WIDTH)
        self.out = rand(WIDTH, WIDTH)
        self.handle = blas.Handle()

    def project(self, x, w):
        """x [tokens, in] times w [out, in] transposed, in bf16."""
        y = torch.empty(x.shape[0], w.shape[0], dtype=torch.bfloat16, device="cuda")
        st = self.handle.gemm_ex(1, 0, w.shape[0], x.shape[0], w.shape[1], 1.0, w, blas.R_16BF,
                                 w.shape[1], x, blas.R_16BF, w.shape[1], 0.0, y, blas.R_16BF,
                                 w.shape[0])
        assert st == 0, f"gemm_ex returned {st}"
        return y


class Server:
    """Sequences, their pages and the cache."""

    def __init__(self, layer, batch, most_tokens, held):
        self.layer, self.batch = layer, batch
        per = -(-most_tokens // PAGE)
        shape = (batch * per, PAGE, KV_HEADS, DIM)
        kind = {"int8": torch.int8, "fp8": torch.float8_e4m3fn, "bf16": torch.bfloat16}[held]
        k, v = (torch.empty(shape, dtype=kind, device="cuda") for _ in range(2))
        scales = [None, None] if held == "bf16" else \
            [torch.empty(shape[0], KV_HEADS, PAGE, device="cuda") for _ in range(2)]
        self.cache = paged.KVCache(k, v, *scales)
        self.free = torch.randperm(shape[0]).tolist()
        self.pages = [[] for _ in range(batch)]
        self.table = torch.zeros(batch, per, dtype=torch.int32, device="cuda")
        self.lens = [0] * batch

    def step(self, xs):
        """New tokens xs[i] [n_i, WIDTH] of every sequence (n_i may be 0): their
        layer outputs, packed, and the queries' log-sum-exps."""
        new = [x.shape[0] for x in xs]
        slots = []
        for i, n in enumerate(new):
            while len(self.pages[i]) * PAGE < self.lens[i] + n:
                self.table[i, len(self.pages[i])] = self.free[-1]
                self.pages[i].append(self.free.pop())
            slots += [self.pages[i][p // PAGE] * PAGE + p % PAGE
                      for p in range(self.lens[i], self.lens[i] + n)]
            self.lens[i] += n
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        qkv = self.layer.project(torch.cat(xs), self.layer.qkv).view(-1, HEADS + 2 * KV_HEADS, DIM)
        q, k, v = qkv.split([HEADS, KV_HEADS, KV_HEADS], 1)
        assert paged.kv_write(self.cache, k, v, i32(slots)) == 0
        o = torch.empty(sum(new), HEADS, DIM, dtype=torch.bfloat16, device="cuda")
        lse = torch.empty(HEADS, sum(new), device="cuda")
        cu = [sum(new[:i]) for i in range(self.batch + 1)]
        assert paged.paged_attention(self.cache, q, o, lse, self.table, i32(cu), i32(self.lens),
                                     max_q=max(new)) == 0
        return self.layer.project(o.view(-1, WIDTH), self.layer.out), q, o, lse

    def read(self, i):
        """K and V of sequence i, contiguous."""
        k, v = (torch.empty(self.lens[i], KV_HEADS, DIM, dtype=torch.bfloat16, device="cuda")
                for _ in range(2))
        cu = torch.tensor([0, self.lens[i]], dtype=torch.int32, device="cuda")
        assert paged.kv_read(self.cache, k, v, self.table[i:i + 1], cu) == 0
        return k, v


def main(held="int8"):
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda n: torch.randn(n, WIDTH, generator=g, device="cuda").bfloat16()  # noqa: E731
    prompts = [300, 17, 129]
    server = Server(Layer(), len(prompts), 400, held)
    left = list(prompts)
    while any(left):                                     # prefill, 128 tokens at a time
        take = [min(128, n) for n in left]
        server.step([rand(n) for n in take])
        left = [a - b for a, b in zip(left, take)]
    for _ in range(5):                                   # decode
        server.step([rand(1) for _ in prompts])
    new = [4, 1, 3]                                      # drafted tokens
    y, q, o, lse = server.step([rand(n) for n in new])
    assert torch.isfinite(y.float()).all()
    worst, at = 0.0, 0
    for i, n in enumerate(new):
        k, v = server.read(i)
        whole = torch.empty(1, n, HEADS, DIM, dtype=torch.bfloat16, device="cuda")
        wlse = torch.empty(1, HEADS, n, device="cuda")
        assert zlift_b200.flash_forward(q[None, at:at + n].contiguous(), k[None], v[None], whole, wlse,
                                        causal=True) == 0
        worst = max(worst, (whole[0].float() - o[at:at + n].float()).abs().max().item()
                    / v.float().abs().max().item())
        assert (wlse[0] - lse[:, at:at + n]).abs().max().item() < 0.05
        at += n
    torch.cuda.synchronize()
    assert blas.device_error() == 0
    # bf16 rounds K, V (read back), the weights and O: 2^-8 each
    assert worst < 4 * 2.0 ** -8, worst
    print(f"{held}: {server.lens} tokens cached, largest difference {worst:.2e} of the largest value")


if __name__ == "__main__":
    main(*sys.argv[1:2])
