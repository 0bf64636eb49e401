"""Captured attention calls keep their workspace, on the GPU."""
import pytest

from tests.test_paged_gpu import Case

pytestmark = pytest.mark.gpu


def test_a_graph_keeps_its_workspace(cuda):
    """Larger calls on the stream of a capture replace the workspace that later
    calls use; the graph's stays its own."""
    import torch
    from zlift_b200 import paged
    one = Case("bf16", "same", new=(1, 1), ctx=(9000, 211), heads=8, kv_heads=2, dim=128, seed=4)
    few = Case("bf16", "same", new=(5, 3), ctx=(3000, 40), heads=8, kv_heads=2, dim=128, seed=5)
    chunk = Case("bf16", "same", new=(150,), ctx=(2000,), heads=8, kv_heads=2, dim=128, seed=6)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    before = paged._workspaces.pop((one.cache.device, s.cuda_stream), None)   # (handles are reused)
    with torch.cuda.stream(s):
        o, lse = one.run(stream=s)
        mine = paged._workspaces[(one.cache.device, s.cuda_stream)]
        place = mine.data_ptr(), mine.data_ptr() + mine.numel()
        del mine
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            assert paged.paged_attention(one.cache, one.q, o, lse, one.table, one.cu, one.lens, 1,
                                         stream=s) == 0
        few.check(stream=s)
        chunk.check(stream=s)
        fill = [torch.full((3 << 20,), 0x5a, dtype=torch.uint8, device=cuda) for _ in range(64)]
        assert all(f.data_ptr() + f.numel() <= place[0] or f.data_ptr() >= place[1] for f in fill)
        for _ in range(3):
            o.fill_(7)
            lse.fill_(7)
            graph.replay()
            s.synchronize()
            eo, el, to, tl = one.exact()
            assert ((o.double() - eo).abs() <= to).all() and ((lse.double() - el).abs() <= tl).all()
        assert all(bool((f == 0x5a).all()) for f in fill)
        chunk.check(stream=s)
    del before
