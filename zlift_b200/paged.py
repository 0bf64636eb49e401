"""Python side of the paged K/V cache entry points (include/zlift_paged.h).

``KVCache`` describes cache tensors laid out [pages, page_size, heads, dim]
(any strides, dim contiguous); ``kv_write``, ``kv_read`` and
``paged_attention`` call the C entries with it.  Like the other attention
calls they fill buffers that the caller made, run on ``stream`` (None: the
legacy default stream, PyTorch's default) and return 0 done, 1 declined,
2 launch failure.  Tensors whose shapes or types contradict each other raise
``ValueError``, which the C side could not see.
"""
from __future__ import annotations

import ctypes
import math

from . import load

c_vp, c_ll, c_int, c_float, c_size = (ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int,
                                      ctypes.c_float, ctypes.c_size_t)

F16, BF16, F32, I8, E4M3 = 0, 1, 2, 3, 4


class CacheBlock(ctypes.Structure):
    """zlift_kv_cache"""
    _fields_ = [
        ("k", c_vp), ("v", c_vp), ("k_scale", c_vp), ("v_scale", c_vp),
        ("page_stride", c_ll), ("row_stride", c_ll), ("head_stride", c_ll),
        ("scale_page_stride", c_ll), ("scale_head_stride", c_ll),
        ("num_pages", c_int), ("page_size", c_int), ("heads", c_int), ("dim", c_int),
        ("type", c_int),
    ]


class RowsBlock(ctypes.Structure):
    """zlift_kv_rows"""
    _fields_ = [
        ("k", c_vp), ("v", c_vp),
        ("k_row_stride", c_ll), ("k_head_stride", c_ll),
        ("v_row_stride", c_ll), ("v_head_stride", c_ll),
        ("tokens", c_int), ("elem", c_int),
    ]


class AttnBlock(ctypes.Structure):
    """zlift_paged_attn_params"""
    _fields_ = [
        ("q", c_vp), ("o", c_vp), ("lse", c_vp),
        ("q_row_stride", c_ll), ("q_head_stride", c_ll),
        ("o_row_stride", c_ll), ("o_head_stride", c_ll), ("lse_head_stride", c_ll),
        ("cu_q", c_vp), ("seq_k", c_vp), ("page_table", c_vp), ("table_stride", c_ll),
        ("table_pages", c_int), ("batch", c_int), ("total_q", c_int), ("max_q", c_int),
        ("heads", c_int), ("elem", c_int), ("causal", c_int), ("scale", c_float),
        ("workspace", c_vp), ("workspace_bytes", c_size),
    ]


assert ctypes.sizeof(CacheBlock) == 96 and CacheBlock.num_pages.offset == 72
assert ctypes.sizeof(RowsBlock) == 56 and RowsBlock.tokens.offset == 48
assert ctypes.sizeof(AttnBlock) == 144 and AttnBlock.workspace.offset == 128

_types = None


def _type(t) -> int:
    global _types
    if _types is None:
        import torch
        _types = {torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32,
                  torch.int8: I8, torch.float8_e4m3fn: E4M3}
    kind = _types.get(t.dtype)
    if kind is None:
        raise ValueError(f"no such element type: {t.dtype}")
    return kind


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _index(t, dims, what):
    import torch
    _need(t.dtype == torch.int32 and t.dim() == dims and t.is_cuda and
          (t.numel() < 2 or t.stride(-1) == 1),
          f"{what}: an int32 CUDA tensor of {dims} dimension(s), contiguous along the last")
    return t


def _stream(stream) -> int:
    return 0 if stream is None else int(getattr(stream, "cuda_stream", stream))


class KVCache:
    """A cache's tensors and their description.

    k, v          [pages, page_size, heads, dim], both with the same strides:
                  float16 or bfloat16, or int8 / float8_e4m3fn with scales
    k_scale, v_scale   float32 [pages, heads, page_size], page_size contiguous
    """

    def __init__(self, k, v, k_scale=None, v_scale=None):
        import torch
        _need(k.dim() == 4 and k.shape == v.shape and k.stride() == v.stride() and
              k.dtype == v.dtype and k.is_cuda and k.device == v.device,
              "k and v: [pages, page_size, heads, dim] CUDA tensors of one type and layout")
        _need(k.stride(3) == 1 or k.shape[3] == 1, "dim is not contiguous")
        kind = _type(k)
        _need(kind != F32, "a cache holds 16 or 8 bits")
        b = CacheBlock()
        b.type = kind
        b.k, b.v = k.data_ptr(), v.data_ptr()
        b.page_stride, b.row_stride, b.head_stride = k.stride(0), k.stride(1), k.stride(2)
        b.num_pages, b.page_size, b.heads, b.dim = k.shape
        _need((kind >= I8) == (k_scale is not None) == (v_scale is not None),
              "an 8-bit cache has scales for k and v, a 16-bit one has none")
        if k_scale is not None:
            shape = (k.shape[0], k.shape[2], k.shape[1])
            for s in (k_scale, v_scale):
                _need(tuple(s.shape) == shape and s.dtype == torch.float32 and
                      s.device == k.device and s.stride() == k_scale.stride() and
                      (s.stride(2) == 1 or s.shape[2] == 1),
                      "scales: float32 [pages, heads, page_size], page_size contiguous")
            b.k_scale, b.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
            b.scale_page_stride, b.scale_head_stride = k_scale.stride(0), k_scale.stride(1)
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.type, self.heads, self.dim, self.device = kind, b.heads, b.dim, k.device
        self.block = b
        self.ref = ctypes.byref(b)

    def _rows(self, k, v):
        _need(k.dim() == 3 and k.shape == v.shape and k.shape[1] == self.heads and
              k.shape[2] == self.dim and k.dtype == v.dtype and k.device == self.device and
              v.device == self.device and k.stride(2) == v.stride(2) == 1,
              "k and v: [tokens, heads, dim] of the cache's heads, dim and device")
        r = RowsBlock()
        r.k, r.v = k.data_ptr(), v.data_ptr()
        r.k_row_stride, r.k_head_stride, _ = k.stride()
        r.v_row_stride, r.v_head_stride, _ = v.stride()
        r.tokens, r.elem = k.shape[0], _type(k)
        return r


def kv_write(cache: KVCache, k, v, slots, stream=None) -> int:
    """Writes packed k, v [tokens, heads, dim] into slots [tokens] (int32:
    page * page_size + offset; negative: skipped)."""
    r = cache._rows(k, v)
    _need(_index(slots, 1, "slots").shape[0] == r.tokens, "one slot for each token")
    return load().zlift_kv_write(cache.ref, ctypes.byref(r), slots.data_ptr(), _stream(stream))


def kv_read(cache: KVCache, k_out, v_out, page_table, cu, starts=None, stream=None) -> int:
    """Reads tokens cu[s]..cu[s+1] of k_out, v_out [tokens, heads, dim] from
    positions starts[s] (default 0) onwards of sequence s, whose pages are
    page_table[s]."""
    r = cache._rows(k_out, v_out)
    _index(page_table, 2, "page_table")
    batch = _index(cu, 1, "cu").shape[0] - 1
    _need(batch >= 0 and page_table.shape[0] == batch, "cu has one entry more than page_table rows")
    if starts is not None:
        _need(_index(starts, 1, "starts").shape[0] == batch, "one start for each sequence")
    return load().zlift_kv_read(cache.ref, ctypes.byref(r), page_table.data_ptr(),
                                page_table.stride(0), page_table.shape[1],
                                None if starts is None else starts.data_ptr(), cu.data_ptr(),
                                batch, _stream(stream))


_workspaces = {}


def _workspace(device, stream: int, nbytes: int):
    """The workspace of a device and stream: zeroed when made, replaced when a
    call wants more.  Made on that stream, so an older one is reused only
    after the work that still reads it."""
    import torch
    ws = _workspaces.get((device, stream))
    if ws is None or ws.numel() < nbytes:
        on = torch.cuda.ExternalStream(stream, device=device) if stream else \
            torch.cuda.default_stream(device)
        with torch.cuda.stream(on):
            ws = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        _workspaces[(device, stream)] = ws
    return ws


def paged_attention(cache: KVCache, q, o, lse, page_table, cu_q, seq_k, max_q, causal=True,
                    scale=None, stream=None, workspace=None) -> int:
    """Attention of packed queries q [total_q, heads, dim] over the cache:
    rows cu_q[s]..cu_q[s+1] are the newest tokens of sequence s, which holds
    seq_k[s] tokens in the pages page_table[s].  o is like q; lse float32
    [heads, total_q] or None.  max_q: the longest chunk, on the host.

    workspace: a zeroed uint8 CUDA tensor of ``attention_workspace`` bytes
    that no concurrent call uses; by default one per device and stream is
    kept (make one call outside a graph capture first, so that it exists).
    """
    import torch
    _need(q.dim() == 3 and q.shape == o.shape and q.dtype == o.dtype and
          q.shape[2] == cache.dim and q.device == cache.device and o.device == cache.device and
          q.stride(2) == o.stride(2) == 1, "q and o: [total_q, heads, dim] of one type")
    _index(page_table, 2, "page_table")
    batch = _index(seq_k, 1, "seq_k").shape[0]
    _need(_index(cu_q, 1, "cu_q").shape[0] == batch + 1 and page_table.shape[0] == batch,
          "cu_q has one entry more than seq_k and page_table rows")
    p = AttnBlock()
    p.q, p.o = q.data_ptr(), o.data_ptr()
    p.q_row_stride, p.q_head_stride, _ = q.stride()
    p.o_row_stride, p.o_head_stride, _ = o.stride()
    if lse is not None:
        _need(lse.dtype == torch.float32 and lse.shape == (q.shape[1], q.shape[0]) and
              (lse.stride(1) == 1 or lse.shape[1] < 2) and lse.device == cache.device,
              "lse: float32 [heads, total_q]")
        p.lse, p.lse_head_stride = lse.data_ptr(), lse.stride(0)
    p.cu_q, p.seq_k, p.page_table = cu_q.data_ptr(), seq_k.data_ptr(), page_table.data_ptr()
    p.table_stride, p.table_pages = page_table.stride(0), page_table.shape[1]
    p.batch, p.total_q, p.max_q, p.heads = batch, q.shape[0], int(max_q), q.shape[1]
    p.elem, p.causal = _type(q), 1 if causal else 0
    p.scale = 1.0 / math.sqrt(cache.dim) if scale is None else scale
    lib, ref, s = load(), ctypes.byref(p), _stream(stream)
    if workspace is None:
        nbytes = lib.zlift_paged_attn_workspace(cache.ref, ref)
        if nbytes:
            workspace = _workspace(cache.device, s, nbytes)
    if workspace is not None:
        p.workspace, p.workspace_bytes = workspace.data_ptr(), workspace.numel()
    return lib.zlift_paged_attn(cache.ref, ref, s)


def attention_workspace(cache: KVCache, heads, total_q, max_q, batch, elem=None) -> int:
    """Bytes of workspace that such calls of ``paged_attention`` want."""
    p = AttnBlock()
    p.batch, p.total_q, p.max_q, p.heads = batch, total_q, max_q, heads
    p.elem = cache.type if cache.type < I8 else (BF16 if elem is None else elem)
    p.scale = 1.0
    fake = 256                       # not followed: only sizes are looked at
    p.q = p.o = p.cu_q = p.seq_k = p.page_table = fake
    p.q_row_stride = p.o_row_stride = heads * cache.dim
    p.q_head_stride = p.o_head_stride = cache.dim
    return load().zlift_paged_attn_workspace(cache.ref, ctypes.byref(p))
