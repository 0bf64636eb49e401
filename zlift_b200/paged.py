"""Python side of the paged K/V cache entry points (include/zlift_paged.h).

``KVCache`` describes cache tensors laid out [pages, page_size, heads, dim]
(any strides, dim contiguous); ``kv_write``, ``kv_read`` and
``paged_attention`` call the C entries with it.  Like the other attention
calls they fill buffers that the caller made, run on ``stream`` (None: the
legacy default stream, PyTorch's default) and return 0 done, 1 declined,
2 launch failure.  Tensors whose shapes or types contradict each other, or
whose GPU is not the current device (on which the C entries launch), raise
``ValueError``, which the C side could not see.
"""
from __future__ import annotations

import ctypes
import math
import struct

import torch

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

# The structures are packed by hand in the calls below: filling a ctypes
# Structure field by field costs several times as much.
_rows_struct = struct.Struct("=2Q4q2i")
_attn_struct = struct.Struct("=3Q5q3Qq7if2Q")
assert _rows_struct.size == ctypes.sizeof(RowsBlock)
assert _attn_struct.size == ctypes.sizeof(AttnBlock)

_types = {torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32, torch.int8: I8,
          torch.float8_e4m3fn: E4M3}
_int32 = torch.int32


def _type(t) -> int:
    kind = _types.get(t.dtype)
    if kind is None:
        raise ValueError(f"no such element type: {t.dtype}")
    return kind


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _index(t, device, what):
    """A one-dimensional index tensor on a device; returns its length."""
    shape = t.shape
    if t.dtype is not _int32 or len(shape) != 1 or t.get_device() != device or \
            not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous int32 tensor of one dimension on the cache's GPU")
    return shape[0]


def _table(t, device):
    """A page table; returns its shape and row stride."""
    shape = t.shape
    if t.dtype is not _int32 or len(shape) != 2 or t.get_device() != device:
        raise ValueError("page_table: int32 [batch, pages] on the cache's GPU")
    stride, one = t.stride()
    if one != 1 and shape[1] > 1:
        raise ValueError("page_table: a row's pages are contiguous")
    return shape[0], shape[1], stride


_one_gpu = None         # in this process: then it is the current one (asking costs 1 us of a call's 6)


def _on(device):
    global _one_gpu
    if _one_gpu is None:
        _one_gpu = torch.cuda.device_count() == 1
    if not _one_gpu and torch.cuda.current_device() != device:
        raise ValueError("the cache's GPU is not the current device")


def _stream(stream) -> int:
    return 0 if stream is None else int(getattr(stream, "cuda_stream", stream))


class KVCache:
    """A cache's tensors and their description.

    k, v          [pages, page_size, heads, dim], both with the same strides:
                  float16 or bfloat16, or int8 / float8_e4m3fn with scales
    k_scale, v_scale   float32 [pages, heads, page_size], page_size contiguous
    """

    def __init__(self, k, v, k_scale=None, v_scale=None):
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
        self.type, self.heads, self.dim, self.device = kind, b.heads, b.dim, k.get_device()
        self.softmax_scale = 1.0 / math.sqrt(b.dim)
        self.block = b
        self.ref = ctypes.byref(b)

    def _rows(self, k, v):
        """zlift_kv_rows of packed k, v, and the number of tokens."""
        shape, kind, device = k.shape, k.dtype, self.device
        if len(shape) != 3 or shape != v.shape or shape[1] != self.heads or \
                shape[2] != self.dim or v.dtype is not kind or k.get_device() != device or \
                v.get_device() != device:
            raise ValueError("k and v: [tokens, heads, dim] of one type, of the cache's heads, "
                             "dim and GPU")
        kr, kh, k1 = k.stride()
        vr, vh, v1 = v.stride()
        if (k1 != 1 or v1 != 1) and shape[2] > 1:
            raise ValueError("k and v: dim is not contiguous")
        _on(device)
        return _rows_struct.pack(k.data_ptr(), v.data_ptr(), kr, kh, vr, vh, shape[0],
                                 _type(k)), shape[0]


def kv_write(cache: KVCache, k, v, slots, stream=None) -> int:
    """Writes packed k, v [tokens, heads, dim] into slots [tokens] (int32:
    page * page_size + offset; negative: skipped; otherwise no two alike)."""
    rows, tokens = cache._rows(k, v)
    if _index(slots, cache.device, "slots") != tokens:
        raise ValueError("one slot for each token")
    return load().zlift_kv_write(cache.ref, rows, slots.data_ptr(),
                                 0 if stream is None else _stream(stream))


def kv_read(cache: KVCache, k_out, v_out, page_table, cu, starts=None, stream=None) -> int:
    """Reads tokens cu[s]..cu[s+1] of k_out, v_out [tokens, heads, dim] from
    positions starts[s] (default 0) onwards of sequence s, whose pages are
    page_table[s]."""
    rows, _ = cache._rows(k_out, v_out)
    batch, pages, stride = _table(page_table, cache.device)
    if _index(cu, cache.device, "cu") != batch + 1:
        raise ValueError("cu has one entry more than page_table has rows")
    if starts is not None and _index(starts, cache.device, "starts") != batch:
        raise ValueError("one start for each sequence")
    return load().zlift_kv_read(cache.ref, rows, page_table.data_ptr(), stride, pages,
                                None if starts is None else starts.data_ptr(), cu.data_ptr(),
                                batch, 0 if stream is None else _stream(stream))


_workspaces = {}        # (device, stream): the one that calls use now
_outgrown = []          # those before it: captured graphs may still use them


def _workspace(device: int, stream: int, nbytes: int):
    """The workspace of a device and stream: zeroed when made, replaced when a
    call wants more.  The old one stays allocated, since a graph captured with
    it goes on using it (a stream needs a few sizes at most, some 100 MB in
    all)."""
    on = torch.cuda.ExternalStream(stream, device=device) if stream else \
        torch.cuda.default_stream(device)
    with torch.cuda.stream(on):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("no workspace for this stream yet: call once before the capture, "
                               "or pass workspace=")
        ws = torch.zeros(nbytes, dtype=torch.uint8, device=torch.device("cuda", device))
    if (device, stream) in _workspaces:
        _outgrown.append(_workspaces[(device, stream)])
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
    kept for good (make one call outside a graph capture first, so that it
    exists).  A captured graph goes on using the workspace of its capture, so
    its replays and the calls on that stream must run one after another, or
    the capture be given a workspace of its own.
    """
    device, kind, shape = cache.device, q.dtype, q.shape
    if len(shape) != 3 or shape != o.shape or o.dtype is not kind or shape[2] != cache.dim or \
            q.get_device() != device or o.get_device() != device:
        raise ValueError("q and o: [total_q, heads, dim] of one type, of the cache's dim and GPU")
    total, heads, _ = shape
    qr, qh, q1 = q.stride()
    orow, oh, o1 = o.stride()
    if (q1 != 1 or o1 != 1) and shape[2] > 1:
        raise ValueError("q and o: dim is not contiguous")
    batch, pages, table_stride = _table(page_table, device)
    if _index(seq_k, device, "seq_k") != batch or _index(cu_q, device, "cu_q") != batch + 1:
        raise ValueError("seq_k has as many entries as page_table has rows, cu_q one more")
    lse_ptr = lse_stride = 0
    if lse is not None:
        lse_stride, l1 = lse.stride()
        if lse.dtype is not torch.float32 or lse.shape != (heads, total) or \
                (l1 != 1 and total > 1) or lse.get_device() != device:
            raise ValueError("lse: float32 [heads, total_q], total_q contiguous")
        lse_ptr = lse.data_ptr()
    _on(device)
    lib, s = load(), 0 if stream is None else _stream(stream)
    ws = workspace if workspace is not None else _workspaces.get((device, s))
    while True:
        p = _attn_struct.pack(q.data_ptr(), o.data_ptr(), lse_ptr, qr, qh, orow, oh, lse_stride,
                              cu_q.data_ptr(), seq_k.data_ptr(), page_table.data_ptr(),
                              table_stride, pages, batch, total, int(max_q), heads, _type(q),
                              1 if causal else 0, cache.softmax_scale if scale is None else scale,
                              0 if ws is None else ws.data_ptr(),
                              0 if ws is None else ws.numel())
        rc = lib.zlift_paged_attn(cache.ref, p, s)
        if rc != 1 or workspace is not None:
            return rc
        # declined: perhaps for want of (more) workspace
        nbytes = lib.zlift_paged_attn_workspace(cache.ref, p)
        if not nbytes or (ws is not None and ws.numel() >= nbytes):
            return rc
        ws = _workspace(device, s, nbytes)


def attention_workspace(cache: KVCache, heads, total_q, max_q, batch, elem=None) -> int:
    """Bytes of workspace that such calls of ``paged_attention`` want (on
    operands that the tensor cores can take)."""
    if elem is None:
        elem = cache.type if cache.type < I8 else BF16
    fake = 256                       # not followed: only sizes are looked at
    row, head = heads * cache.dim, cache.dim
    p = _attn_struct.pack(fake, fake, 0, row, head, row, head, 0, fake, fake, fake, 0, 0, batch,
                          total_q, max_q, heads, elem, 1, 1.0, 0, 0)
    return load().zlift_paged_attn_workspace(cache.ref, p)
