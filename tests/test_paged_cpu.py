"""CPU: the paged-cache entries of include/zlift_paged.h are exported, their
structures match the Python images, and what they refuse is refused before
any launch."""
import ctypes
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_entries_are_exported(built_lib):
    import zlift_b200
    src = open(os.path.join(ROOT, "include", "zlift_paged.h")).read()
    names = set(re.findall(r"ZLIFT_API\s+(?:int|size_t)\s+(\w+)\s*\(", src))
    assert len(names) == 4
    out = subprocess.run(["nm", "-D", "--defined-only", zlift_b200.LIBCUBLAS], capture_output=True,
                         text=True, check=True).stdout
    assert names <= {line.split()[-1] for line in out.splitlines() if " T " in line}
    assert names <= {n for n, _, _ in zlift_b200.SIGNATURES}


def test_header_compiles_as_c_with_the_same_layout(tmp_path):
    from zlift_b200 import paged
    lines = ["#include <stdio.h>", '#include "zlift_paged.h"', "int main(void) {"]
    want = []
    for py, c in ((paged.CacheBlock, "zlift_kv_cache"), (paged.RowsBlock, "zlift_kv_rows"),
                  (paged.AttnBlock, "zlift_paged_attn_params")):
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        want.append(ctypes.sizeof(py))
        for name, _ in py._fields_:
            lines.append(f'printf("%zu\\n", offsetof({c}, {name}));')
            want.append(getattr(py, name).offset)
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-o", str(exe),
                    str(src)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in got] == want


def _cache(**kw):
    from zlift_b200 import paged
    b = paged.CacheBlock()
    b.k = b.v = 0x10000
    b.num_pages, b.page_size, b.heads, b.dim, b.type = 8, 16, 2, 128, paged.BF16
    b.page_stride, b.row_stride, b.head_stride = 16 * 256, 256, 128
    b.scale_page_stride, b.scale_head_stride = 32, 16
    for k, v in kw.items():
        setattr(b, k, v)
    return b


def _rows(**kw):
    from zlift_b200 import paged
    r = paged.RowsBlock()
    r.k = r.v = 0x10000
    r.k_row_stride = r.v_row_stride = 256
    r.k_head_stride = r.v_head_stride = 128
    r.tokens, r.elem = 4, paged.BF16
    for k, v in kw.items():
        setattr(r, k, v)
    return r


BAD_CACHES = [dict(k=None), dict(v=None), dict(type=2), dict(type=5), dict(type=-1), dict(type=3),
              dict(type=4, k_scale=0x1000), dict(num_pages=0), dict(page_size=0), dict(heads=0),
              dict(dim=0), dict(num_pages=1 << 28, page_size=16), dict(heads=-2), dict(dim=1 << 20)]


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_bad_caches_are_declined(built_lib, bad):
    c = _cache(**bad)
    r = _rows()
    assert built_lib.zlift_kv_write(ctypes.byref(c), ctypes.byref(r), 0x1000, None) == 1
    assert built_lib.zlift_kv_read(ctypes.byref(c), ctypes.byref(r), 0x1000, 4, 4, None, 0x1000, 1,
                                   None) == 1
    p = _params()
    assert built_lib.zlift_paged_attn(ctypes.byref(c), ctypes.byref(p), None) == 1
    assert built_lib.zlift_paged_attn_workspace(ctypes.byref(c), ctypes.byref(p)) == 0


def test_write_and_read_refusals(built_lib):
    c = _cache()

    def write(r, slots=0x1000):
        return built_lib.zlift_kv_write(ctypes.byref(c), r and ctypes.byref(r), slots, None)

    def read(r, table=0x1000, pages=4, cu=0x1000, batch=1):
        return built_lib.zlift_kv_read(ctypes.byref(c), r and ctypes.byref(r), table, 4, pages, None,
                                       cu, batch, None)

    assert built_lib.zlift_kv_write(None, ctypes.byref(_rows()), 0x1000, None) == 1
    for f in (write, read):
        assert f(None) == 1
        assert f(_rows(elem=0)) == 1                         # another 16-bit type
        assert f(_rows(elem=2)) == 1                         # fp32 and a 16-bit cache
        assert f(_rows(elem=7)) == 1
        assert f(_rows(tokens=-1)) == 1
        assert f(_rows(k=None)) == 1
        assert f(_rows(v=None)) == 1
        assert f(_rows(tokens=0, k=None)) == 0               # nothing to do
    assert write(_rows(), slots=None) == 1
    assert read(_rows(), cu=None) == 1
    assert read(_rows(), table=None) == 1
    assert read(_rows(), batch=-1) == 1
    assert read(_rows(), pages=-1) == 1
    assert read(_rows(), pages=1 << 28) == 1
    assert read(_rows(), batch=0) == 0
    c.type, c.k_scale, c.v_scale = 3, 0x1000, 0x1000
    assert write(_rows(elem=2)) == 1                         # fp32 is an output only


def _params(**kw):
    from zlift_b200 import paged
    p = paged.AttnBlock()
    p.q = p.o = 0x10000
    p.cu_q = p.seq_k = p.page_table = 0x1000
    p.q_row_stride = p.o_row_stride = 1024
    p.q_head_stride = p.o_head_stride = 128
    p.table_stride = p.table_pages = 4
    p.batch, p.total_q, p.max_q, p.heads, p.elem, p.causal, p.scale = 2, 2, 1, 8, paged.BF16, 1, 0.1
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(o=None), dict(cu_q=None), dict(seq_k=None), dict(page_table=None),
    dict(elem=0), dict(elem=2), dict(elem=3), dict(batch=-1), dict(total_q=-1), dict(table_pages=-1),
    dict(heads=0), dict(heads=3), dict(heads=-8), dict(table_pages=1 << 28)])
def test_attention_refusals(built_lib, bad):
    c, p = _cache(), _params(**bad)
    assert built_lib.zlift_paged_attn(ctypes.byref(c), ctypes.byref(p), None) == 1
    assert built_lib.zlift_paged_attn_workspace(ctypes.byref(c), ctypes.byref(p)) == 0


def test_attention_of_nothing(built_lib):
    c = _cache()
    assert built_lib.zlift_paged_attn(ctypes.byref(c), None, None) == 1
    assert built_lib.zlift_paged_attn(None, ctypes.byref(_params()), None) == 1
    for p in (_params(batch=0), _params(total_q=0), _params(batch=0, q=None, cu_q=None)):
        assert built_lib.zlift_paged_attn(ctypes.byref(c), ctypes.byref(p), None) == 0
    c.dim = 257
    assert built_lib.zlift_paged_attn(ctypes.byref(c), ctypes.byref(_params()), None) == 1


def test_python_checks(built_lib):
    """Contradicting tensors raise before anything reaches the library."""
    import torch
    from zlift_b200 import paged
    k = torch.zeros(4, 16, 2, 8, dtype=torch.float16)
    with pytest.raises(ValueError):
        paged.KVCache(k, k)                                  # not on a GPU
    with pytest.raises(ValueError):
        paged._type(torch.zeros(2, dtype=torch.float64))
    with pytest.raises(ValueError):
        paged._index(torch.zeros(3, dtype=torch.int32), 0, "slots")
    with pytest.raises(ValueError):
        paged._table(torch.zeros(3, 4, dtype=torch.int32), 0)
