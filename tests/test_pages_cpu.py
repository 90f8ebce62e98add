"""No GPU: what the paged operators refuse, before anything is launched."""
import ctypes as C

import pytest
import torch

from mesh_llm_b200 import build, capi

P = 1 << 20  # an address that no call may follow


def cache(**kw):
    d = dict(k=P, v=P, k_scale=None, v_scale=None, n_pages=4, page_stride=0, type=capi.TYPE_F16, page_size=16, n_kv=2, head_dim=128)
    d.update(kw)
    return capi.KvPages(**d)


def batch(**kw):
    d = dict(row_start=P, pos0=P, table=P, rows=3, n_seq=1, table_len=4, table_stride=4)
    d.update(kw)
    return capi.PageBatch(**d)


def append(c=None, b=None, type=0, k=P, ks=256, v=P, vs=256, theta=1e4):
    build.build()
    return capi.lib().b200_kv_pages_append(C.byref(c or cache()), C.byref(b or batch()), type, k, ks, v, vs, theta, 1, None)


def attend(c=None, b=None, type=0, q=P, qs=1024, n_head=8, most=1, theta=1e4, window=0, scale=0.0, out=2 * P, os=1024, scratch=P, nbytes=1 << 40):
    build.build()
    return capi.lib().b200_attention_pages(C.byref(c or cache()), C.byref(b or batch()), type, q, qs, n_head, most, theta, 1, window, scale, out, os,
                                           scratch, nbytes, None)


BAD_CACHE = [dict(type=0), dict(type=8), dict(head_dim=96), dict(head_dim=256), dict(page_size=8), dict(page_size=24), dict(page_size=0), dict(page_size=8192),
             dict(n_kv=0), dict(n_pages=0), dict(n_pages=1 << 40), dict(k=None), dict(v=P + 8), dict(page_stride=100), dict(page_stride=2 * 16 * 128 + 4),
             dict(type=capi.TYPE_F8_E4M3), dict(type=capi.TYPE_F8_E4M3, k_scale=P, v_scale=P + 2)]
BAD_BATCH = [dict(rows=-1), dict(rows=1 << 40), dict(n_seq=-1), dict(row_start=None), dict(pos0=None), dict(table=None), dict(pos0=P + 2), dict(table_len=-1),
             dict(table_len=5), dict(table_len=1 << 28, table_stride=1 << 28), dict(table_len=(1 << 27) - 255, table_stride=1 << 27)]


@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_caches_refused(bad):
    assert append(cache(**bad)) == -1 and attend(cache(**bad)) == -1


@pytest.mark.parametrize("bad", BAD_BATCH, ids=str)
def test_batches_refused(bad):
    assert append(b=batch(**bad)) == -1 and attend(b=batch(**bad)) == -1


@pytest.mark.parametrize("bad", [dict(type=12), dict(k=None), dict(v=P + 4), dict(ks=255), dict(vs=258), dict(ks=-256), dict(theta=-1.0), dict(theta=float("nan")),
                                 dict(theta=float("inf"))], ids=str)
def test_append_arguments_refused(bad):
    assert append(**bad) == -1


@pytest.mark.parametrize("bad", [dict(type=8), dict(q=None), dict(out=2 * P + 8), dict(qs=1023), dict(os=1026), dict(n_head=7), dict(n_head=0), dict(n_head=8192), dict(window=-1),
                                 dict(scale=-1.0), dict(scale=float("inf")), dict(theta=-2.0), dict(most=-1), dict(scratch=None), dict(scratch=P + 8), dict(nbytes=16),
                                 dict(b=batch(rows=1 << 29))], ids=str)
def test_attention_arguments_refused(bad):
    assert attend(**bad) == -1


@pytest.mark.parametrize("out, stride", [(P, 1024), (P + 16, 1024), (P + 2 * 4096 + 4080, 1024), (P - 2 * 4096 - 4080, 1024), (P + 4096, 2048), (P - 4096, 2048)], ids=str)
def test_results_over_queries_refused(out, stride):
    assert attend(out=out, os=stride) == -1  # queries: 3 rows of 4096 bytes from P on


def test_nothing_to_do_is_no_launch():
    for b in (batch(rows=0), batch(n_seq=0, row_start=None, pos0=None, table=None)):
        assert append(b=b) == 0 and attend(b=b) == 0
    assert capi.lib().b200_attention_pages_scratch_bytes(C.byref(cache(head_dim=96)), 8, 1) == 0


def test_python_refuses_cpu_tensors_and_shapes():
    from mesh_llm_b200 import ops

    x = torch.zeros((3, 2, 128))
    pages = torch.zeros((4, 2, 16, 128), dtype=torch.float16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.kv_pages_append(x, x, pages, pages, i[None, :1], i, i[:1], 1e4, 1)
    with pytest.raises(ValueError):
        ops.attention_pages(x, pages, pages, i[None, :1], i, i[:1], 1, 1e4, 1)


def test_python_refuses_shared_pages_and_tables():
    """pools and tables whose rows lie over one another (expanded views), before the device is looked at"""
    from mesh_llm_b200 import ops

    x = torch.zeros((3, 2, 128))
    pages = torch.zeros((4, 2, 16, 128), dtype=torch.float16)
    i = torch.zeros(3, dtype=torch.int32)
    table = torch.zeros((2, 4), dtype=torch.int32)
    with pytest.raises(ValueError, match="its own"):
        ops.kv_pages_append(x, x, pages[:1].expand(4, -1, -1, -1), pages[:1].expand(4, -1, -1, -1), table, i, i[:2], 1e4, 1)
    for t in (table[:1].expand(2, -1), table.as_strided((2, 4), (2, 1)), table.T[:2]):
        with pytest.raises(ValueError, match="contiguous rows"):
            ops.kv_pages_append(x, x, pages, pages, t, i, i[:2], 1e4, 1)
    for window, most in ((-1, 1), ((1 << 30) + 1, 1), ((1 << 32) + 5, 1), (0, -1), (0, 1 << 32)):
        with pytest.raises(ValueError, match="window"):
            ops.attention_pages(x, pages, pages, table, i, i[:2], most, 1e4, 1, window=window)


def test_descriptor_layout():
    """the ctypes mirrors have the sizes and offsets a C compiler gives the header's structs"""
    import os
    import subprocess
    import tempfile

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = '#include <stddef.h>\n#include <stdio.h>\n#include "%s/include/b200_kquant.h"\nint main(void) {\n' % root
    for name, mirror in (("b200_kv_pages", capi.KvPages), ("b200_page_batch", capi.PageBatch)):
        src += 'printf("%%zu", sizeof(%s));' % name
        for f, _ in mirror._fields_:
            src += 'printf(" %%zu", offsetof(%s, %s));' % (name, f)
        src += 'printf("\\n");'
    with tempfile.TemporaryDirectory() as d:
        open(d + "/l.c", "w").write(src + "return 0; }\n")
        subprocess.check_call(["gcc", "-o", d + "/l", d + "/l.c"])
        lines = subprocess.check_output([d + "/l"], text=True).splitlines()
    for line, mirror in zip(lines, (capi.KvPages, capi.PageBatch)):
        assert [int(x) for x in line.split()] == [C.sizeof(mirror)] + [getattr(mirror, f).offset for f, _ in mirror._fields_]
