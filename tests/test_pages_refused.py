"""No GPU: calls of the paged operators that are refused before anything is launched, each a call that would be let through but for one thing."""
import ctypes as C

import pytest

from mesh_llm_b200 import build, capi

M = 1 << 20  # places of the call's buffers, which none of these calls may reach
PLACES = dict(k_pool=16 * M, v_pool=32 * M, ks=48 * M, vs=49 * M, q=64 * M, k=80 * M, v=96 * M, out=112 * M, scratch=1024 * M)
THROUGH = -3  # the status of a call that is let through: there is no device


def cache(type=capi.TYPE_F16, **kw):
    f8 = type == capi.TYPE_F8_E4M3
    d = dict(k=PLACES["k_pool"], v=PLACES["v_pool"], k_scale=PLACES["ks"] if f8 else None, v_scale=PLACES["vs"] if f8 else None, n_pages=4, page_stride=0, type=type,
             page_size=16, n_kv=2, head_dim=128)
    return capi.KvPages(**{**d, **kw})


def batch(**kw):
    return capi.PageBatch(**{**dict(row_start=M, pos0=M, table=M, rows=3, n_seq=1, table_len=4, table_stride=4), **kw})


def append(c=None, b=None, type=0, k=PLACES["k"], ks=256, v=PLACES["v"], vs=256):
    build.build()
    return capi.lib().b200_kv_pages_append(C.byref(c or cache()), C.byref(b or batch()), type, k, ks, v, vs, 1e4, 1, None)


def attend(c=None, b=None, type=0, q=PLACES["q"], qs=1024, out=PLACES["out"], os=1024, scratch=PLACES["scratch"], most=1):
    build.build()
    return capi.lib().b200_attention_pages(C.byref(c or cache()), C.byref(b or batch()), type, q, qs, 8, most, 1e4, 1, 0, 0.0, out, os, scratch, 1 << 40, None)


@pytest.fixture(autouse=True)
def no_device():
    import torch

    if torch.cuda.is_available():
        pytest.skip("the calls that are let through would run")


def test_the_calls_that_are_varied_are_let_through():
    for type in (capi.TYPE_F16, capi.TYPE_F8_E4M3):
        assert append(cache(type)) == THROUGH
        assert attend(cache(type)) == THROUGH and attend(cache(type), most=100) == THROUGH


@pytest.mark.parametrize("stride", [1 << 62, 1 << 61, 1 << 60, (1 << 48) // 3 + 16, -1 << 62])
def test_strides_whose_products_pass_64_bits(stride):
    """4 << 62 bytes are none in 64 bits: the place of results within a row of queries was worked out by a division by it"""
    assert append(ks=stride) == -1 and append(vs=stride) == -1
    for type in (0, 1):
        assert attend(type=type, qs=stride) == -1 and attend(type=type, os=stride) == -1
        assert attend(type=type, qs=stride, out=PLACES["q"] + 16) == -1
        assert attend(type=type, qs=stride, os=stride, out=PLACES["q"] + 16) == -1
    assert attend(b=batch(rows=1), qs=1 << 40) == THROUGH  # one row has no next


def test_pools_whose_size_passes_64_bits():
    for n, stride in ((0x7fffffff, 1 << 36), (1 << 20, 1 << 30)):
        assert append(cache(n_pages=n, page_stride=stride)) == -1 and attend(cache(n_pages=n, page_stride=stride)) == -1
