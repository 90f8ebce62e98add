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


PAGE = 2 * 16 * 128  # elements of a page


def test_results_and_scratch_over_the_cache():
    for type, es in ((capi.TYPE_F16, 2), (capi.TYPE_F8_E4M3, 1)):
        c = cache(type)
        for pool in ("k_pool", "v_pool"):
            at = PLACES[pool]
            for out in (at, at + 4 * PAGE * es - 16, at - 3 * 4096 + 16):
                assert attend(c, out=out) == -1, (pool, out - at)
                assert attend(c, scratch=out) == -1
            assert attend(c, out=at + 4 * PAGE * es) == THROUGH and attend(c, out=at - 3 * 4096) == THROUGH
    c = cache(capi.TYPE_F8_E4M3)
    for scales in ("ks", "vs"):
        assert attend(c, out=PLACES[scales]) == -1 and attend(c, scratch=PLACES[scales]) == -1
    assert attend(out=PLACES["scratch"]) == -1 and attend(q=PLACES["scratch"] + 4096) == -1
    wide = cache(page_stride=3 * PAGE)
    assert attend(wide, out=PLACES["k_pool"] + 3 * 3 * PAGE * 2 + 2 * PAGE - 16) == -1
    assert attend(wide, out=PLACES["k_pool"] + (3 * 3 + 1) * PAGE * 2) == THROUGH


def test_append_into_pools_that_overlap():
    k = PLACES["k_pool"]
    assert append(cache(v=k)) == -1 and append(cache(v=k + 2 * PAGE)) == -1 and append(cache(k=PLACES["v_pool"] + 8 * PAGE - 16)) == -1
    assert append(cache(v=k + 2 * 4 * PAGE)) == THROUGH  # one behind the other
    for first, second in ((k, k + 2 * PAGE), (k + 2 * PAGE, k)):  # in turn
        assert append(cache(k=first, v=second, page_stride=2 * PAGE)) == THROUGH
        assert append(cache(k=first, v=second, page_stride=2 * PAGE - 16)) == -1
    assert append(cache(v=k + 2 * PAGE - 16, page_stride=2 * PAGE)) == -1
    f8 = capi.TYPE_F8_E4M3
    assert append(cache(f8, v_scale=PLACES["ks"])) == -1 and append(cache(f8, v_scale=PLACES["ks"] + 28)) == -1 and append(cache(f8, v_scale=PLACES["ks"] + 32)) == THROUGH
    assert append(cache(f8, k_scale=k)) == -1
    assert attend(cache(v=k)) == THROUGH  # attention only reads them


def test_append_of_rows_that_lie_in_the_cache():
    for rows in ("k", "v"):
        for pool in ("k_pool", "v_pool"):
            assert append(**{rows: PLACES[pool] + 4096}) == -1
    assert append(v=PLACES["k"]) == THROUGH  # both only read


def test_what_is_refused_is_refused_for_itself():
    """the refusals of one argument each, of a call that is let through without it"""
    from tests.test_pages_cpu import BAD_BATCH, BAD_CACHE

    for bad in BAD_CACHE:
        d = {**dict(k_scale=None, v_scale=None), **bad}
        assert append(cache(**d)) == -1 and attend(cache(**d)) == -1, bad
    for bad in BAD_BATCH:
        assert append(b=batch(**bad)) == -1 and attend(b=batch(**bad)) == -1, bad
    for bad in (dict(type=12), dict(k=None), dict(v=PLACES["v"] + 4), dict(ks=255), dict(vs=258), dict(ks=-256)):
        assert append(**bad) == -1, bad
    for bad in (dict(type=8), dict(q=None), dict(out=None), dict(out=PLACES["out"] + 8), dict(qs=1023), dict(os=1026), dict(most=-1), dict(scratch=None), dict(scratch=PLACES["scratch"] + 8)):
        assert attend(**bad) == -1, bad
    q = PLACES["q"]
    for out, stride in ((q, 1024), (q + 16, 1024), (q + 2 * 4096 + 4080, 1024), (q - 2 * 4096 - 4080, 1024), (q + 4096, 2048), (q - 4096, 2048)):
        assert attend(out=out, os=stride) == -1
    assert attend(qs=2048, os=2048, out=q + 4096) == THROUGH  # parts of the same rows


def test_strides_of_dimensions_of_length_one_say_nothing():
    """pools of one KV head as views of [pages, positions, heads, hd], or of one page: what is left to refuse is that they are not on a GPU"""
    import torch

    from mesh_llm_b200 import ops

    i = torch.zeros(2, dtype=torch.int32)
    for n_pages, n_kv, good in ((4, 1, True), (1, 1, True), (1, 2, False), (4, 2, False)):
        pool = torch.zeros((n_pages, 16, n_kv, 128), dtype=torch.float16).permute(0, 2, 1, 3)
        x = torch.zeros((3, n_kv, 128))
        with pytest.raises(ValueError, match="CUDA" if good else "its own"):
            ops.kv_pages_append(x, x, pool, pool.clone(memory_format=torch.preserve_format), i[None, :1], i, i[:1], 1e4, 1)
    one = torch.zeros((4, 2, 16, 128), dtype=torch.float16)[1:2]
    other = torch.zeros((1, 2, 16, 128), dtype=torch.float16).as_strided((1, 2, 16, 128), (77, 2048, 128, 1))
    x = torch.zeros((3, 2, 128))
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_pages_append(x, x, one, other, i[None, :1], i, i[:1], 1e4, 1)
    with pytest.raises(ValueError, match="one shape and layout"):
        big = torch.zeros((8, 2, 16, 128), dtype=torch.float16)
        ops.kv_pages_append(x, x, big[::2], big[:4], i[None, :1], i, i[:1], 1e4, 1)


def test_waits_that_give_up_are_told_apart():
    """a code of b200_check_device_waits names the paged kernels' wait: four bits of their own (every wait of theirs has a number below 16)"""
    import os
    import re

    src = os.path.join(os.path.dirname(os.path.abspath(capi.__file__)), "csrc")
    text = open(os.path.join(src, "kq_capi.cu")).read()
    body = re.search(r"int kq_device_wait_errors\(\) \{(.*?)\n\}", text, re.S).group(1)
    shifts = {}
    for names, shift in re.findall(r"\(+((?:kq_\w+_error_fetch\(\)(?: \| )?)+)\)? << (\d+)\)", body):
        for name in re.findall(r"kq_(\w+)_error_fetch", names):
            shifts[name] = int(shift)
    assert shifts["pages"] == 24 and [n for n, s in shifts.items() if s == 24] == ["pages"]
    codes = [int(c) for c in re.findall(r"wait(?:_all)?\(sh\.[^;]*, (\d+)\)", open(os.path.join(src, "kq_pages_prompt.cu")).read())]
    assert len(codes) >= 10 and 0 < min(codes) and max(codes) < 16
