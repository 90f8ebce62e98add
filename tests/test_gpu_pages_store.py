"""What append leaves in e4m3 pages: rows of every type, heads below, at and above the eight that a CTA may take, scales of keys and values in every block.

Tolerances: a code is half a step of 2^-4 off, below the type's normal range 2^-10 of its scale; what 32-bit rotation leaves: four roundings of terms of at
most sqrt(2) |x|, 2^-21 of the largest element.
"""
import numpy as np
import pytest
import torch

from tests.pages_util import BLOCK, Batch, Cache, turned

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def randn(seed, n, heads, hd, dtype, gain=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn((n, heads, hd), generator=g, device="cuda") * gain
    x[..., ::13] *= 3.0
    x *= 2.0 ** torch.randint(-3, 4, (n, heads, 1), generator=g, device="cuda")  # heads and rows are not all alike
    return x.to(dtype)


def scale_of(x):
    """of rows [n, n_kv, hd] in one block: the smallest power of two in [2^-15, 2^7] that brings the largest to at most 448"""
    top = x.abs().amax((0, 2)).cpu().numpy()
    return torch.from_numpy(2.0 ** np.clip(np.ceil(np.log2(np.maximum(top, 1e-30) / 448.0)), -15, 7)).cuda()


def same_scale(x, got, slack):
    """got is x's scale, or the next one where rotation's last bits decide"""
    return (got == scale_of(x * (1 - slack))).logical_or(got == scale_of(x * (1 + slack))).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n_kv", [1, 4, 5, 8, 11])
@pytest.mark.parametrize("hd, neox, theta", [(64, 0, 1e4), (64, 1, 1e6), (128, 0, 1e6), (128, 1, 1e4), (128, 1, 0.0)])
def test_rows_of_every_type(n_kv, dtype, hd, neox, theta):
    new, past, page = [1, 37, 5, 16, 300], [0, 9, 14, 32, 3], 48
    c = Cache(5, 310, page, n_kv, hd, F8, seed=50)
    total = Batch(past, [0] * 5)
    c.append(randn(51, total.rows, n_kv, hd, dtype, 0.2), randn(52, total.rows, n_kv, hd, dtype, 0.2), total, theta, neox)
    b = Batch(new, past)
    was, old = c.values(), (c.ks.clone(), c.vs.clone())
    raw = [x.view(torch.uint8).clone() for x in (c.k, c.v)]
    wide = randn(53, b.rows, 2 * n_kv + 2, hd, dtype)  # keys and values as columns of one projection
    k, v = wide[:, 1:1 + n_kv], wide[:, 1 + n_kv:1 + 2 * n_kv]
    c.append(k, v, b, theta, neox)
    touched = torch.zeros((c.n_pages, c.page), dtype=torch.bool, device="cuda")
    for s, at, t, p in b.spans():
        pos = torch.arange(p, p + t, device="cuda")
        for x, want, scales, slack in ((0, turned(k[at:at + t], pos, theta, neox), c.ks, 2.0 ** -20), (1, v[at:at + t].double(), c.vs, 0.0)):
            got, before = c.rows(s, p + t)[x], c.rows(s, p + t, [was[x], was[x]])[0]
            for blk in range(p // BLOCK, (p + t - 1) // BLOCK + 1):
                lo, hi = max(p, blk * BLOCK), min(p + t, blk * BLOCK + BLOCK)
                pg, ib = int(c.table[s, blk * BLOCK // page]), blk * BLOCK % page // BLOCK
                w, sc = want[lo - p:hi - p], scales[pg, :, ib].double()
                if lo > blk * BLOCK:  # the block held rows
                    prior = old[x][pg, :, ib].double()
                    assert (sc >= prior).all() and ((sc == prior) | (sc <= scale_of(w * (1 + slack)))).all()
                    assert (torch.maximum(prior, scale_of(w * (1 - slack))) <= sc).all()
                    # exact but for codes that fell below the normal range
                    assert ((got[blk * BLOCK:lo] - before[blk * BLOCK:lo]).abs() <= sc[None, :, None] * 2.0 ** -10).all()
                else:
                    assert same_scale(w, sc, slack)
                off = (got[lo:hi] - w).abs()
                assert (off <= w.abs() * 2.0 ** -4 + w.abs().amax((0, 2), keepdim=True) * 2.0 ** -21 + sc[None, :, None] * 2.0 ** -10).all()
        for blk in range(p // BLOCK, (p + t - 1) // BLOCK + 1):
            first = blk * BLOCK
            touched[c.table[s, first // page].long(), first % page:min(first + BLOCK, p + t - first // page * page)] = True
    for x, y in zip((c.k, c.v), raw):  # nothing else was written
        keep = ~touched[:, None, :, None].expand(-1, n_kv, -1, hd)
        assert torch.equal(x.view(torch.uint8)[keep], y[keep])


def test_scales_of_both_pools_position_by_position():
    """a block filled position by position ends under the scale of a block filled at once, in every block of keys and values"""
    n_kv, hd, n = 9, 128, 100
    k, v = randn(54, n, n_kv, hd, torch.bfloat16), randn(55, n, n_kv, hd, torch.bfloat16)
    a, b = (Cache(1, 112, 48, n_kv, hd, F8, seed=51) for _ in "ab")
    a.append(k, v, Batch([n], [0]), 1e4, 1)
    for i in range(n):
        b.append(k[i:i + 1], v[i:i + 1], Batch([1], [i]), 1e4, 1)
    for x, y in ((a.ks, b.ks), (a.vs, b.vs)):
        for blk in range((n + BLOCK - 1) // BLOCK):
            pg, ib = a.table[0, blk * BLOCK // 48].long(), blk * BLOCK % 48 // BLOCK
            assert torch.equal(x[pg, :, ib], y[pg, :, ib])
    for x, y, s in zip(a.rows(0, n), b.rows(0, n), (a.ks, a.vs)):
        # half a step of the smallest code, for each of the two roundings of a code below the normal range
        pos = torch.arange(n, device="cuda")
        sc = s[a.table[0].long()[pos // 48], :, pos % 48 // BLOCK].double()[..., None]
        assert ((x - y).abs() <= 2.0 ** -9 * sc).all()


@pytest.mark.parametrize("exponent", [-15, -7, 0, 7])
def test_every_code_times_its_scale_is_an_f16_number(exponent):
    """all 254 numbers that a code can be, at the ends of the scales' range: attention sees exactly them, over either page type"""
    codes = torch.tensor([x for x in range(256) if x & 0x7F != 0x7F], dtype=torch.uint8, device="cuda").view(F8).float()
    n, hd = 16, 128
    x = torch.zeros((n, 1, hd), device="cuda")
    x.view(-1)[:254] = codes * 2.0 ** exponent  # 448 2^e among them: the block's scale is 2^e
    c = Cache(1, n, 16, 1, hd, F8, seed=52)
    c.append(x, x, Batch([n], [0]), 0.0, 0)
    pg = c.table[0, 0].long()
    assert c.ks[pg, 0, 0] == 2.0 ** exponent and c.vs[pg, 0, 0] == 2.0 ** exponent
    values = c.rows(0, n)[1]
    assert torch.equal(values, x.double())
    assert torch.equal(values.half().double(), values)
    # a query that sees one position alone gives it back, from either kernel
    for most in (1, 100):
        q = torch.zeros((n, 1, hd), device="cuda")
        got = c.attend(q, Batch([n], [0]), 0.0, 0, window=1, max_rows=most)
        assert torch.equal(got.double(), values)


@pytest.mark.parametrize("dtype", [torch.float16, F8])
def test_pools_of_one_head_as_views(dtype):
    """[pages, positions, 1, hd] seen as [pages, 1, positions, hd]: the memory of a pool of one KV head"""
    c, d = (Cache(2, 60, 32, 1, 64, dtype, seed=53) for _ in "cd")
    byte = torch.uint8 if dtype == F8 else torch.int16
    d.k, d.v = (x.view(byte).reshape(c.n_pages, 32, 1, 64).permute(0, 2, 1, 3).view(dtype) for x in (d.k, d.v))
    assert d.k.stride(1) == 64
    b = Batch([20, 3], [0, 50])
    k, v, q = randn(56, b.rows, 1, 64, torch.float32), randn(57, b.rows, 1, 64, torch.float32), randn(58, b.rows, 6, 64, torch.float32)
    for x in (c, d):
        x.append(k, v, b, 1e4, 0)
    assert torch.equal(c.k.view(byte), d.k.view(byte)) and torch.equal(c.v.view(byte), d.v.view(byte))
    late = Batch([20, 0], [0, 0])  # the second sequence's earlier positions were never written
    assert torch.equal(c.attend(q, late, 1e4, 0)[:20], d.attend(q, late, 1e4, 0)[:20])
