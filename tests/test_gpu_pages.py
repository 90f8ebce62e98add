"""The paged cache and the attention over it against plain 64-bit arithmetic.

Tolerances, in terms of u = the half step of a type relative to the value (f16 2^-11, bf16 2^-8, f32 2^-24, e4m3 2^-4):
- a stored key is the rotated one rounded once: u of the page type, plus what 32-bit rotation leaves (four roundings of terms of at most
  sqrt(2) |x|: 2^-22 of the pair's length); an e4m3 code below the type's normal range is off by up to 2^-10 of its scale.
- attention in f32: queries and probabilities in 22 bits each, sums of 32 bits over up to 10^4 terms: 2^-22 on scores of size up to about 10 in
  base 2 gives 2^-18 relative on a probability, and as much on an output next to the size of the values: 2e-5 of the largest value leaves room for both.
- attention in f16 or bf16: the query's rotation is rounded to f16 (2^-12 of a score of about 10: 0.003 on a probability at worst), probabilities to f16,
  the output to its own type: 0.004 of the largest value plus u of the result.
"""
import numpy as np
import pytest
import torch

from tests.pages_util import BLOCK, Batch, Cache, attention, turned

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def rows(seed, n, heads, hd, dtype=torch.float32, gain=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn((n, heads, hd), generator=g, device="cuda") * gain
    x[..., ::13] *= 3.0
    return x.to(dtype)


def expect_scale(amax):
    """smallest power of two in [2^-15, 2^7] that brings amax to at most 448"""
    e = np.ceil(np.log2(np.maximum(amax, 1e-30) / 448.0))
    return 2.0 ** np.clip(e, -15, 7)


def fill(cache, past, seed, theta, neox, dtype=torch.float32, chunk=4096, gain=1.0):
    """puts `past` positions of each sequence in, at most `chunk` at a time"""
    done = [0] * len(past)
    i = 0
    while any(d < p for d, p in zip(done, past)):
        new = [min(chunk, p - d) for d, p in zip(done, past)]
        b = Batch(new, done)
        cache.append(rows(seed + i, b.rows, cache.n_kv, cache.hd, dtype, gain), rows(seed + 1000 + i, b.rows, cache.n_kv, cache.hd, dtype, gain), b, theta, neox)
        done = [d + n for d, n in zip(done, new)]
        i += 1


def close(got, want, dtype):
    torch.cuda.synchronize()
    top = want.abs().max().item()
    d = (got.double() - want).abs()
    if dtype == torch.float32:
        assert d.max().item() <= 2e-5 * top, d.max().item() / top
    else:
        u = torch.finfo(dtype).eps / 2
        assert (d <= 0.004 * top + u * want.abs()).all(), (d.max().item(), top)


# ---- append
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("neox", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page", [16, 48])
def test_append_f16(hd, neox, dtype, page):
    new, past, n_kv = [1, 17, 0, 40, 16], [0, 5, 3, 15, 100], 3
    c, b = Cache(5, 130, page, n_kv, hd, torch.float16, seed=1), Batch(new, past)
    k, v = rows(1, b.rows, n_kv, hd, dtype), rows(2, b.rows, n_kv, hd, dtype)
    before = [x.clone() for x in (c.k, c.v)]
    c.append(k, v, b, 1e6, neox)
    for s, at, t, p in b.spans():
        pos = torch.arange(p, p + t, device="cuda")
        gk, gv = (x[p:] for x in c.rows(s, p + t))
        want = turned(k[at:at + t], pos, 1e6, neox)
        size = k[at:at + t].double().abs().amax()if t else 0
        assert t == 0 or ((gk - want).abs() <= want.abs() * 2.0 ** -11 + size * 2.0 ** -21 + 2.0 ** -25).all()
        assert ((gv - v[at:at + t].double()).abs() <= v[at:at + t].double().abs() * 2.0 ** -11 + 2.0 ** -25).all()
        idx = c.table[s].long()[pos // page], pos % page
        for x, y in zip((c.k, c.v), before):
            y[idx[0], :, idx[1]] = x[idx[0], :, idx[1]]
    for x, y in zip((c.k, c.v), before):  # nothing else was written
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("neox", [0, 1])
@pytest.mark.parametrize("page", [16, 32, 80])
def test_append_e4m3(hd, neox, page):
    """codes, scales and what a block keeps when its scale grows"""
    n_kv, theta = 9, 1e6
    new, past = [1, 37, 5, 16, 3], [0, 9, 14, 32, 47]
    c, b = Cache(5, 64, page, n_kv, hd, F8, seed=2), Batch(new, past)
    fill(c, past, 10, theta, neox, gain=0.2)  # small values first: the new ones make the scales grow
    old = c.values()
    old_scales = c.ks.clone(), c.vs.clone()
    k, v = rows(3, b.rows, n_kv, hd), rows(4, b.rows, n_kv, hd)
    c.append(k, v, b, theta, neox)
    for s, at, t, p in b.spans():
        pos = torch.arange(p, p + t, device="cuda")
        for x, want, scale, was, was_scale in ((0, turned(k[at:at + t], pos, theta, neox), c.ks, old[0], old_scales[0]),
                                               (1, v[at:at + t].double(), c.vs, old[1], old_scales[1])):
            got = c.rows(s, p + t)[x]
            for blk in range(p // BLOCK, (p + t - 1) // BLOCK + 1):
                lo, hi = max(p, blk * BLOCK), min(p + t, blk * BLOCK + BLOCK)
                pg, ib = int(c.table[s, blk * BLOCK // page]), blk * BLOCK % page // BLOCK
                amax = want[lo - p:hi - p].abs().amax((0, 2)).cpu().numpy()
                e = expect_scale(amax)
                if lo > blk * BLOCK:  # the block held rows
                    e = np.maximum(e, was_scale[pg, :, ib].cpu().numpy())
                    held = slice(blk * BLOCK, lo)
                    gone = torch.from_numpy(e).cuda()[None, :, None]
                    kept = c.rows(s, p + t, [was, was])[x][held]
                    assert ((got[held] - kept).abs() <= gone * 2.0 ** -10).all()  # exact but for codes that fell below the normal range
                np.testing.assert_array_equal(scale[pg, :, ib].cpu().numpy(), e)
                sc = torch.from_numpy(e).cuda()[None, :, None]
                w = want[lo - p:hi - p]
                assert ((got[lo:hi] - w).abs() <= w.abs() * (2.0 ** -4 + 2.0 ** -20) + sc * 2.0 ** -10).all()


def test_append_position_by_position_is_append_at_once():
    """a power-of-two scale costs a rescaled code nothing: only the scale's own history can differ, and here it does not"""
    n_kv, hd, n = 2, 128, 50
    k, v = rows(5, n, n_kv, hd), rows(6, n, n_kv, hd)
    a, b = (Cache(1, 64, 32, n_kv, hd, F8, seed=3) for _ in "ab")
    a.append(k, v, Batch([n], [0]), 1e4, 1)
    for i in range(n):
        b.append(k[i:i + 1], v[i:i + 1], Batch([1], [i]), 1e4, 1)
    for x, y in zip(a.rows(0, n), b.rows(0, n)):
        # a code below the normal range of an earlier, smaller scale may round differently: half a step of the smallest code
        assert ((x - y).abs() <= 2.0 ** -9 * torch.maximum(a.ks.max(), a.vs.max()).double()).all()
    assert (a.ks >= 0).all() and torch.equal(a.ks.view(-1, n_kv, 2)[a.table[0].long()][0], b.ks.view(-1, n_kv, 2)[b.table[0].long()][0])


@pytest.mark.parametrize("cache", [torch.float16, F8])
def test_append_out_of_range_and_nan(cache):
    c = Cache(1, 32, 16, 1, 128, cache)
    k, v = rows(7, 20, 1, 128), rows(8, 20, 1, 128)
    k[2, 0, 5], k[3, 0, 6], v[4, 0, 7], v[5, 0, 8], v[6, 0, 9], k[7, 0, 10] = 1e9, -float("inf"), float("inf"), -1e30, float("nan"), float("nan")
    c.append(k, v, Batch([20], [0]), 0.0, 0)
    gk, gv = c.rows(0, 20)
    top = 65504.0 if cache == torch.float16 else 57344.0
    assert gk[2, 0, 5] == top and gk[3, 0, 6] == -top and gv[4, 0, 7] == top and gv[5, 0, 8] == -top
    assert gv[6, 0, 9] == 0 and torch.isnan(gk[6]).sum() == 1 and torch.isnan(gk[7]).sum() == 1 and torch.isnan(gk).sum() == 2
    assert torch.isfinite(gv).all()


def test_append_places_that_are_not_there():
    """absent pages, positions past the table, sequences without positions and rows nobody owns: nothing is written for them"""
    c = Cache(4, 64, 16, 2, 64, torch.float16, seed=4)
    c.table[1, 1] = -1
    c.table[2, 0] = c.n_pages
    before = c.k.clone()
    b = Batch([20, 40, 16, 5], [60, 0, 0, -1], first=3)
    k = rows(9, b.rows + 6, 2, 64)
    c.append(k, k, b, 1e4, 1)
    changed = (c.k.view(torch.int16) != before.view(torch.int16)).any(-1).any(1)  # [n_pages, page]
    want = torch.zeros_like(changed)
    for pos in range(60, 64):
        want[c.table[0, pos // 16].item(), pos % 16] = True
    for pos in list(range(16)) + list(range(32, 40)):
        want[c.table[1, pos // 16].item(), pos % 16] = True
    assert torch.equal(changed, want)


# ---- attention
SHAPES = [(1, 1), (5, 1), (8, 2), (12, 1), (16, 2), (7, 7), (40, 1)]


@pytest.mark.parametrize("cache", [torch.float16, F8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", SHAPES)
def test_decode(cache, dtype, heads):
    n_head, n_kv = heads
    past = [0, 1, 15, 16, 63, 64, 200, 1000]
    c, b = Cache(8, 1010, 16, n_kv, 128, cache, seed=5), Batch([1] * 8, past)
    fill(c, past, 20, 1e4, 1)
    q = rows(11, 8, n_head, 128, dtype)
    c.append(rows(12, 8, n_kv, 128, dtype), rows(13, 8, n_kv, 128, dtype), b, 1e4, 1)
    close(c.attend(q, b, 1e4, 1), attention(c, q, b, 1e4, 1), dtype)


@pytest.mark.parametrize("cache", [torch.float16, F8])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window", [0, 1, 20, 100])
@pytest.mark.parametrize("neox", [0, 1])
def test_ragged(cache, hd, window, neox):
    """rows of several sequences, several row tiles, windows, pages that end inside a tile"""
    new, past = [3, 0, 1, 11, 2, 40], [300, 7, 0, 77, 129, 0]
    n_head, n_kv = 6, 2
    c, b = Cache(6, 310, 48, n_kv, hd, cache, seed=6), Batch(new, past, first=2)
    fill(c, past, 30, 1e6, neox)
    q = rows(14, b.rows, n_head, hd)
    c.append(rows(15, b.rows, n_kv, hd), rows(16, b.rows, n_kv, hd), b, 1e6, neox)
    for most in (1, 40):
        out = torch.full((b.rows + 4, n_head, hd), 7.0, device="cuda")
        got = c.attend(torch.cat((q, q[:4])), b, 1e6, neox, window=window, max_rows=most, out=out)
        close(got[2:b.rows], attention(c, q, b, 1e6, neox, window)[2:], torch.float32)
        assert (got[:2] == 7).all() and (got[b.rows:] == 7).all()  # rows nobody owns


@pytest.mark.parametrize("cache", [torch.float16, F8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1, 64), (5, 1, 128), (8, 2, 128), (14, 2, 64)])
def test_prompts(cache, dtype, shape):
    """one sequence, from nothing and behind a long past: one and many tiles of rows, tiles of keys that end anywhere"""
    n_head, n_kv, hd = shape
    for new, past, page in ((130, 0, 16), (67, 61, 48), (300, 1000, 128), (513, 129, 64)):
        c, b = Cache(1, new + past, page, n_kv, hd, cache, seed=10), Batch([new], [past])
        fill(c, [past], 110, 1e6, 1)
        q = rows(33, new, n_head, hd, dtype)
        c.append(rows(34, new, n_kv, hd, dtype), rows(35, new, n_kv, hd, dtype), b, 1e6, 1)
        close(c.attend(q, b, 1e6, 1), attention(c, q, b, 1e6, 1), dtype)


@pytest.mark.parametrize("cache", [torch.float16, F8])
@pytest.mark.parametrize("window", [0, 64, 333])
def test_prompts_and_steps_in_one_call(cache, window):
    new, past = [200, 1, 0, 3, 90, 1, 400, 65], [10, 700, 5, 129, 0, 0, 600, 128]
    n_head, n_kv, hd = 10, 2, 128
    c, b = Cache(8, 1000, 32, n_kv, hd, cache, seed=11), Batch(new, past, first=1)
    fill(c, past, 120, 1e4, 0)
    q = rows(36, b.rows, n_head, hd)
    c.append(rows(37, b.rows, n_kv, hd), rows(38, b.rows, n_kv, hd), b, 1e4, 0)
    out = torch.full((b.rows + 2, n_head, hd), 7.0, device="cuda")
    got = c.attend(torch.cat((q, q[:2])), b, 1e4, 0, window=window, out=out)
    close(got[1:b.rows], attention(c, q, b, 1e4, 0, window)[1:], torch.float32)
    assert (got[0] == 7).all() and (got[b.rows:] == 7).all()
    assert torch.equal(c.attend(torch.cat((q, q[:2])), b, 1e4, 0, window=window, out=torch.full_like(out, 7.0)), got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_e4m3_pages_give_what_the_f16_pages_of_their_values_give(dtype):
    c = Cache(3, 700, 32, 2, 128, F8, seed=7)
    past = [699, 31, 300]
    fill(c, past, 40, 1e6, 1)
    b = Batch([1, 1, 1], [p - 1 for p in past])
    d = Cache(3, 700, 32, 2, 128, torch.float16, seed=7)
    for x, y in zip((d.k, d.v), c.values()):
        assert torch.equal(y.half().double(), y) or torch.isnan(y).any()
        x.copy_(y.half())
    q = rows(17, 3, 16, 128, dtype)
    x, y = c.attend(q, b, 1e6, 1), d.attend(q, b, 1e6, 1)
    # the same products; their sums run in another order: 32-bit sums of a few hundred terms
    assert ((x.double() - y.double()).abs() <= (2e-6 if dtype == torch.float32 else 0.01) * y.double().abs().max()).all()


@pytest.mark.parametrize("cache", [torch.float16, F8])
@pytest.mark.parametrize("split", [False, True])
def test_what_no_row_sees_does_not_matter(cache, split):
    """NaN behind the last position, in dropped pages, and a token whose own v or k is NaN: later rows alone see it"""
    n = 40
    c, b = Cache(1, 96, 16, 1, 128, cache), Batch([n], [21])
    fill(c, [21], 50, 1e4, 1)
    q, k, v = rows(18, n, 4, 128), rows(19, n, 1, 128), rows(20, n, 1, 128)
    v[30, 0, 3] = float("nan")
    k[35, 0, 99] = float("nan")
    c.append(k, v, b, 1e4, 1)
    c.table[0, 0] = -1  # a page that is gone
    got = c.attend(q, b, 1e4, 1, max_rows=n if split else 1)
    assert torch.isfinite(got[:30]).all() and torch.isnan(got[30:]).all()
    seen = c.attend(q, b, 1e4, 1, window=5, max_rows=n if split else 1)
    assert torch.isnan(seen[30:]).all() and torch.isfinite(seen[:30]).all()
    none = Cache(1, 96, 16, 1, 128, cache)
    none.table[:] = -1
    assert (none.attend(q, b, 1e4, 1, max_rows=n if split else 1) == 0).all()
    assert (c.attend(q, Batch([n], [-1]), 1e4, 1, max_rows=n if split else 1) == 0).all()


@pytest.mark.parametrize("cache", [torch.float16, F8])
def test_large_and_small_queries(cache):
    """a query row is used at its own size: rows of 1e-6 and of 1e6 alike"""
    c, b = Cache(2, 300, 16, 1, 128, cache), Batch([1, 1], [299, 120])
    fill(c, [300, 121], 60, 0.0, 0, gain=0.02)
    q = rows(21, 2, 4, 128)
    for gain, scale in ((1e6, 1e-6), (1e-6, 1e6), (1e-20, 1e20)):
        x = q * gain
        close(c.attend(x, b, 0.0, 0, scale=scale), attention(c, x, b, 0.0, 0, scale=scale), torch.float32)


def test_views_strides_and_pools():
    """q, k, v as views of one projection, both pools interleaved in one allocation, a table that is a view"""
    n_kv, n_head, hd, n = 2, 6, 64, 5
    qkv = rows(22, n, n_head + 2 * n_kv, hd)
    q, k, v = qkv[:, :n_head], qkv[:, n_head:n_head + n_kv], qkv[:, n_head + n_kv:]
    c, b = Cache(2, 64, 32, n_kv, hd, torch.float16), Batch([2, 3], [10, 30])
    fill(c, [10, 30], 70, 1e4, 0)
    pool = torch.zeros((c.n_pages, 2, n_kv, 32, hd), dtype=torch.float16, device="cuda")
    pool[:, 0], pool[:, 1] = c.k, c.v
    table = torch.full((2, 5), -1, dtype=torch.int32, device="cuda")
    table[:, :2] = c.table
    c.append(k.contiguous(), v.contiguous(), b, 1e4, 0)
    want = c.attend(q.contiguous(), b, 1e4, 0)
    d = Cache(2, 64, 32, n_kv, hd, torch.float16)
    d.k, d.v, d.table = pool[:, 0], pool[:, 1], table[:, :2]
    d.append(k, v, b, 1e4, 0)
    out = torch.zeros((n, n_head + 1, hd), device="cuda")
    d.attend(q, b, 1e4, 0, out=out[:, :n_head])
    assert torch.equal(out[:, :n_head], want) and (out[:, n_head] == 0).all()
    at = c.table.long().flatten()
    assert torch.equal(d.k[at].view(torch.int16), c.k[at].view(torch.int16))
    odd = torch.zeros(n * n_head * hd + 1, device="cuda")[1:].view(n, n_head, hd)  # rows off their alignment are copied
    odd.copy_(q)
    assert torch.equal(d.attend(odd, b, 1e4, 0), want)


@pytest.mark.parametrize("cache", [torch.float16, F8])
@pytest.mark.parametrize("n_seq", [1, 33, 300])
def test_many_sequences_twice_the_same(cache, n_seq):
    g = np.random.default_rng(n_seq)
    past = [int(x) for x in g.integers(0, 400, n_seq)]
    new = [int(x) for x in g.integers(0, 3, n_seq)]
    new[0] = max(new[0], 1)
    c, b = Cache(n_seq, 402, 16, 2, 128, cache, seed=8), Batch(new, past)
    fill(c, past, 80, 1e4, 1)
    q = rows(23, b.rows, 8, 128)
    c.append(rows(24, b.rows, 2, 128), rows(25, b.rows, 2, 128), b, 1e4, 1)
    x = c.attend(q, b, 1e4, 1)
    close(x, attention(c, q, b, 1e4, 1), torch.float32)
    for _ in range(3):
        assert torch.equal(c.attend(q, b, 1e4, 1), x)


@pytest.mark.parametrize("cache", [torch.float16, F8])
def test_steps_in_a_graph_and_on_a_stream(cache):
    """append, then attention, captured once with the positions on the device and replayed as they move on"""
    n_seq, n_kv, n_head, hd = 3, 2, 8, 128
    past = [14, 0, 100]
    c, e = (Cache(n_seq, 160, 16, n_kv, hd, cache, seed=9) for _ in "ce")
    for x in (c, e):
        fill(x, past, 90, 1e4, 1)
    b = Batch([1] * n_seq, past)
    q, k, v = rows(26, n_seq, n_head, hd), rows(27, n_seq, n_kv, hd), rows(28, n_seq, n_kv, hd)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        c.append(k, v, b, 1e4, 1)
        out = c.attend(q, b, 1e4, 1)
    for step in range(40):
        for i, x in enumerate((q, k, v)):
            x.copy_(rows(100 + 3 * step + i, *x.shape))
        b.pos0.copy_(torch.tensor([p + step for p in past], dtype=torch.int32))
        g.replay()
        eager = Batch([1] * n_seq, [p + step for p in past])
        e.append(k, v, eager, 1e4, 1)
        assert torch.equal(out, e.attend(q, eager, 1e4, 1)), step
    eager = Batch([1] * n_seq, [p + 39 for p in past])
    close(out, attention(c, q, eager, 1e4, 1), torch.float32)


def test_far_positions():
    """angles are worked out in 64 bits: position 10^6 is as exact as position 10"""
    hd, n_kv, at = 128, 1, 1_000_003
    page = 4096
    from mesh_llm_b200 import ops

    k, v, _, _ = ops.kv_pages(2, page, n_kv, hd)
    table = torch.full((1, at // page + 1), -1, dtype=torch.int32, device="cuda")
    table[0, -1] = 1
    b = Batch([2], [at])
    x = rows(29, 2, n_kv, hd)
    ops.kv_pages_append(x, x, k, v, table, b.start, b.pos0, 1e6, 1)
    want = turned(x, torch.tensor([at, at + 1], device="cuda"), 1e6, 1)
    got = k[1, :, at % page:at % page + 2].transpose(0, 1).double()
    assert ((got - want).abs() <= want.abs() * 2.0 ** -11 + x.abs().max().double() * 2.0 ** -21).all()
    q = rows(30, 2, 4, hd)
    y = ops.attention_pages(q, k, v, table, b.start, b.pos0, 2, 1e6, 1)
    n = at % page + 2  # the page's earlier positions are there too, as zeros
    w = (turned(q, torch.tensor([at, at + 1], device="cuda"), 1e6, 1)[1] @ k[1, 0, :n].double().T / hd ** 0.5).softmax(-1) @ v[1, 0, :n].double()
    close(y[1], w, torch.float32)


@pytest.mark.parametrize("heads", [(2, 2), (1, 5)])
@pytest.mark.parametrize("dtype", [torch.float16, F8])
@pytest.mark.parametrize("window", [1, 1000, 1 << 30])
def test_positions_past_32_bits(window, dtype, heads):
    """a sequence whose rows pass position 2^31 - 1, far behind its table: it stores nothing, sees nothing, and disturbs no other"""
    n_kv, n_head = heads
    c = Cache(3, 100, 16, n_kv, 64, dtype)
    fill(c, [90, 90, 90], 60, 0.0, 1)
    b = Batch([4, 300, 30], [86, 2 ** 31 - 9, 2 ** 31 - 1])
    held = [x.clone().view(torch.uint8) for x in (c.k, c.v)]
    ordinary = Batch([4, 0, 0], [86, 0, 0])
    x = rows(61, b.rows, n_kv, 64)
    c.append(x, x, Batch([0, 300, 30], b.past), 0.0, 1)
    assert all(torch.equal(was, now.view(torch.uint8)) for was, now in zip(held, (c.k, c.v)))
    q = rows(62, b.rows, n_head, 64)
    want = attention(c, q, ordinary, 0.0, 1, window)
    for most in (1, 300):  # either kernel
        y = c.attend(q, b, 0.0, 1, window=window, max_rows=most)
        assert (y[4:] == 0).all()
        close(y[:4], want[:4], torch.float32)


def test_results_beside_queries():
    """queries and results as parts of one buffer's rows; results over the queries are refused"""
    c = Cache(2, 60, 16, 2, 64, torch.float16)
    fill(c, [40, 50], 70, 1e4, 1)
    b = Batch([20, 3], [40, 50])
    x = rows(71, b.rows, 2, 64)
    c.append(x, x, b, 1e4, 1)
    both = rows(72, b.rows, 8, 64)
    q, out = both[:, :4], both[:, 4:]
    want = attention(c, q, b, 1e4, 1)
    for most in (1, 20):
        assert c.attend(q, b, 1e4, 1, max_rows=most, out=out) is out
        close(out, want, torch.float32)
    with pytest.raises(RuntimeError, match="over queries"):
        c.attend(q, b, 1e4, 1, out=both[:, 2:6])
    with pytest.raises(RuntimeError, match="over queries"):
        c.attend(q, b, 1e4, 1, out=q)


def test_offsets_past_32_bits():
    """the last page of a pool of more than 2^31 elements"""
    from mesh_llm_b200 import ops

    hd, n_kv, page = 128, 8, 256
    n_pages = (1 << 31) // (hd * n_kv * page) + 3
    k, v, ks, vs = ops.kv_pages(n_pages, page, n_kv, hd, F8)
    k2 = torch.zeros((n_pages, n_kv, page, hd), dtype=torch.float16, device="cuda")
    table = torch.tensor([[n_pages - 1, n_pages - 2]], dtype=torch.int32, device="cuda")
    b = Batch([300], [0])
    x, q = rows(31, 300, n_kv, hd), rows(32, 300, 16, hd)
    ops.kv_pages_append(x, x, k, v, table, b.start, b.pos0, 1e6, 1, k_scale=ks, v_scale=vs)
    ops.kv_pages_append(x, x, k2, k2.clone(), table, b.start, b.pos0, 1e6, 1)
    small = Cache(1, 300, page, n_kv, hd, F8, junk=False)
    small.append(x, x, b, 1e6, 1)
    for i in range(2):
        assert torch.equal(k[table[0, i].long()].view(torch.uint8), small.k[small.table[0, i].long()].view(torch.uint8))
    one = Batch([1], [299])
    y = ops.attention_pages(q[299:], k, v, table, one.start, one.pos0, 1, 1e6, 1, k_scale=ks, v_scale=vs)
    assert torch.equal(y, small.attend(q[299:], one, 1e6, 1))
    z = torch.zeros_like(k2[:1])
    ops.kv_pages_append(x[:256], x[:256], z, z.clone(), torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.tensor([0, 256], dtype=torch.int32, device="cuda"),
                        one.pos0 * 0, 1e6, 1)
    assert torch.equal(k2[n_pages - 1], z[0])


@pytest.mark.parametrize("new", [33, 40, 65, 100, 129])
def test_prompts_that_fill_part_of_a_tile(new):
    """row tiles without a second half or with idle warps, over a last tile of keys whose other places hold NaN"""
    for cache, hd in ((torch.float16, 128), (torch.float16, 64), (F8, 128)):
        c, b = Cache(1, new + 150, 16, 1, hd, cache, seed=12), Batch([new], [70])
        fill(c, [70], 130, 1e4, 1)
        q = rows(39, new, 2, hd)
        c.append(rows(40, new, 1, hd), rows(41, new, 1, hd), b, 1e4, 1)
        for window in (0, 30):
            close(c.attend(q, b, 1e4, 1, window=window), attention(c, q, b, 1e4, 1, window), torch.float32)


@pytest.mark.parametrize("cache", [torch.float16, F8])
def test_a_prompt_in_chunks_and_steps_is_the_prompt_at_once(cache):
    """append and attention together as an engine uses them: chunks of any size, then single tokens, against one call and against 64 bits"""
    n, n_kv, n_head, hd, theta = 400, 2, 10, 128, 1e6
    q, k, v = rows(50, n, n_head, hd), rows(51, n, n_kv, hd), rows(52, n, n_kv, hd)
    one, many = (Cache(1, n, 48, n_kv, hd, cache, seed=13) for _ in "ab")
    b = Batch([n], [0])
    one.append(k, v, b, theta, 1)
    whole = one.attend(q, b, theta, 1)
    parts, at = [], 0
    for t in (1, 130, 5, 16, 200, 17) + (1,) * 31:
        step = Batch([t], [at])
        many.append(k[at:at + t], v[at:at + t], step, theta, 1)
        parts.append(many.attend(q[at:at + t], step, theta, 1))
        at += t
    assert at == n
    close(whole, attention(one, q, b, theta, 1), torch.float32)
    close(parts[-1], attention(many, q, b, theta, 1)[n - 1:], torch.float32)
    if cache == torch.float16:  # e4m3: a block's earlier rows were quantised under the scale it had then
        close(torch.cat(parts), attention(one, q, b, theta, 1), torch.float32)


@pytest.mark.parametrize("cache", [torch.float16, F8])
def test_scratch_of_any_content_and_two_graphs_on_it(cache):
    import ctypes as C

    from mesh_llm_b200 import capi, ops

    new, past = [300, 1, 40], [100, 900, 0]
    c, b = Cache(3, 1000, 32, 2, 128, cache, seed=14), Batch(new, past)
    fill(c, past, 140, 1e4, 1)
    q = rows(53, b.rows, 16, 128)
    c.append(rows(54, b.rows, 2, 128), rows(55, b.rows, 2, 128), b, 1e4, 1)
    want = c.attend(q, b, 1e4, 1)
    pages, batch = ops._pages_call(q, c.k, c.v, c.table, b.start, b.pos0, c.ks, c.vs)
    need = capi.lib().b200_attention_pages_scratch_bytes(pages, 16, b.most)
    scratch = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")  # NaN everywhere
    out = [torch.zeros_like(q) for _ in "ab"]

    def call(o):
        capi.check(capi.lib().b200_attention_pages(pages, batch, 0, q.data_ptr(), q.stride(0), 16, b.most, 1e4, 1, 0, 0.0, o.data_ptr(), o.stride(0),
                                                   scratch.data_ptr(), need, capi.cur_stream()))

    call(out[0])
    assert torch.equal(out[0], want)
    graphs = [torch.cuda.CUDAGraph() for _ in "ab"]
    for g, o in zip(graphs, out):
        with torch.cuda.graph(g):
            call(o)
    for o in out:
        o.zero_()
    for _ in range(3):
        for g in graphs:
            g.replay()
    assert torch.equal(out[0], want) and torch.equal(out[1], want)


@pytest.mark.parametrize("theta", [0.01, 0.7, 1.0, 1e9])
def test_rotation_bases(theta):
    c, b = Cache(1, 4000, 16, 1, 64, torch.float16), Batch([3], [3990])
    k = rows(56, 3, 1, 64)
    c.append(k, k, b, theta, 0)
    want = turned(k, torch.arange(3990, 3993, device="cuda"), theta, 0)
    # fast turns: a frequency of f turns a position is a 64-bit fraction of one, rounded from 53 bits
    assert ((c.rows(0, 3993)[0][3990:] - want).abs() <= want.abs() * 2.0 ** -11 + k.abs().max().double() * 2.0 ** -21).all()


def test_calls_on_two_streams_at_once():
    c, b = Cache(4, 2000, 16, 2, 128, torch.float16, seed=15), Batch([1] * 4, [1999, 100, 700, 5])
    fill(c, [2000, 101, 701, 6], 150, 1e4, 1)
    q = rows(57, 4, 8, 128)
    want = c.attend(q, b, 1e4, 1)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for i in range(30):
        with torch.cuda.stream(streams[i % 3]):
            got.append(c.attend(q, b, 1e4, 1))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


def test_tables_of_no_pages():
    c = Cache(2, 32, 16, 1, 64, torch.float16)
    c.table = torch.empty((2, 0), dtype=torch.int32, device="cuda")
    b = Batch([1, 100], [5, 0])
    before = c.k.clone()
    c.append(rows(58, 101, 1, 64), rows(59, 101, 1, 64), b, 1e4, 1)
    assert torch.equal(c.k.view(torch.int16), before.view(torch.int16))
    assert (c.attend(rows(60, 101, 4, 64), b, 1e4, 1) == 0).all()
