"""Prompts whose CTAs work for long: several items one after another, each of many units of 128 keys (sums put aside, rings that turn, pages looked up ahead), and
offsets past 32 bits in attention.

Tolerances, relative to the largest value of the result: f32 1e-5 (a score of up to about 20 in base 2 from queries of 22 bits and a rotation of 32: 2^-22 each,
5e-6 on a probability; sums cut off by the tensor cores: 4e-6); f16, bf16: queries of f16's bits at least, 2^-12 of each of 128 products, at six standard
deviations 0.002 on a probability, and half a step of the result's type.
"""
import pytest
import torch

from tests.pages_util import Batch, Cache, attention

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
ROWS, UNIT, SETUP = 256, 128, 6  # of the prompts' kernel: rows of an item, keys of a unit, units that setting an item up counts as


def sharing(batch, n_head, n_kv, window):
    """(most units of keys of one item in one CTA, most items in one CTA) by the rule that the kernel shares a batch out with"""
    g = n_head // n_kv
    order = []  # units of the items: sequence, head, tile
    for _, _, t, p in batch.spans():
        tiles = []
        for tile in range(-(-t * g // ROWS) if t * g > 64 else 0):  # shorter ones are the other kernel's
            first, last = tile * ROWS // g, min(t - 1, (tile * ROWS + ROWS - 1) // g)
            lo = max(0, p + first - window + 1) // UNIT * UNIT if window else 0
            tiles.append(max(1, -(-(p + last + 1 - lo) // UNIT)))
        order += tiles * n_kv
    ctas = torch.cuda.get_device_properties(0).multi_processor_count
    per = -(-sum(u + SETUP for u in order) // ctas)
    units, of, at = 0, {}, 0
    for u in order:
        done = 0
        while done < SETUP + u:
            cta = (at + done) // per
            upto = min(SETUP + u, (cta + 1) * per - at)
            keys = max(0, upto - SETUP) - max(0, done - SETUP)
            if keys:
                units = max(units, keys)
                of[cta] = of.get(cta, 0) + 1
            done = upto
        at += SETUP + u
    return units, max(of.values())


def randn(seed, n, heads, hd, dtype=torch.float32):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn((n, heads, hd), generator=g, device="cuda")
    x[..., ::13] *= 3.0
    return x.to(dtype)


def filled(past, new, page, n_kv, hd, cache, theta, neox):
    total = [p + t for p, t in zip(past, new)]
    c = Cache(len(past), max(total), page, n_kv, hd, cache, seed=40)
    b = Batch(total, [0] * len(past))
    c.append(randn(41, b.rows, n_kv, hd), randn(42, b.rows, n_kv, hd), b, theta, neox)
    return c


def close(got, want):
    top, d = want.abs().max().item(), (got.double() - want).abs()
    if got.dtype == torch.float32:
        assert d.max().item() <= 1e-5 * top, d.max().item() / top
    else:
        u = torch.finfo(got.dtype).eps / 2
        assert (d <= 0.002 * top + u * want.abs()).all(), (d.max().item(), top)


@pytest.mark.parametrize("cache", [torch.float16, F8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape, window", [((40, 8, 128, 1024, 3000, 64), 0), ((40, 8, 128, 1024, 3000, 64), 2001), ((16, 2, 128, 2000, 3000, 48), 0),
                                           ((16, 2, 64, 2500, 2777, 256), 0), ((16, 2, 64, 2500, 2777, 16), 1900)])
def test_ctas_of_many_units_and_items(shape, window, dtype, cache):
    n_head, n_kv, hd, new, past, page = shape
    b = Batch([new], [past])
    units, items = sharing(b, n_head, n_kv, window)
    assert units > 12 and items >= 2, (units, items)  # sums put aside twice over in f32; every ring turns
    c = filled([past], [new], page, n_kv, hd, cache, 1e6, 1)
    q = randn(43, new, n_head, hd, dtype)
    got = c.attend(q, b, 1e6, 1, window=window)
    close(got, attention(c, q, b, 1e6, 1, window))
    assert torch.equal(c.attend(q, b, 1e6, 1, window=window), got)


@pytest.mark.parametrize("cache", [torch.float16, F8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_prompts_and_steps_in_one_call(dtype, cache):
    new, past = [900, 1, 700, 3, 1200, 0], [2500, 4000, 0, 100, 4000, 9]
    n_head, n_kv, hd = 10, 2, 128
    b = Batch(new, past)
    units, items = sharing(b, n_head, n_kv, 0)
    assert units > 12 and items >= 2, (units, items)
    c = filled(past, new, 32, n_kv, hd, cache, 1e4, 0)
    q = randn(44, b.rows, n_head, hd, dtype)
    close(c.attend(q, b, 1e4, 0), attention(c, q, b, 1e4, 0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cache", [torch.float16, F8])
def test_attention_over_offsets_past_32_bits(cache, dtype):
    """both kernels over the last pages of a pool of more than 2^31 elements, against the same pages in a small one"""
    from mesh_llm_b200 import ops

    hd, n_kv, page, n = 128, 8, 256, 300
    n_pages = (1 << 31) // (hd * n_kv * page) + 3
    big = ops.kv_pages(n_pages, page, n_kv, hd, cache)
    small = filled([0], [n], page, n_kv, hd, cache, 1e6, 1)
    table = torch.tensor([[n_pages - 1, n_pages - 2]], dtype=torch.int32, device="cuda")
    for x, y in zip(big, (small.k, small.v, small.ks, small.vs)):
        for i in range(2):
            if x is not None:
                x.view(torch.uint8)[n_pages - 1 - i] = y.view(torch.uint8)[small.table[0, i].long()]
    for new in (1, n):
        b = Batch([new], [n - new])
        q = randn(45, new, 16, hd, dtype)
        got = ops.attention_pages(q, big[0], big[1], table, b.start, b.pos0, new, 1e6, 1, k_scale=big[2], v_scale=big[3])
        assert torch.equal(got, small.attend(q, b, 1e6, 1))


@pytest.mark.parametrize("cache", [torch.float16, F8])
def test_prompts_captured_once_with_lengths_that_change(cache):
    """a graph of append and attention follows the rows and positions that the device holds at its replay, prompts and steps in any place"""
    n_head, n_kv, hd, rows = 10, 2, 128, 500
    c, e = (Cache(4, 900, 32, n_kv, hd, cache, seed=41) for _ in "ce")
    q, k, v = randn(46, rows, n_head, hd), randn(47, rows, n_kv, hd), randn(48, rows, n_kv, hd)
    b = Batch([rows, 0, 0, 0], [0, 0, 0, 0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.append(k, v, b, 1e4, 1)
        out = c.attend(q, b, 1e4, 1, max_rows=rows)
    past = [0, 0, 0, 0]
    for new in ([rows, 0, 0, 0], [1, 300, 2, 197], [1, 1, 350, 1], [0, 80, 1, 400], [3, 1, 1, 1], [90, 90, 90, 90]):
        step = Batch(new, past)
        b.start.copy_(step.start)
        b.pos0.copy_(step.pos0)
        out.zero_()
        g.replay()
        e.append(k[:step.rows], v[:step.rows], step, 1e4, 1)
        assert torch.equal(out[:step.rows], e.attend(q[:step.rows], step, 1e4, 1, max_rows=rows))
        assert (out[step.rows:] == 0).all()
        close(out[:step.rows], attention(e, q[:step.rows], step, 1e4, 1))
        past = [p + t for p, t in zip(past, new)]


def test_prompts_on_streams_at_once():
    c, b = filled([900], [300], 64, 2, 128, torch.float16, 1e4, 1), Batch([300], [900])
    q = randn(49, 300, 16, 128, torch.bfloat16)
    want = c.attend(q, b, 1e4, 1)
    close(want, attention(c, q, b, 1e4, 1))
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for i in range(30):
        with torch.cuda.stream(streams[i % 3]):
            got.append(c.attend(q, b, 1e4, 1))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


@pytest.mark.parametrize("cache", [torch.float16, F8])
def test_more_sequences_than_threads_and_more_heads_than_rows(cache):
    """700 sequences of which some are prompts; 300 query heads on one KV head"""
    new = [1 if i % 100 else 150 for i in range(700)]
    past = [(37 * i) % 190 for i in range(700)]
    c, b = filled(past, new, 16, 1, 64, cache, 1e4, 1), Batch(new, past)
    q = randn(50, b.rows, 2, 64)
    close(c.attend(q, b, 1e4, 1), attention(c, q, b, 1e4, 1))
    for t in (1, 3, 40):
        c, b = filled([500], [t], 32, 1, 128, cache, 1e4, 0), Batch([t], [500])
        q = randn(51, t, 300, 128)
        for most in (t, 0):
            close(c.attend(q, b, 1e4, 0, max_rows=most), attention(c, q, b, 1e4, 0))
