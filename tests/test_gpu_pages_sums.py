"""What the prompts' kernel makes of its sums, with inputs whose exact results are known: one query element meets one key element, so that the scores are the
keys' first elements, and every CTA sums many units of 128 keys.

The tensor cores cut a product off at 2^-25 of the sum that it joins, and a step's sum to 24 bits, instead of rounding.
"""
import pytest
import torch

from tests.pages_util import Batch, Cache, attention

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def first_element(rows, heads, hd, dtype=torch.float32):
    q = torch.zeros((rows, heads, hd), dtype=dtype, device="cuda")
    q[..., 0] = 1
    return q


def filled(scores, values, page, cache):
    """a sequence with keys of these scores [n, n_kv] and these values [n, n_kv, hd]"""
    n, n_kv, hd = values.shape
    c = Cache(1, n, page, n_kv, hd, cache, seed=30)
    k = torch.zeros((n, n_kv, hd), device="cuda")
    k[..., 0] = scores
    c.append(k, values, Batch([n], [0]), 0.0, 0)
    return c


def eighths(seed, n, n_kv, hd):
    """1, 1.125 .. 1.875: exact in every page type"""
    g = torch.Generator("cuda").manual_seed(seed)
    return 1 + torch.randint(0, 8, (n, n_kv, hd), generator=g, device="cuda") / 8


@pytest.mark.parametrize("cache", [torch.float16, F8])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("weight", ["alone", "first", "middle", "equal"])
def test_sums_that_lose_nothing(weight, hd, cache):
    """Rows whose weight is on one of their keys (which may be the only one that they see), or whose keys all weigh the same: O loses nothing, so its divisor must not either.
    Roundings left: the second part of a probability of 2^6 (1 + d) cut off in O and in the divisor, 2^-23 each; pieces joined, two products and a sum
    for each of the two, the division and its product: 6 of 2^-24.  Together 10 2^-24."""
    n_kv, n_head = 8, 40
    new, past = (600, 0) if weight == "alone" else (512, 3000)
    n = new + past
    scores = torch.zeros((n, n_kv), device="cuda")
    if weight in ("alone", "first"):
        scores[1:] = -40
    elif weight == "middle":
        scores[:1700] = -40
        scores[1701:] = -40
    c = filled(scores, eighths(1, n, n_kv, hd), 64, cache)
    q, b = first_element(new, n_head, hd), Batch([new], [past])
    got, want = c.attend(q, b, 0.0, 0, scale=1.0).double(), attention(c, q, b, 0.0, 0, scale=1.0)
    off = ((got - want).abs() / want.abs()).max().item()
    assert off <= 10 * 2.0 ** -24, off


def some_rows(scores, values, new, past, n_head):
    """rows and what they are, from the definition in 64 bits: the queries are alike, so the heads of a KV head are too"""
    at = sorted({0, min(1, new - 1), new // 2, new - 1})
    out = []
    for r in at:
        n = past + r + 1
        w = torch.softmax(scores[:n].double(), 0)
        out.append(torch.einsum("nh,nhd->hd", w, values[:n].double()).repeat_interleave(n_head // values.shape[1], 0))
    return at, torch.stack(out)


def one_beside_many(below, ones, n, n_kv, hd):
    """scores of the first key 0, of the others -below; values 1, or f16 numbers from 1 to 2"""
    scores = torch.full((n, n_kv), -below, device="cuda")
    scores[0] = 0
    g = torch.Generator("cuda").manual_seed(2)
    values = torch.ones((n, n_kv, hd), device="cuda")
    if not ones:
        values += torch.rand(values.shape, generator=g, device="cuda")
    return scores, values.half().float()


@pytest.mark.parametrize("below, ones, n_kv, new, past, bound", [(10.0, False, 8, 512, 3000, 1.2e-5), (14.0, True, 8, 512, 3000, 1.2e-5), (16.0, True, 8, 512, 3000, 1.2e-5),
                                                                 (18.0, False, 8, 512, 3000, 1.2e-5), (14.0, False, 4, 1280, 60000, 1e-5)])
def test_one_key_that_outweighs_many(below, ones, n_kv, new, past, bound):
    """A large weight, then thousands of small ones whose products are cut off at 2^-25 of the sum.  O is put aside once a unit has added little, so two units of
    128 keys can lose that much of each product: 7.6e-6; the cut-off results of their 32 steps, of which the divisor's take back half: 1e-6; the roundings of
    the test above: 6e-7; the small weights among themselves, 4e-6 of their part, which is at most a half: 2e-6 (a twentieth behind 60000 keys: 2e-7); their f16 parts, 2^-25 each
    where the large one is 2^11: 1e-6 behind 60000."""
    scores, values = one_beside_many(below, ones, new + past, n_kv, 128)
    c = filled(scores, values, 64, torch.float16)
    at, want = some_rows(scores, values, new, past, 40)
    got = c.attend(first_element(new, 40, 128), Batch([new], [past]), 0.0, 0, scale=1.0)[at].double()
    off = ((got - want).abs() / want).max().item()
    assert off <= bound, off


def half_steps(got, want):
    """the largest difference, in half steps of got's type at want"""
    u = torch.finfo(got.dtype).eps / 2
    return ((got.double() - want).abs() / (2.0 ** want.abs().log2().floor() * u)).max().item()


@pytest.mark.parametrize("cache", [torch.float16, F8])
@pytest.mark.parametrize("below", [2.0, 6.0, 9.0])
def test_f16_prompts_round_once(below, cache):
    """Probabilities enter f16 prompts in one f16 part, half a step of 2^-11 off at most, and the divisor is their sum: the weights of one key and of all others, at most a
    quarter multiplied, are off by 2^-11 against each other, over values at most 1 apart: 1/4 half step of results from 1 to 2.  27 units of 128 keys, each cut off by
    1.9e-6: 0.1 half steps.  With the result's own rounding 1.35."""
    n_kv, new, past = 8, 512, 3000
    scores, values = one_beside_many(below, False, new + past, n_kv, 128)
    if cache == F8:
        values = eighths(3, new + past, n_kv, 128)
    c = filled(scores, values, 64, cache)
    at, want = some_rows(scores, values, new, past, 40)
    off = half_steps(c.attend(first_element(new, 40, 128, torch.float16), Batch([new], [past]), 0.0, 0, scale=1.0)[at], want)
    assert off <= 1.35, off


@pytest.mark.parametrize("dtype, past, bound", [(torch.float16, 60000, 1.75), (torch.bfloat16, 150000, 1.45)])
@pytest.mark.parametrize("below", [14.0, 11.0, 0.0])
def test_long_rows_of_16_bits(below, dtype, past, bound):
    """A CTA sums hundreds of units of 128 keys, each cut off by 1.9e-6 of what it joins: by 32 of them, f16, or 128, bf16, at most.  In half steps of results from 1 to
    2: f16 0.12 and, as probabilities are rounded, 1/2 at most (1/4 of the test above, twice over for sums of unlike units); bf16 2 x 0.06, its probabilities and their sum
    2 x 2^-11 x 2^7 = 0.12 and as much again for the units', the cubic 2 x 0.02.  With the result's own rounding 1.75 and 1.45."""
    n_kv, new = 4, 1280
    scores, values = one_beside_many(below, False, new + past, n_kv, 128)
    c = filled(scores, values, 64, torch.float16)
    at, want = some_rows(scores, values, new, past, 40)
    off = half_steps(c.attend(first_element(new, 40, 128, dtype), Batch([new], [past]), 0.0, 0, scale=1.0)[at], want)
    assert off <= bound, off


@pytest.mark.parametrize("cache", [torch.float16, F8])
@pytest.mark.parametrize("dtype, bound", [(torch.float32, 256.0), (torch.float16, 1.2), (torch.bfloat16, 1.45)])
def test_steps_of_long_rows(dtype, bound, cache):
    """120 sequences over the pages of one, so that a CTA sums an item of 131072 keys alone, 2048 steps a warp.  f32: each step is added with a rounding of 2^-24 at
    most, of O and of the divisor: four times the square root of 2 x 2048, 256 half steps.  f16: both parts, the same 256 half steps of f32 are 1/32 of f16's: with the
    result's own rounding and the second parts' 1.2.  bf16: the tensor cores add up a warp's steps over f16 pages, 16 products a step cut off by 2^-26 each: 4.9e-4, an eighth of a half
    step of results from 1 to 2, twice that where they are near 2; probabilities 2 x 2^-11 x 2^7 / 2; 1.45."""
    n, n_kv, n_seq = 131072, 4, 120
    g = torch.Generator("cuda").manual_seed(4)
    scores = -12 + torch.randn((n, n_kv), generator=g, device="cuda")
    scores[0] = 0
    values = eighths(5, n, n_kv, 128)
    c = filled(scores, values, 256, cache)
    k = c.rows(0, n)[0][..., 0]  # the scores as the pages have them
    c.table = c.table.expand(n_seq, -1).contiguous()
    _, want = some_rows(k, values, 1, n - 1, 8)
    q = first_element(n_seq, 8, 128, dtype)
    got = c.attend(q, Batch([1] * n_seq, [n - 1] * n_seq), 0.0, 0, scale=1.0)
    off = half_steps(got, want.expand(n_seq, -1, -1))
    assert off <= bound, off


@pytest.mark.parametrize("past", [1536, 8000])
@pytest.mark.parametrize("cache", [torch.float16, F8])
def test_f32_prompts_of_random_rows(cache, past):
    """Relative 2-norm of the error of ordinary rows, whose values are of either sign.  O's steps are cut off to 24 bits, half a last bit each on average, and the divisor's are too;
    what is left is the products' own cutting, 2^-26 of the sum for each of 768 keys at most and of either sign (0.5 sqrt(768) 2^-26 sqrt(1/3): 1.2e-7 for each part), the
    spread of 192 cuts of up to 2^-23 (sqrt(192 / 12) 2^-23 x 2/3 as sums grow: 3.2e-7, O's and the divisor's: 4.5e-7), half of the bias where they do not match (96 x 2^-24 x 2/3 / 2 / 2: 9.5e-7),
    and scores of 22 and 24 bits (2^-22 of up to 3: 7e-7 on a probability, over many keys 4e-7).  Together 1.2e-6."""
    g = torch.Generator("cuda").manual_seed(6)
    n_head, n_kv, new = 40, 8, 512
    k, v = (torch.randn((new + past, n_kv, 128), generator=g, device="cuda") for _ in "kv")
    c = Cache(1, new + past, 64, n_kv, 128, cache, seed=31)
    c.append(k, v, Batch([new + past], [0]), 1e6, 1)
    q, b = torch.randn((new, n_head, 128), generator=g, device="cuda"), Batch([new], [past])
    want = attention(c, q, b, 1e6, 1)
    off = ((c.attend(q, b, 1e6, 1).double() - want).norm() / want.norm()).item()
    assert off <= 1.2e-6, off
