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
