"""How exactly attention over the cache held in 4 bits computes its scores: products
of the queries with the numbers that the codes stand for, summed in fp32, whatever
the sizes of the other products beside them.  The bounds are kv_ref's, which count
fp32 products and sums: off by (D + 8) 2^-24 of the sum of the products' magnitudes.
"""
import pytest
import torch

import test_kv_cache_mx4_gpu as G

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
ROWS = (1, 40, 100, 300)  # of a cache head: few for either type, and many


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("q", ROWS)
def test_products_that_cancel(q, D, dtype):
    """Two channels of queries and keys are far larger than the others and cancel:
    2 x 512 x 48 beside products of about 1."""
    b = G.make([(q, 300), (min(q, 9), 50)], 4, 4, D, 16, dtype, seed=q + D)
    b["q"][..., 5] = b["q"][..., 6] = 512
    codes, scales = b["c"][:2]
    codes[..., :16] = 0
    codes[..., 2], codes[..., 3] = 7 << 4, 15  # elements 5 and 6: 6 and -6 scales
    scales[..., 0].masked_fill_(scales[..., 0] != 255, 127 + 3)
    G.check(b)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("q", ROWS)
def test_small_numbers_beside_large_ones(q, D, dtype):
    """A channel of the queries is 2^16 times the others, and 0 in the keys."""
    b = G.make([(q, 300), (min(q, 9), 50)], 4, 4, D, 16, dtype, seed=q + D)
    b["q"] = b["q"] * 2.0 ** -7
    b["q"][..., 8::32] = 512
    codes = b["c"][0]
    codes[..., 4::16] &= 0xf0  # element 8 of each block
    G.check(b, scale=2.0 ** 7 * D ** -0.5)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("q", ROWS)
def test_a_query_with_an_infinity(q, dtype):
    """In bf16 it follows the products, and a score of -inf weighs nothing; in fp32
    the row is NaN."""
    b = G.make([(q, 200)], 4, 4, 64, 16, dtype, seed=q, poison=False)
    b["c"][0][..., 3] = 0x22  # elements 6 and 7: 1 scale, in every key
    clean = G.call(b)
    b["q"][0, 1, 6], b["q"][q - 1, 2, 7] = -torch.inf, torch.inf
    out = G.call(b)
    nan = torch.zeros_like(out, dtype=torch.bool)
    nan[q - 1, 2] = True
    nan[0, 1] = dtype == F32 and q <= 200  # (with more new tokens than all, row 0 sees no key)
    zero = torch.zeros_like(nan)
    zero[0, 1] = not nan[0, 1].any()
    assert torch.equal(torch.isnan(out), nan)
    assert not out[zero].any() and torch.equal(out[~nan & ~zero], clean[~nan & ~zero])
