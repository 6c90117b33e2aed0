"""Attention over caches in 4 bits that are not near: keys and values laid out
differently, or pages 2^24 bytes and more apart.  Their places are found by products
of 64 bits or of units of 16 bytes, in code that the usual caches do not reach; the
references and bounds are those of test_kv_cache_mx4_gpu.py."""
import pytest
import torch

import mx4_ref as M
import test_kv_cache_mx4_gpu as G

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
DIMS = [8, 40, 64, 80, 96, 104, 128, 160, 200, 256]


def spread(t, layout):
    """The same contents with other strides."""
    if layout == "nhd":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    pages, heads, size, b = t.shape
    if layout == "padded":  # tokens further apart (rows of codes stay on 16 bytes)
        out = torch.zeros(pages, heads, size, b + (16 if b % 16 == 0 else 3), dtype=t.dtype, device=t.device)[..., :b]
    else:  # "pages": 2^24 bytes and more apart
        stride = (1 << 24) + 64
        buf = torch.empty((pages - 1) * stride + heads * size * b, dtype=t.dtype, device=t.device)
        out = buf.as_strided(t.shape, (stride, size * b, b, 1))
    out.copy_(t)
    return out


def apart(c, layout):
    kc, ks, vc, vs = c
    if layout == "scales":  # codes alike, scales not
        return kc, ks, vc, spread(vs, "padded")
    if layout == "pages":
        return tuple(spread(t, "pages") for t in c)
    return kc, ks, spread(vc, layout), spread(vs, layout)


def both(lens, H, KV, D, page, dtype, layout, seed, **kw):
    """Checked against the reference, and bit for bit against a near cache."""
    b = G.make(lens, H, KV, D, page, dtype, seed=seed)
    near = G.call(b, **kw)
    b["c"] = apart(b["c"], layout)
    out = G.check(b, **kw)
    assert torch.equal(out, near)
    return b


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("layout", ["nhd", "padded", "scales"])
def test_values_laid_out_otherwise(layout, D, dtype):
    both([(1, 300), (5, 40), (1, 1)], 8, 2, D, 16, dtype, layout, D)            # few rows
    both([(70, 199), (90, 90), (3, 33)], 8, 2, D, 24, dtype, layout, D + 1)     # many
    both([(1, 700), (2, 90)], 4, 4, D, 16, dtype, layout, D + 2, window=100)
    both([(60, 250), (41, 250)], 4, 2, D, 16, dtype, layout, D + 3, window=31)
    both([(64, 64), (33, 33)], 8, 2, D, 8, dtype, layout, D + 4, causal=False)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_pages_far_apart(D, dtype):
    for q in (1, 100):
        both([(q, 150), (min(q, 20), 35)], 8, 2, D, 16, dtype, "pages", q + D)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("layout", ["nhd", "scales"])
def test_long(layout, dtype):
    both([(1, 9001), (3, 4500)], 8, 2, 128, 64, dtype, layout, 1)
    both([(80, 5003)], 8, 2, 64, 64, dtype, layout, 2)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D,page", [(64, 16), (80, 24), (96, 16), (128, 16), (256, 32)])
@pytest.mark.parametrize("layout", ["nhd", "scales"])
def test_not_finite(layout, D, page, dtype):
    """A block that is not a number shows in the rows that see it, a value's in its
    columns only."""
    group, last = 4, M.blocks(D) - 1
    for q, n in ((1, 90), (3, 70), (40, 200), (200, 200)):
        b = G.make([(q, n), (min(q, 5), 33)], 8, 2, D, page, dtype, seed=q)
        clean = G.call(b)
        held = [t.clone() for t in b["c"]]
        toks = sorted({n - 1, n - q // 2 - 1, max(n - q, 0), 3})
        want = torch.zeros_like(clean, dtype=torch.bool)
        row = torch.arange(n - q, n, device=G.DEV)
        for tok, block in zip(toks, [last, 0, last, 0]):
            G.poisoned(b, 0, tok, page, 1, block)
            want[:q, group:, 32 * block:32 * block + 32] |= (row >= tok)[:, None, None]
        b["c"] = apart(b["c"], layout)
        out = G.call(b)
        assert torch.equal(torch.isnan(out), want) and torch.equal(out[~want], clean[~want])
        tok = n - q // 2 - 1
        held[1][b["table"][0, tok // page].item(), 0, tok % page, last] = 253
        b["c"] = apart(held, layout)
        out, want = G.call(b), torch.zeros_like(want)
        want[:q, :group] = (row >= tok)[:, None, None]
        assert torch.equal(torch.isnan(out), want) and torch.equal(out[~want], clean[~want])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_rows_that_see_nothing_and_pages_outside(D, dtype):
    b = G.make([(1, 50), (30, 30), (4, 9), (70, 200)], 8, 2, D, 16, dtype, seed=9)
    b["c"] = apart(b["c"], "nhd")
    b["ctx"] = G.i32([0, 11, 9, 200])
    for at, page in ((3, -1), (5, 2 ** 31 - 1), (7, b["c"][0].size(0))):
        b["table"][3, at] = page
    out = G.check(b)
    assert not out[:20].any() and out[20:].any()
    one = dict(b, q=b["q"][:4].contiguous(), cu=G.i32([0, 1, 2, 3, 4]), max_q=1)
    G.check(one)
