"""GPU parity of the cache held in 4 bits against plain references (mx4_ref.py):
codes and scales exactly, rotated queries and attention in float64 within the
bounds of kv_ref.py, which count fp32 products and sums, weights and outputs of
the operands' type; the cache's numbers take part exactly, so they add nothing."""
import math
import random

import pytest
import torch

import kv_ref as R
import mx4_ref as M
import zentorch  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda"
ops = torch.ops.zentorch
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _announce(request):
    print(f"\n[case] {request.node.name}", flush=True)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def i64(v):
    return torch.tensor(v, dtype=torch.int64, device=DEV)


def laid_out(c, layout):
    """The cache's four tensors in another layout, of the same contents."""
    kc, ks, vc, vs = c
    pages, heads, size, b = kc.shape
    nb = ks.size(3)
    if layout == "pair":   # keys and values of a page beside each other
        codes, scales = torch.stack([kc, vc], 1), torch.stack([ks, vs], 1)
        return codes[:, 0], scales[:, 0], codes[:, 1], scales[:, 1]
    if layout == "nhd":    # a page's tokens outermost
        return tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in c)
    if layout == "rows":   # a page's codes and scales, of keys and values, in one piece
        # rows of codes on 16 bytes; the scales at an odd place behind them
        piece = -(-(2 * heads * size * (b + nb) + 1) // 16) * 16
        buf = torch.zeros(pages, piece, dtype=torch.uint8, device=kc.device)
        out, n = [], heads * size
        for i, t in enumerate((kc, vc)):
            codes = buf.as_strided(t.shape, (piece, size * b, b, 1), i * n * b)
            codes.copy_(t)
            out.append(codes)
        for i, t in enumerate((ks, vs)):
            scales = buf.as_strided(t.shape, (piece, size * nb, nb, 1), 2 * n * b + 1 + i * n * nb)
            scales.copy_(t)
            out.append(scales)
        return out[0], out[2], out[1], out[3]
    return c


def make(lens, H, KV, D, page, dtype, seed=0, spare=3, width=None, layout="hnd", poison=True):
    """A batch of (new, all) tokens over scattered pages.  What no sequence
    holds is NaN, so that a kernel that reads it shows it."""
    g = torch.Generator().manual_seed(seed)
    r = random.Random(seed)
    counts = [-(-n // page) for _, n in lens]
    pool = sum(counts) + spare
    ids = r.sample(range(pool), sum(counts))
    width = width or max(counts + [1]) + 1
    rows, at = [], 0
    for n in counts:
        rows.append(ids[at:at + n] + [r.choice([-1, pool, 2 ** 31 - 1])] * (width - n))
        at += n
    cu = [0]
    for q, _ in lens:
        cu.append(cu[-1] + q)
    q = (torch.randn(cu[-1], H, D, generator=g) * (torch.rand(H, 1, generator=g) * 2 + 0.5)).to(dtype)
    c = M.filled(pool, KV, page, D, seed=seed)
    if poison:
        held = torch.zeros(pool, page, dtype=torch.bool)
        for i, (_, n) in enumerate(lens):
            for j in range(n):
                held[rows[i][j // page], j % page] = True
        for t in c:
            t.masked_fill_(~held[:, None, :, None].to(DEV), 255)
    return dict(q=q.to(DEV), c=laid_out(c, layout), table=i32(rows), cu=i32(cu),
                ctx=i32([n for _, n in lens]), max_q=max([q for q, _ in lens] + [0]))


def call(b, **kw):
    return ops.zentorch_paged_attention_mxfp4(b["q"], *b["c"], b["table"], b["cu"], b["ctx"],
                                              kw.pop("max_q", b["max_q"]), **kw)


def check(b, out=None, **kw):
    out = call(b, **kw) if out is None else out
    torch.cuda.synchronize()
    kw.pop("max_q", None)
    ref, bound = M.attention(b["q"], b["c"], b["table"], b["cu"], b["ctx"], **kw)
    assert out.shape == b["q"].shape and out.dtype == b["q"].dtype
    err = (out.double() - ref).abs()
    assert torch.isfinite(out).all(), "not finite"
    assert (err <= bound).all(), f"off by {(err - bound).max().item()} over a bound of {bound.max().item()}"
    return out


HEADS = [(8, 2), (4, 4), (7, 1), (16, 2), (6, 2), (24, 2)]


# ------------------------------------------------------------- write, read
def rope(n, rot, seed=0):
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.arange(n, dtype=torch.float64)[:, None] * f
    return (torch.cat([a.cos(), a.sin()], 1) * 1.1).float().to(DEV)


def tokens(T, H, KV, D, dtype, seed, fused=True):
    """Query, key and value, whose blocks have all kinds of sizes."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H + 2 * KV, D, generator=g)
    x = x * torch.exp2(torch.randint(-30, 30, (T, H + 2 * KV, 1), generator=g).float())
    x = x * torch.exp2(torch.randint(-3, 3, (T, H + 2 * KV, D), generator=g).float())
    x[:, :, ::7] = (x[:, :, ::7] * 4).round() / 4  # numbers halfway between two codes among them
    x = x.to(dtype).to(DEV)
    if fused:
        x = x.flatten(1)
        return tuple(t.unflatten(1, (-1, D)) for t in x.split([H * D, KV * D, KV * D], dim=1))
    return tuple(t.contiguous() for t in x.split([H, KV, KV], dim=1))


def check_append(T, H, KV, D, rot, page, dtype, interleaved=False, seed=0, layout="hnd", pos=None, fused=True,
                 length=512, qkv=None):
    r = random.Random(seed)
    pool = -(-T // page) + 2
    where = r.sample(range(pool * page), T)
    if T > 2:
        where[1], where[T - 1] = -1, pool * page  # padding, and a slot past the pool
    q, k, v = qkv or tokens(T, H, KV, D, dtype, seed, fused)
    pos = i64([r.randrange(length) for _ in range(T)]) if pos is None else pos
    table, slots = rope(length, rot), i64(where)
    before = laid_out(M.cache(pool, KV, page, D, fill=0x5a), layout)
    c = laid_out(M.cache(pool, KV, page, D, fill=0x5a), layout)
    out = ops.zentorch_rotary_cache_append_mxfp4(q, k, v, pos, table, slots, *c, interleaved=interleaved)
    torch.cuda.synchronize()
    ref, bound = R.rotary(q, pos, table, interleaved)
    nan = torch.isnan(ref)
    over = q.double().abs().amax(-1, keepdim=True).expand_as(ref) * 2.2 > torch.finfo(F32).max
    # (the difference of two infinite products is a NaN that 64 bits do not have)
    assert torch.equal(torch.isnan(out)[~over], nan[~over])
    # The bound counts roundings relative to their results.  Below the smallest
    # normal number a rounding is off by half the smallest step instead: 2^-150
    # for each of three in fp32, and in bf16 2^-134 for the last.
    bound = bound + 3 * 2.0 ** -150 + (2.0 ** -134 if dtype == BF else 0)
    # And a result that the bound takes past the largest number may be infinite,
    # as may one whose products (each up to 1.1 times an input) are.
    most = torch.finfo(dtype).max
    wide = over | (ref.abs() + bound > most)
    assert ((out.double() - ref).abs() <= bound)[~nan & ~wide].all()
    key, _ = R.rotary(k, pos, table, interleaved)
    want = [t.clone() for t in before]
    held = (slots >= 0) & (slots < pool * page)
    at = slots[held] // page, slice(None), slots[held] % page
    for i, x in enumerate((key, v)):
        want[2 * i][at], want[2 * i + 1][at] = M.quantise(x[held])
    for got, w, name in zip(c, want, ("key codes", "key scales", "value codes", "value scales")):
        assert torch.equal(got, w), f"{name}: {(got != w).sum().item()} bytes differ"
    back = ops.zentorch_cache_read_mxfp4(*c, slots, D, dtype=dtype)
    torch.cuda.synchronize()
    for i, got in enumerate(back):
        w = torch.zeros(T, KV, D, dtype=torch.float64, device=DEV)
        w[held] = M.values(want[2 * i][at], want[2 * i + 1][at], D)
        assert got.shape == w.shape and got.dtype == dtype
        torch.testing.assert_close(got.double(), w, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [8, 24, 32, 40, 64, 72, 80, 96, 128, 200, 256])
def test_append_head_dims(D, dtype):
    for rot in {D, max(2, D // 2), max(2, D // 4 * 2 - 2), 2}:
        for il in (False, True):
            check_append(9, 6, 2, D, rot, 16, dtype, il, seed=D + rot)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,H,KV,page", [(1, 32, 8, 16), (2, 1, 1, 1), (5, 7, 7, 3), (33, 12, 2, 24), (700, 28, 4, 128)])
def test_append_batches(T, H, KV, page, dtype):
    check_append(T, H, KV, 128, 128, page, dtype, seed=T)
    check_append(T, H, KV, 64, 32, page, dtype, True, seed=T, fused=False)


@pytest.mark.parametrize("layout", ["pair", "nhd", "rows"])
def test_append_layouts(layout):
    for dtype in (BF, F32):
        check_append(20, 4, 2, 80, 80, 8, dtype, seed=3, layout=layout)
        check_append(20, 4, 3, 128, 64, 8, dtype, seed=4, layout=layout)


def test_append_borders():
    """Numbers on and next to every border between two codes and two scales:
    a key at position 0 is turned by an angle of 0 (the table's factor is 1.1,
    so values alone are exact there), and values are not turned."""
    T, D = 64, 128
    r = random.Random(0)
    rows = torch.zeros(T, 1, D, dtype=torch.float64)
    cuts = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    for t in range(T):
        e = r.choice([-125, -100, -1, 0, 3, 100, 124])
        for b in range(4):
            top = r.choice([3.5, 4.0, 6.0, 6.9999995, 7.0, 5.0, 13.999999])
            for i in range(32):
                x = top if i == 5 else r.choice(cuts) * (1 + r.choice([0, 0, 2.0 ** -23, -2.0 ** -24, 2.0 ** -7]))
                rows[t, 0, 32 * b + i] = r.choice([-1, 1]) * x * 2.0 ** e
    rows = rows.to(DEV)
    for dtype in (F32, BF):
        v = rows.to(dtype)
        check_append(T, 1, 1, D, 64, 16, dtype, seed=1, qkv=(v.clone(), v.clone(), v), pos=i64([0] * T))


def test_append_extremes():
    """Zeros, the smallest and the largest numbers, infinities and NaN."""
    D = 64
    kinds = [0.0, -0.0, 2.0 ** -149, 2.0 ** -133, 2.0 ** -126, 2.0 ** -124, 2.0 ** 127, 3.3895313892515355e38,
             math.inf, -math.inf, math.nan, 1.0]
    for dtype in (F32, BF):
        v = torch.zeros(len(kinds), 2, D, device=DEV, dtype=dtype)
        for i, x in enumerate(kinds):
            v[i, 0, 40] = x
            v[i, 1] = x
            v[i, 1, ::3] = 0.75
        pos = i64([-1] * len(kinds))  # rows without a position are not turned
        check_append(len(kinds), 2, 2, D, D, 16, dtype, qkv=(v.clone(), v.clone(), v), pos=pos)
    # turned: sums past the largest fp32 number, and positions past the table
    k = torch.full((3, 1, D), 3e38, device=DEV)
    check_append(3, 1, 1, D, D, 16, F32, qkv=(torch.ones_like(k), k, k), pos=i64([100, 511, 600]), length=512)


def test_append_of_nothing():
    c = M.cache(4, 2, 16, 64)
    q, kv, none = torch.empty(0, 4, 64, device=DEV), torch.empty(0, 2, 64, device=DEV), i64([])
    assert ops.zentorch_rotary_cache_append_mxfp4(q, kv, kv, none, rope(8, 64), none, *c).shape == (0, 4, 64)
    assert ops.zentorch_cache_read_mxfp4(*c, none, 64)[0].shape == (0, 2, 64)
    c = M.cache(0, 2, 16, 64)  # no pages: every slot is outside
    one = i64([0])
    k, v = ops.zentorch_cache_read_mxfp4(*c, one, 64, dtype=F32)
    assert k.dtype == F32 and not k.any() and not v.any()


def test_read_any_bytes():
    """Every code under every scale byte, as often as asked for."""
    scales = torch.arange(256, dtype=torch.uint8, device=DEV).view(16, 1, 16, 1)
    codes = torch.arange(16, dtype=torch.uint8, device=DEV).mul(17).expand(16, 1, 16, 16).contiguous()
    slots = i64(list(range(256)) + [3] * 50 + [-1, 256, -2 ** 60, 2 ** 60])
    for dtype in (F32, BF):
        k, v = ops.zentorch_cache_read_mxfp4(codes, scales, codes.flip(3), scales, slots, 32, dtype=dtype)
        want = M.values(codes, scales, 32).view(256, 1, 32)
        want = torch.cat([want, want[3:4].expand(50, 1, 32), want.new_zeros(4, 1, 32)])
        torch.testing.assert_close(k.double(), want, rtol=0, atol=0, equal_nan=True)
        torch.testing.assert_close(v.double(), want.unflatten(2, (16, 2)).flip(2).flatten(2), rtol=0, atol=0,
                                   equal_nan=True)


# -------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [8, 24, 32, 64, 72, 80, 96, 128, 160, 200, 256])
def test_attn_head_dims(D, dtype):
    check(make([(1, 77), (5, 40), (70, 70)], 8, 2, D, 16, dtype, seed=D))
    check(make([(1, 300), (1, 1)], 8, 2, D, 16, dtype, seed=D + 1))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H,KV", HEADS)
def test_attn_groups(H, KV, dtype):
    check(make([(1, 130), (3, 33), (1, 1), (50, 129)], H, KV, 64, 16, dtype, seed=H))
    check(make([(1, 200), (1, 513)], H, KV, 128, 16, dtype, seed=H + 1))


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 32, 64, 100, 128])
@pytest.mark.parametrize("q", [1, 2, 60])
def test_attn_pages(page, q):
    check(make([(q, 61 + page), (q, 200), (min(q, 7), 7)], 8, 2, 128, page, BF, seed=page))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000])
def test_attn_lengths(n, dtype):
    """Decoding, whole sequences, and a chunk of every such length."""
    check(make([(1, n), (n, n), (min(n, 16), n)], 4, 2, 64, 16, dtype, seed=n))
    check(make([(1, n)], 4, 1, 64, 16, dtype, seed=n))
    check(make([(n, n)], 4, 2, 64, 16, dtype, seed=n), causal=False)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("window", [1, 2, 16, 31, 100, 1000])
@pytest.mark.parametrize("D", [64, 128])
def test_attn_window(window, D, dtype):
    check(make([(1, 300), (40, 300), (130, 130), (1, 5)], 8, 2, D, 16, dtype, seed=window), window=window)
    check(make([(1, 700), (2, 90)], 8, 2, D, 16, dtype, seed=window), window=window)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attn_many_ragged(dtype):
    r = random.Random(5)
    lens = [(1 if r.random() < 0.7 else r.randint(1, 90), r.randint(1, 700)) for _ in range(67)]
    lens = [(min(q, n), n) for q, n in lens]
    check(make(lens, 12, 2, 80, 24, dtype, seed=5))
    check(make([(1, n) for _, n in lens], 12, 2, 80, 24, dtype, seed=6))


@pytest.mark.parametrize("q", [1, 4, 16, 40, 300])
def test_attn_long(q):
    """Few rows, a long axis: the work of one row is split and joined."""
    check(make([(q, 20011), (q, 9973)], 8, 2, 128, 64, BF, seed=q))
    if q <= 40:
        check(make([(q, 5003)], 8, 2, 64, 64, F32, seed=q))


@pytest.mark.parametrize("layout", ["pair", "nhd", "rows"])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_attn_layouts(layout, D):
    for dtype in (BF, F32):
        check(make([(1, 100), (70, 99), (3, 40)], 8, 2, D, 16, dtype, seed=D, layout=layout))
    check(make([(1, 1000)], 8, 2, D, 16, BF, seed=D, layout=layout))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 40.0])
def test_attn_scale(scale, dtype):
    check(make([(1, 100), (40, 90)], 8, 2, 64, 16, dtype, seed=2), scale=scale)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_attn_rows_that_see_nothing(D, dtype):
    b = make([(1, 50), (30, 30), (4, 9)], 8, 2, D, 16, dtype, seed=9)
    # no keys, more new tokens than all tokens, no new tokens, and rows past the last sequence
    b["ctx"] = i32([0, 11, 9])
    b["q"] = torch.cat([b["q"], b["q"][:3]])
    out = check(b)
    assert not out[:1].any() and not out[1:20].any() and not out[35:].any() and out[20:35].any()
    b["table"].fill_(-1)  # every page is outside the pool
    assert not call(b).any()


def test_attn_pages_outside():
    b = make([(1, 200), (40, 200)], 8, 2, 128, 16, BF, seed=4)
    for at, page in ((3, -1), (5, 2 ** 31 - 1), (7, b["c"][0].size(0))):
        b["table"][:, at] = page
    check(b)


def test_attn_descending():
    b = make([(3, 50), (30, 30), (4, 9)], 8, 2, 64, 16, BF, seed=9)
    b["cu"] = i32([0, 33, 3, 37])
    assert not call(b).any()


def poisoned(b, seq, tok, page, head, block):
    """Makes a block of a token's value not a number."""
    p = b["table"][seq, tok // page].item()
    b["c"][3][p, head, tok % page, block] = 255


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 16), (256, 32), (80, 24)])
def test_attn_not_finite(D, page, dtype):
    """A value that is not finite shows in the rows that see it, in its block's
    columns only; a key that is not in the whole row."""
    for q, n in ((1, 90), (3, 70), (40, 200), (200, 200)):
        b = make([(q, n), (min(q, 5), 33)], 8, 2, D, page, dtype, seed=q)
        clean = check(b)
        last = M.blocks(D) - 1
        toks = sorted({n - 1, n - q // 2 - 1, max(n - q, 0), 3})
        for tok, block in zip(toks, [last, 0, last, 0]):
            poisoned(b, 0, tok, page, 1, block)
        out = call(b)
        group = 4
        want = torch.zeros_like(out, dtype=torch.bool)
        for tok, block in zip(toks, [last, 0, last, 0]):
            for r in range(q):
                if n - q + r >= tok:
                    want[r, group:, 32 * block:32 * block + 32] = True
        assert torch.equal(torch.isnan(out), want)
        assert torch.equal(out[~want], clean[~want])
        b = make([(q, n), (min(q, 5), 33)], 8, 2, D, page, dtype, seed=q)
        tok = n - q // 2 - 1
        b["c"][1][b["table"][0, tok // page].item(), 0, tok % page, 0] = 254
        out = call(b)
        want = torch.zeros_like(out, dtype=torch.bool)
        for r in range(q):
            if n - q + r >= tok:
                want[r, :group] = True
        assert torch.equal(torch.isnan(out), want)
        assert torch.equal(out[~want], clean[~want])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attn_query_not_finite(dtype):
    for q, n in ((1, 90), (40, 200)):
        b = make([(q, n)], 8, 2, 128, 16, dtype, seed=q)
        clean = call(b)
        b["q"][0, 3, 17], b["q"][q - 1, 6, 100] = math.nan, math.inf
        out = call(b)
        want = torch.zeros_like(out, dtype=torch.bool)
        want[0, 3] = want[q - 1, 6] = True
        assert torch.isnan(out[want]).all() and torch.equal(out[~want], clean[~want])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("q,n", [(1, 300), (40, 300)])
def test_attn_huge_scores(q, n, dtype):
    """One key of each row wins by far; its value comes out as it is held."""
    b = make([(q, n)], 4, 2, 64, 16, dtype, seed=1)
    out = call(b, scale=1e30)
    assert torch.isfinite(out).all()
    k, v = M.values(*b["c"][:2], 64), M.values(*b["c"][2:], 64)
    tok = torch.arange(n, device=DEV)
    page, off = b["table"][0].long()[tok // 16], tok % 16
    for h in range(4):
        s = b["q"][:, h].double() @ k[page, h // 2, off].t()
        s = s.masked_fill(tok[None] > torch.arange(n - q, n, device=DEV)[:, None], -math.inf)
        best = s.topk(2, dim=1)
        # where the second is not within fp32's roundings of the first
        far = best.values[:, 0] - best.values[:, 1] > 1e-4 * best.values[:, 0].abs()
        assert torch.equal(out[:, h].double()[far], v[page, h // 2, off][best.indices[:, 0]][far])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attn_largest_values(dtype):
    """Values of the largest scale keep their size on the way to the outputs."""
    for q, n in ((1, 500), (60, 500)):
        b = make([(q, n)], 8, 2, 64, 16, dtype, seed=3)
        b["c"][2].fill_(0x77), b["c"][3].fill_(252)  # 6 * 2^125 everywhere
        out = call(b).double()
        assert ((out / (6 * 2.0 ** 125) - 1).abs() <= 2 * R.HALF_STEP[dtype] + 600 * R.U32).all()


def test_attn_offsets_past_32_bits():
    """Codes and scales further from the cache's start than 2^32 bytes."""
    page, D = 16, 128
    stride = 1 << 30  # bytes between two pages
    buf = torch.empty(6 * stride, dtype=torch.uint8, device=DEV)
    c = []
    for i, b in enumerate((64, 4, 64, 4)):
        c.append(buf.as_strided((6, 2, page, b), (stride, page * b, b, 1), i * 65536))
    for t, x in zip(c, M.filled(6, 2, page, D, seed=8)):
        t.copy_(x)
    g = torch.Generator().manual_seed(0)
    for q in (1, 90):
        b = dict(q=torch.randn(q, 8, D, generator=g).bfloat16().to(DEV), c=tuple(c), table=i32([[5, 0, 4, 2, 3, 1]]),
                 cu=i32([0, q]), ctx=i32([93]), max_q=q)
        check(b)
    slots = i64([95, 90, 3, 64])
    k, v = ops.zentorch_cache_read_mxfp4(*c, slots, D)
    for i, got in enumerate((k, v)):
        want = M.values(c[2 * i], c[2 * i + 1], D).transpose(1, 2).flatten(0, 1)[slots]
        assert torch.equal(got.double(), want)
    x = torch.randn(4, 2, D, generator=g).bfloat16().to(DEV)
    ops.zentorch_rotary_cache_append_mxfp4(x, x, x, i64([-1] * 4), rope(4, D), slots, *c)
    back = ops.zentorch_cache_read_mxfp4(*c, slots, D)
    want = M.values(*M.quantise(x), D)
    assert torch.equal(back[0].double(), want) and torch.equal(back[1].double(), want)


def test_strided_inputs():
    """Queries and tables of other strides, int32 inputs that are views."""
    b = make([(1, 100), (33, 80)], 8, 2, 64, 16, BF, seed=6)
    plain = call(b)
    wide = torch.zeros(34, 8, 3, 64, dtype=BF, device=DEV)
    wide[:, :, 1] = b["q"]
    b["q"] = wide[:, :, 1]
    odd = torch.zeros(34 * 8 * 64 + 1, dtype=BF, device=DEV)[1:].view(34, 8, 64)
    for name in ("table", "cu", "ctx"):
        t = b[name]
        b[name] = torch.stack([t, t], -1)[..., 0]
    assert torch.equal(call(b), plain)
    odd.copy_(b["q"])
    b["q"] = odd
    assert torch.equal(call(b), plain)
    b["q"] = torch.flip(torch.flip(plain * 0 + wide[:, :, 1], [0]), [0])
    assert torch.equal(call(b), plain)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_side_stream_and_graph(dtype):
    """A step on another stream, captured and replayed with other contents
    between; every replay equals the eager result."""
    def batch(seed):
        b = make([(1, 200), (40, 100), (1, 77)], 8, 2, 128, 16, dtype, seed=seed, poison=False)
        g = torch.Generator().manual_seed(seed)
        x = torch.randn(42, 12, 128, generator=g).to(dtype).to(DEV)
        return b, x

    table = rope(256, 128)
    slots = i64(list(range(0, 42)))
    pos = i64(list(range(42)))

    def step(b, x):
        q = ops.zentorch_rotary_cache_append_mxfp4(x[:, :8], x[:, 8:10], x[:, 10:], pos, table, slots, *b["c"])
        out = ops.zentorch_paged_attention_mxfp4(q, *b["c"], b["table"], b["cu"], b["ctx"], 40)
        return (out, *ops.zentorch_cache_read_mxfp4(*b["c"], slots, 128, dtype=dtype))

    want = []
    for seed in (1, 2, 3):
        b, x = batch(seed)
        want.append([t.clone() for t in step(b, x)])
    torch.cuda.synchronize()
    b, x = batch(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(b, x)
    side.synchronize()
    assert all(torch.equal(a, w) for a, w in zip(got, want[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(b, x)
    for i, seed in enumerate((2, 3, 1, 2)):
        b2, x2 = batch(seed)
        x.copy_(x2)
        for t, y in zip(b["c"], b2["c"]):
            t.copy_(y)
        for name in ("table", "cu", "ctx"):
            b[name].copy_(b2[name])
        graph.replay()
        torch.cuda.synchronize()
        for a, w in zip(got, want[seed - 1]):
            assert torch.equal(a, w)
        junk = torch.randn(1 << 20, device=DEV).sum().item()  # work of its own between the replays
        assert math.isfinite(junk)


def test_pages_move_with_their_scales():
    """Fork, compact and page copies serve codes and scales as any cache."""
    c = M.filled(8, 2, 16, 64, seed=5)
    before = [t.clone() for t in c]
    copies = i32([[1, 6], [-1, -1], [3, 0]])
    for t in (c[0::2], c[1::2]):
        ops.zentorch_cache_copy_pages(list(t), copies)
    for t, w in zip(c, before):
        w[6], w[0] = w[1].clone(), w[3].clone()
        assert torch.equal(t, w)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_served_batch(dtype):
    """Steps as a program makes them: pages for the new tokens, their keys and
    values written, attention over them, a fork, pages gathered; what the cache
    holds is followed token by token, and every step's attention checked."""
    H, KV, D, size, pages, W = 8, 2, 80, 16, 40, 8
    r = random.Random(3)
    table = torch.full((4, W), -1, dtype=torch.int32, device=DEV)
    lens, refs = i32([0] * 4), i32([0] * pages)
    c = M.cache(pages, KV, size, D, fill=255)
    held = [[] for _ in range(4)]  # per sequence, its tokens' (key, value)
    cos_sin = rope(W * size, D)
    for step, new in enumerate(((37, 5, 64, 18), (1, 1, 1, 1), (3, 1, 2, 1), "fork", (1, 1, 1, 1), (20, 2, 1, 7))):
        if new == "fork":
            parents = [0, 0, 2, 0]
            table, lens, refs, copies = ops.zentorch_cache_fork(table, lens, refs, i32(parents), size)
            ops.zentorch_cache_copy_pages([c[0], c[2]], copies)
            ops.zentorch_cache_copy_pages([c[1], c[3]], copies)
            held = [list(held[p]) for p in parents]
            table, refs, copies = ops.zentorch_cache_compact(table, refs)
            ops.zentorch_cache_copy_pages([c[0], c[2]], copies)
            ops.zentorch_cache_copy_pages([c[1], c[3]], copies)
            continue
        T = sum(new)
        cu = i32([sum(new[:i]) for i in range(5)])
        table, lens, refs, pos, slots = ops.zentorch_cache_extend(table, lens, refs, cu, size, T)
        q, k, v = tokens(T, H, KV, D, dtype, seed=10 * step + r.randrange(5))
        k, v, q = (x / x.double().abs().amax(-1, keepdim=True).to(dtype) for x in (k, v, q))
        q = ops.zentorch_rotary_cache_append_mxfp4(q, k, v, pos, cos_sin, slots, *c)
        key, _ = R.rotary(k, pos, cos_sin, False)
        at = 0
        for i, n in enumerate(new):
            held[i] += [(M.values(*M.quantise(key[j]), D), M.values(*M.quantise(v[j].double()), D))
                        for j in range(at, at + n)]
            at += n
        assert lens.tolist() == [len(s) for s in held]
        for i in range(4):
            tok = torch.arange(len(held[i]), device=DEV)
            where = table[i].long()[tok // size] * size + tok % size
            for got, j in zip(ops.zentorch_cache_read_mxfp4(*c, where, D, dtype=dtype), (0, 1)):
                assert torch.equal(got.double(), torch.stack([t[j] for t in held[i]]))
        check(dict(q=q, c=c, table=table, cu=cu, ctx=lens, max_q=max(new)))


def test_many_sequences():
    """As many sequences as a call takes, more items than a round of any loop."""
    r = random.Random(7)
    lens = [(1, r.randint(1, 40)) for _ in range(1024)]
    check(make(lens, 4, 2, 64, 16, BF, seed=7))
    check(make(lens, 2, 1, 256, 8, F32, seed=8))
    lens = [(r.randint(1, 30), 30) for _ in range(1023)] + [(400, 700)]
    check(make(lens, 4, 2, 64, 16, BF, seed=9))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows", [16, 17, 32, 33, 48, 49, 64, 65, 80])
def test_attn_around_the_kernels_borders(rows, D, dtype):
    check(make([(rows, 300), (1, 40), (min(rows, 7), 7)], 2, 2, D, 16, dtype, seed=rows))
    check(make([(rows, 150)] * 3, 2, 2, D, 16, dtype, seed=rows + 1), max_q=1)  # too small a value costs time only


def test_whole_items():
    """Fewer items than workgroups, of about one length: none is cut."""
    for n, kv in ((128, 16), (256, 37), (300, 3), (500, 1)):
        check(make([(n, n)] * 3, kv, kv, 64, 16, F32, seed=n), causal=False)
        check(make([(n, n)] * 2, kv, kv, 64, 16, BF, seed=n))


def test_two_streams_at_once():
    """Calls of different sizes on two streams, with nothing between them."""
    bs = [make([(1, 3000), (1, 77)], 8, 2, 128, 16, BF, seed=1), make([(300, 900)], 8, 2, 256, 16, BF, seed=2)]
    want = [call(b) for b in bs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in bs], [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(call(bs[i]))
    torch.cuda.synchronize()
    for w, out in zip(want, got):
        assert all(torch.equal(x, w) for x in out)


def test_compiled():
    """The in-place op under torch.compile, against eager."""
    x = torch.randn(6, 12, 64, generator=torch.Generator().manual_seed(0)).bfloat16().to(DEV)
    table, slots, pos = rope(64, 64), i64([3, 40, 7, -1, 9, 20]), i64([0, 5, 9, 3, 1, 2])

    def step(x, kc, ks, vc, vs):
        q = ops.zentorch_rotary_cache_append_mxfp4(x[:, :8], x[:, 8:10], x[:, 10:], pos, table, slots, kc, ks, vc, vs)
        k, v = ops.zentorch_cache_read_mxfp4(kc, ks, vc, vs, slots, 64)
        return q * 2, k, v

    a, b = M.cache(4, 2, 16, 64, fill=3), M.cache(4, 2, 16, 64, fill=3)
    want = step(x, *a)
    got = torch.compile(step, backend="aot_eager", fullgraph=True)(x, *b)
    assert all(torch.equal(y, w) for y, w in zip((*got, *b), (*want, *a)))


def refused(word, f, *args, **kw):
    with pytest.raises(RuntimeError) as e:
        f(*args, **kw)
    assert word in str(e.value), str(e.value)


def test_refusals():
    kc, ks, vc, vs = M.filled(4, 2, 16, 64)
    x = torch.randn(3, 2, 64, device=DEV).bfloat16()
    q = torch.randn(3, 4, 64, device=DEV).bfloat16()
    pos, table = i64([0, 1, 2]), rope(8, 64)
    append, read, attn = (ops.zentorch_rotary_cache_append_mxfp4, ops.zentorch_cache_read_mxfp4,
                          ops.zentorch_paged_attention_mxfp4)
    rest = (i32([[0, 1, 2, 3]]), i32([0, 3]), i32([20]), 3)
    for c, word in (((kc.to(torch.int8), ks, vc, vs), "uint8"), ((kc, ks.float(), vc, vs), "uint8"),
                    ((kc[..., :16], ks, vc, vs), "32 bytes a row"), ((kc, ks[..., :1], vc, vs), "2 bytes a row"),
                    ((kc, ks, vc[:3], vs), "pages"), ((kc, ks, vc, vs[:, :1]), "pages"), ((kc[0], ks, vc, vs), "must be"),
                    ((kc.cpu(), ks, vc, vs), "GPU"), ((kc.transpose(2, 3).contiguous().transpose(2, 3), ks, vc, vs), "dense")):
        refused(word, attn, q, *c, *rest)
        refused(word, read, *c, pos, 64)
        refused(word, append, q, x, x, pos, table, pos, *c)
    odd = torch.zeros(4 * 2 * 16 * 32 + 8, dtype=torch.uint8, device=DEV)[8:].view(4, 2, 16, 32)
    for c in ((odd, ks, vc, vs), (kc, ks, odd, vs)):
        refused("16-byte", attn, q, *c, *rest)
        refused("16-byte", read, *c, pos, 64)
    good = kc, ks, vc, vs
    refused("bytes a row", attn, torch.randn(3, 4, 96, device=DEV), *good, *rest)
    refused("multiple of 8", read, *good, pos, 60)
    refused("positive", read, *good, pos, 0)
    refused("bfloat16 or float32", attn, q.half(), *good, *rest)
    refused("multiple of the cache's", attn, q[:, :3], *good, *rest)
    refused("window", attn, q, *good, *rest, causal=False, window=4)
    refused("int32", attn, q, *good, rest[0].long(), *rest[1:])
    refused("cu_seqlens", attn, q, *good, rest[0], i32([0, 1, 3]), *rest[2:])
    refused("dtype", read, *good, pos, 64, dtype=torch.float16)
    refused("int64", read, *good, pos.int(), 64)
    refused("one type", append, q, x.float(), x.float(), pos, table, pos, *good)
    refused("key and value", append, q, x[:2], x[:2], pos, table, pos, *good)
    refused("int64", append, q, x, x, pos[:2], table, pos, *good)
    refused("float32", append, q, x, x, pos, table.double(), pos, *good)
    refused("single memory location", append, q, x, x, pos, table, pos, kc, ks, kc, vs)
    refused("unsupported operation", append, q, x, x, pos, table, pos, kc[:1].expand(4, 2, 16, 32), ks, vc, vs)


def test_near_cache_past_2_to_the_31():
    """Keys and values laid out alike, their pages 2.5 GB from first to last."""
    page, D, pages, stride = 16, 128, 300, 1 << 23
    buf = torch.empty(pages * stride, dtype=torch.uint8, device=DEV)
    c = [buf.as_strided((pages, 2, page, b), (stride, page * b, b, 1), at)
         for b, at in ((64, 0), (4, 65536), (64, 131072), (4, 196608))]
    for t, x in zip(c, M.filled(pages, 2, page, D, seed=4)):
        t.copy_(x)
    g = torch.Generator().manual_seed(0)
    r = random.Random(1)
    for q in (1, 90):
        b = dict(q=torch.randn(2 * q, 8, D, generator=g).bfloat16().to(DEV), c=tuple(c),
                 table=i32([r.sample(range(256, 300), 8), r.sample(range(300), 7) + [299]]), cu=i32([0, q, 2 * q]),
                 ctx=i32([120, 128]), max_q=q)
        check(b)
        b["q"] = b["q"].float()
        check(b)


def test_slots_past_2_to_the_31():
    """Every page is the same memory here, which reading allows."""
    kc, ks, vc, vs = M.filled(1, 2, 4096, 32, seed=2)
    c = [t.expand(1 << 20, -1, -1, -1) for t in (kc, ks, vc, vs)]
    slots = i64([((1 << 20) - 1) * 4096 + 5, (1 << 31) - 1, 1 << 31, (1 << 32) - 1, 1 << 32, 7])
    for got, (codes, scales) in zip(ops.zentorch_cache_read_mxfp4(*c, slots, 32), ((kc, ks), (vc, vs))):
        want = M.values(codes, scales, 32)[0].transpose(0, 1)[slots % 4096]
        want[4] = 0  # past the pool
        assert torch.equal(got.double(), want)
