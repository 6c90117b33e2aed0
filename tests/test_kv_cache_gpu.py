"""GPU parity of the paged-cache ops against plain references (kv_ref.py):
attention and rotary positions in float64 within a bound derived there, the
page upkeep exactly."""
import math
import random

import pytest
import torch

import kv_ref as R
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


def make(lens, H, KV, D, page, dtype, seed=0, spare=3, width=None, layout="hnd", poison=True):
    """A batch of (new, all) tokens over scattered pages.  What no sequence
    holds is NaN (and inf), so that a kernel that reads it shows it."""
    g = torch.Generator().manual_seed(seed)
    r = random.Random(seed)
    counts = [-(-n // page) for _, n in lens]
    pool = sum(counts) + spare
    ids = r.sample(range(pool), sum(counts))
    width = width or max(counts + [1]) + 1
    rows, at = [], 0
    for c in counts:
        rows.append(ids[at:at + c] + [r.choice([-1, pool, 2 ** 31 - 1])] * (width - c))
        at += c
    cu = [0]
    for q, _ in lens:
        cu.append(cu[-1] + q)
    q = (torch.randn(cu[-1], H, D, generator=g) * (torch.rand(H, 1, generator=g) * 2 + 0.5)).to(dtype)
    k = torch.randn(pool, KV, page, D, generator=g)
    v = torch.randn(pool, KV, page, D, generator=g)
    if poison:
        held = torch.zeros(pool, page, dtype=torch.bool)
        for i, (_, n) in enumerate(lens):
            for j in range(n):
                held[rows[i][j // page], j % page] = True
        bad = ~held[:, None, :, None].expand_as(k)
        k[bad], v[bad] = math.nan, math.inf
    k, v = k.to(dtype), v.to(dtype)
    if layout == "pair":   # keys and values of a page beside each other
        both = torch.stack([k, v], 1).to(DEV)
        k, v = both[:, 0], both[:, 1]
    elif layout == "nhd":  # a page's tokens outermost
        k = k.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
        v = v.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    return dict(q=q.to(DEV), k=k.to(DEV), v=v.to(DEV), table=i32(rows), cu=i32(cu),
                ctx=i32([n for _, n in lens]), max_q=max([q for q, _ in lens] + [0]))


def call(b, **kw):
    return ops.zentorch_paged_attention(b["q"], b["k"], b["v"], b["table"], b["cu"], b["ctx"],
                                        kw.pop("max_q", b["max_q"]), **kw)


def check(b, out=None, **kw):
    out = call(b, **kw) if out is None else out
    torch.cuda.synchronize()
    kw.pop("max_q", None)
    ref, bound = R.attention(b["q"], b["k"], b["v"], b["table"], b["cu"], b["ctx"], **kw)
    assert out.shape == b["q"].shape and out.dtype == b["q"].dtype
    err = (out.double() - ref).abs()
    assert torch.isfinite(out).all(), "not finite"
    assert (err <= bound).all(), f"off by {(err - bound).max().item()} over a bound of {bound.max().item()}"
    return out


HEADS = [(8, 2), (4, 4), (7, 1), (16, 2), (6, 2), (24, 2)]


# -------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [8, 64, 72, 80, 96, 128, 200, 256])
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
        check(make([(q, 6007)], 8, 2, 64, 16, F32, seed=q))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("q", [1, 64])
def test_attn_empty_rows(q, dtype):
    """Sequences without context, with no new tokens, with more new tokens
    than context (the first ones stand before position 0 and see nothing),
    and rows of no sequence: zeros."""
    b = make([(q, 70), (q, 0), (0, 33), (q, 64), (0, 0)], 8, 2, 64, 16, dtype, seed=1)
    b["ctx"][3] = max(q // 2, 0) if q > 1 else 0
    pad = torch.full((5, 8, 64), math.nan, dtype=dtype, device=DEV)
    b["q"] = torch.cat([b["q"], pad])
    out = call(b)
    torch.cuda.synchronize()
    assert torch.equal(out[-5:], torch.zeros_like(out[-5:]))
    ref, bound = R.attention(b["q"], b["k"], b["v"], b["table"], b["cu"], b["ctx"])
    assert ((out.double() - ref).abs() <= bound)[:-5].all()
    assert out[q:2 * q].eq(0).all()
    check(make([(0, 20), (0, 0)], 8, 2, 64, 16, dtype))
    check(make([(q, 0), (q, 0)], 8, 2, 64, 16, dtype))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("q", [1, 3, 90])
def test_attn_bad_pages(q, dtype):
    """Pages outside the pool are not seen, whole rows of them among them."""
    b = make([(q, 200), (q, 190), (q, 100)], 8, 2, 64, 16, dtype, seed=3)
    b["table"][0, 3], b["table"][0, 12], b["table"][1, 0] = -1, b["k"].size(0), -(2 ** 31)
    b["table"][2, :] = -5
    out = check(b)
    assert out[2 * q:].eq(0).all()
    check(b, causal=False)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("q,window", [(4, 0), (4, 3), (7, 0), (40, 0), (40, 9), (200, 0), (200, 70)])
def test_attn_values_that_are_not_finite(q, window, D, dtype):
    """Keys and values of some of the chunk's own tokens are NaN or infinite:
    the rows that see none of them keep every bit, the others show it."""
    lens = [(q, 300), (min(q, 9), 9)]
    clean, b = (make(lens, 8, 2, D, 16, dtype, seed=D) for _ in "ab")
    want = check(clean, window=window)
    bad = {299, 300 - q // 2, 300 - q + 1}

    def put(cache, value, tokens):
        for p in tokens:
            cache[b["table"][0, p // 16], :, p % 16] = value

    put(b["v"], math.inf, {299})
    put(b["v"], math.nan, bad - {299})
    put(b["k"], math.nan, {299})
    out = call(b, window=window)
    pos = torch.arange(300 - q, 300, device=DEV)
    sees = torch.zeros(q, dtype=torch.bool, device=DEV)
    for p in bad:
        sees |= (pos >= p) & ((pos - p < window) if window else True)
    assert sees.any() and not sees.all()
    assert torch.equal(out[:q][~sees], want[:q][~sees]) and torch.equal(out[q:], want[q:])
    assert not torch.isfinite(out[:q][sees]).any()


def test_attn_no_pool():
    b = make([(1, 0), (3, 0)], 8, 2, 64, 16, BF, spare=0)
    assert b["k"].size(0) == 0
    b["ctx"][:] = 16
    b["table"][:] = 0
    assert call(b).eq(0).all()


@pytest.mark.parametrize("layout", ["pair", "nhd"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_attn_layouts(layout, dtype):
    lens = [(1, 90), (33, 64), (1, 17)]
    a, b = make(lens, 8, 2, 128, 16, dtype, seed=9), make(lens, 8, 2, 128, 16, dtype, seed=9, layout=layout)
    qkv = torch.randn(b["q"].size(0), 12 * 128, device=DEV).to(dtype)
    qkv[:, :8 * 128] = b["q"].flatten(1)
    b["q"] = qkv[:, :8 * 128].view(-1, 8, 128)  # a slice of the fused projection
    assert torch.equal(check(a), check(b))
    odd = torch.empty(b["q"].numel() + 1, dtype=dtype, device=DEV)[1:].view(b["q"].shape)
    odd.copy_(b["q"])
    b["q"] = odd
    b["table"] = torch.cat([b["table"], b["table"]], 1)[:, :b["table"].size(1)]
    assert torch.equal(call(a), call(b))


def test_attn_scale_and_sharp():
    b = make([(1, 500), (130, 300)], 8, 2, 128, 16, BF, seed=2)
    check(b, scale=0.5)
    check(b, scale=0.0)
    check(b, scale=-0.1)
    b["q"] *= 30  # nearly all the weight on one key; scores of thousands
    check(b)


def test_attn_max_query_len_is_a_hint():
    b = make([(1, 90), (150, 300), (2, 2)], 8, 2, 64, 16, BF, seed=2)
    for m in (0, 1, 150, 10 ** 9):
        check(b, max_q=m)


def test_attn_past_32_bits():
    """Elements past 2^32 bytes and 2^31 elements from the cache's start."""
    page, KV, D = 64, 8, 128
    pool = 2 ** 31 // (page * KV * D) + 40
    k = torch.empty(pool, KV, page, D, dtype=BF, device=DEV)
    v = torch.empty_like(k)
    b = make([(1, 500), (20, 300)], 16, KV, D, page, BF, seed=4)
    n = b["k"].size(0)
    k[-n:], v[-n:] = b["k"], b["v"]
    b["table"] = torch.where((b["table"] >= 0) & (b["table"] < n), b["table"] + (pool - n), -1)
    small = check(b | dict(k=k[-n:], v=v[-n:], table=b["table"] - (pool - n)))
    assert torch.equal(call(b | dict(k=k, v=v)), small)


def test_attn_repeats_bit_for_bit():
    b = make([(1, 3000), (40, 3000), (1, 17)], 16, 2, 128, 16, BF, seed=8)
    one = call(b)
    for _ in range(3):
        assert torch.equal(call(b), one)


def test_attn_side_stream():
    b = make([(1, 900), (40, 300)], 16, 2, 128, 16, BF, seed=8)
    one = check(b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        two = call(b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(one, two)


# ------------------------------------------------------------------ rotary
def table_of(length, rot):
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.arange(length, dtype=torch.float64)[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float().to(DEV)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,D,rot", [(1, 1, 64, 64), (7, 3, 128, 128), (33, 5, 80, 32), (4, 2, 96, 48),
                                       (5, 2, 20, 6), (3, 1, 2, 2), (9, 4, 72, 16), (300, 8, 256, 256)])
def test_rotary(T, H, D, rot, interleaved, dtype):
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, H, D, generator=g).to(dtype).to(DEV)
    table = table_of(500, rot)
    pos = torch.randint(0, 500, (T,), generator=g).to(DEV)
    pos[-1] = -1
    y = ops.zentorch_rotary_embedding(x, pos, table, interleaved=interleaved)
    ref, bound = R.rotary(x, pos, table, interleaved)
    assert ((y.double() - ref).abs() <= bound).all()
    assert torch.equal(y[..., rot:], x[..., rot:]) and torch.equal(y[-1], x[-1])
    # slices with strides, unaligned ones among them, give the same bits
    wide = torch.randn(T, H + 1, D + 1, generator=g).to(dtype).to(DEV)
    wide[:, :H, 1:] = x
    assert torch.equal(ops.zentorch_rotary_embedding(wide[:, :H, 1:], pos, table, interleaved=interleaved), y)
    # a position past the table shows
    far = ops.zentorch_rotary_embedding(x, torch.full_like(pos, 500), table, interleaved=interleaved)
    assert far[..., :rot].isnan().all() and torch.equal(far[..., rot:], x[..., rot:])


def test_rotary_refusals():
    x, t = torch.randn(4, 2, 64, device=DEV).bfloat16(), table_of(10, 64)
    pos = torch.zeros(4, dtype=torch.int64, device=DEV)
    for args in ((x.half(), pos, t), (x, pos[:3], t), (x, pos.int(), t), (x, pos, t.bfloat16()),
                 (x, pos, t[:, :63]), (x[..., :32], pos, t), (x[0], pos, t), (x, pos.cpu(), t)):
        with pytest.raises(RuntimeError):
            ops.zentorch_rotary_embedding(*args)
    assert ops.zentorch_rotary_embedding(x[:0], pos[:0], t).shape == (0, 2, 64)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("layout", ["hnd", "pair", "nhd"])
@pytest.mark.parametrize("T,H,KV,D,rot,page", [(1, 4, 2, 64, 64, 16), (37, 8, 2, 128, 128, 16), (50, 7, 1, 80, 32, 24),
                                               (130, 2, 2, 20, 10, 3)])
def test_append(T, H, KV, D, rot, page, layout, dtype):
    g = torch.Generator().manual_seed(T)
    for il in (False, True):
        qkv = torch.randn(T, (H + 2 * KV) * D, generator=g).to(dtype).to(DEV)
        q, k, v = (s.view(T, -1, D) for s in qkv.split([H * D, KV * D, KV * D], 1))
        pool = -(-T // page) + 3
        perm = torch.randperm(pool * page, generator=g)[:T]
        perm[-1:] = -1                # padding
        if T > 2:
            perm[0] = pool * page     # past the cache
        slots = perm.to(DEV)
        pos = torch.randint(0, 400, (T,), generator=g).to(DEV)
        table = table_of(400, rot)
        shape = (pool, KV, page, D)
        if layout == "pair":
            kc, vc = torch.full((pool, 2, KV, page, D), 7.0, dtype=dtype, device=DEV).unbind(1)
        elif layout == "nhd":
            kc, vc = (torch.full((pool, page, KV, D), 7.0, dtype=dtype, device=DEV).transpose(1, 2) for _ in "kv")
        else:
            kc, vc = (torch.full(shape, 7.0, dtype=dtype, device=DEV) for _ in "kv")
        out = ops.zentorch_rotary_cache_append(q, k, v, pos, table, slots, kc, vc, interleaved=il)
        assert torch.equal(out, ops.zentorch_rotary_embedding(q, pos, table, interleaved=il))
        kr = ops.zentorch_rotary_embedding(k, pos, table, interleaved=il)
        ref, bound = R.rotary(k, pos, table, il)
        assert ((kr.double() - ref).abs() <= bound).all()
        wk, wv = (torch.full(shape, 7.0, dtype=dtype, device=DEV) for _ in "kv")
        ok = (slots >= 0) & (slots < pool * page)
        wk[slots[ok] // page, :, slots[ok] % page] = kr[ok]
        wv[slots[ok] // page, :, slots[ok] % page] = v[ok]
        assert torch.equal(kc, wk) and torch.equal(vc, wv)


def test_append_refusals():
    x, k = torch.randn(4, 4, 64, device=DEV), torch.randn(4, 2, 64, device=DEV)
    t, pos = table_of(10, 64), torch.zeros(4, dtype=torch.int64, device=DEV)
    kv = torch.zeros(5, 2, 16, 64, device=DEV)
    f = ops.zentorch_rotary_cache_append
    for args in ((x, k[:3], k, pos, t, pos, kv, kv), (x, k, k[:, :1], pos, t, pos, kv, kv),
                 (x, k, k, pos, t, pos.int(), kv, kv), (x, k.bfloat16(), k, pos, t, pos, kv, kv),
                 (x, k, k, pos, t, pos, kv.bfloat16(), kv), (x, k, k, pos, t, pos, kv, kv[:4]),
                 (x, k, k, pos, t, pos, kv.transpose(2, 3), kv.transpose(2, 3)), (x, k, k, pos, t, pos, kv[0], kv[0])):
        with pytest.raises(RuntimeError):
            f(*args)
    with pytest.raises(RuntimeError, match="16-byte"):
        odd = torch.zeros(5 * 2 * 16 * 64 + 1, device=DEV)[1:].view(5, 2, 16, 64)
        ops.zentorch_paged_attention(x, odd, odd, i32([[0]]), i32([0, 4]), i32([4]), 4)
    for bad in (dict(window=-1), dict(causal=False, window=2)):
        with pytest.raises(RuntimeError, match="window"):
            ops.zentorch_paged_attention(x, kv, kv, i32([[0]]), i32([0, 4]), i32([4]), 4, **bad)
    for args in ((x, kv, kv, i32([0]), i32([0, 4]), i32([4]), 4), (x, kv, kv, i32([[0]]), i32([0]), i32([4]), 4),
                 (x, kv, kv, i32([[0]]).long(), i32([0, 4]), i32([4]), 4), (x[:, :3], kv, kv, i32([[0]]), i32([0, 4]), i32([4]), 4),
                 (x.bfloat16(), kv, kv, i32([[0]]), i32([0, 4]), i32([4]), 4), (x, kv, kv[..., :32], i32([[0]]), i32([0, 4]), i32([4]), 4)):
        with pytest.raises(RuntimeError):
            ops.zentorch_paged_attention(*args)


# ------------------------------------------------------------------- pages
def pages_of(lens, page, spare, width, seed):
    r = random.Random(seed)
    counts = [-(-n // page) for n in lens]
    pool = sum(counts) + spare
    ids = r.sample(range(pool), sum(counts))
    rows, refs, at = [], [0] * pool, 0
    for c in counts:
        rows.append(ids[at:at + c] + [-1] * (width - c))
        at += c
    for p in ids:
        refs[p] = 1
    return rows, refs


@pytest.mark.parametrize("S,new,ctx,page,spare", [
    (1, 1, 0, 16, 1), (1, 1, 16, 16, 1), (5, 1, 100, 16, 9), (64, 1, 900, 16, 80), (33, 40, 90, 8, 400),
    (9, 300, 500, 24, 60),     # the free pages do not suffice for all
    (4, 3, 10, 1, 5), (700, 1, 60, 16, 300), (3, 0, 30, 16, 0), (2, 1, 31, 16, 0)])
def test_extend(S, new, ctx, page, spare):
    r = random.Random(S + new)
    lens = [r.randint(0, ctx) for _ in range(S)]
    news = [r.randint(0, new) if new > 1 else new for _ in range(S)]
    width = max(-(-(n + k) // page) for n, k in zip(lens, news)) + 1
    if S == 9:
        width -= 3  # and some rows do not fit their table
        lens = [min(n, width * page) for n in lens]
    rows, refs = pages_of(lens, page, spare, width, S)
    cu = [0]
    for k in news:
        cu.append(cu[-1] + k)
    T = cu[-1] + 3
    got = ops.zentorch_cache_extend(i32(rows).view(S, width), i32(lens), i32(refs), i32(cu), page, T)
    want = R.extend(rows, lens, refs, cu, page, T)
    assert [t.tolist() for t in got] == [list(w) for w in want]


def test_extend_large_pool():
    lens = [5000 + i for i in range(40)]
    rows, refs = pages_of(lens, 8, 30000, 700, 1)
    cu = [16 * i for i in range(41)]
    got = ops.zentorch_cache_extend(i32(rows), i32(lens), i32(refs), i32(cu), 8, cu[-1])
    want = R.extend(rows, lens, refs, cu, 8, cu[-1])
    assert [t.tolist() for t in got] == [list(w) for w in want]


@pytest.mark.parametrize("S,ctx,page,spare", [(1, 5, 16, 1), (2, 40, 16, 2), (16, 100, 16, 16), (64, 700, 16, 70),
                                              (50, 90, 24, 3), (256, 300, 8, 260), (8, 64, 1, 0), (1200, 20, 4, 700)])
@pytest.mark.parametrize("kind", ["mixed", "one", "none", "same"])
def test_fork(S, ctx, page, spare, kind):
    r = random.Random(S + page)
    lens = [r.randint(0, ctx) for _ in range(S)]
    width = -(-ctx // page) + 1
    rows, refs = pages_of(lens, page, spare, width, S)
    par = {"mixed": [r.choice([i, -1, r.randrange(S), r.randrange(S)]) for i in range(S)], "one": [S - 1] * S,
           "none": [-1] * S, "same": list(range(S))}[kind]
    for _ in range(2):  # the second step starts from shared pages
        got = ops.zentorch_cache_fork(i32(rows), i32(lens), i32(refs), i32(par), page)
        want = R.fork(rows, lens, refs, par, page)
        assert [t.tolist() for t in got] == [list(w) for w in want]
        rows, lens, refs = want[:3]
        par = [r.choice([i, -1, r.randrange(S), S, 2 ** 31 - 1]) for i in range(S)]


def test_pages_bad_ids():
    """Holes and ids outside the pool in a table are passed on and counted nowhere."""
    rows, lens, refs = [[-1, 99, 2], [3, 4, -7]], [40, 33], [0, 0, 1, 1, 1, 0]
    got = ops.zentorch_cache_extend(i32(rows), i32(lens), i32(refs), i32([0, 2, 5]), 16, 5)
    want = R.extend(rows, lens, refs, [0, 2, 5], 16, 5)
    assert [t.tolist() for t in got] == [list(w) for w in want]
    got = ops.zentorch_cache_fork(i32(rows), i32(lens), i32(refs), i32([1, 1]), 16)
    want = R.fork(rows, lens, refs, [1, 1], 16)
    assert [t.tolist() for t in got] == [list(w) for w in want]
    got = ops.zentorch_cache_compact(i32(rows), i32(refs))
    want = R.compact(rows, refs)
    assert [t.tolist() for t in got] == [list(w) for w in want]


@pytest.mark.parametrize("pages,share", [(1, 1.0), (2, 0.5), (7, 0.4), (64, 0.0), (64, 1.0), (1000, 0.5), (5001, 0.9), (4096, 0.1)])
def test_compact(pages, share):
    r = random.Random(pages)
    used = sorted(r.sample(range(pages), int(pages * share)))
    refs = [0] * pages
    for p in used:
        refs[p] = r.randint(1, 3)
    rows = [[r.choice(used + [-1]) for _ in range(9)] for _ in range(5)]
    got = ops.zentorch_cache_compact(i32(rows), i32(refs))
    want = R.compact(rows, refs)
    assert [t.tolist() for t in got] == [list(w) for w in want]


@pytest.mark.parametrize("dtype", [BF, F32, torch.int8])
@pytest.mark.parametrize("layers,shape", [(1, (9, 2, 16, 64)), (3, (9, 2, 2, 24, 80)), (70, (5, 1, 3, 5)),
                                          (2, (6, 33000))])
def test_copy_pages(layers, shape, dtype):
    caches = [torch.randint(-99, 99, shape, device=DEV).to(dtype) for _ in range(layers)]
    want = [c.clone() for c in caches]
    pairs = [[0, 1], [-1, -1], [0, 4], [2, 3], [3, shape[0]], [-1, 2], [2 ** 31 - 1, 0]]
    for w in want:
        w[1], w[4], w[3] = w[0].clone(), w[0].clone(), w[2].clone()
    ops.zentorch_cache_copy_pages(caches, i32(pairs))
    assert all(torch.equal(a, b) for a, b in zip(caches, want))
    # the keys of pairs that lie beside their values
    both = torch.randn(5, 2, 3, 4, 8, device=DEV)
    kept = both.clone()
    kept[4, 0] = both[1, 0]
    ops.zentorch_cache_copy_pages([both[:, 0]], i32([[1, 4]]))
    assert torch.equal(both, kept)


def test_page_op_refusals():
    c = torch.zeros(4, 2, 3, 8, device=DEV)
    for caches, pairs in (([c], i32([[0, 1, 2]])), ([c], i32([0, 1])), ([c, c[:3]], i32([[0, 1]])), ([c.cpu()], i32([[0, 1]])),
                          ([c[:, :, :, ::2]], i32([[0, 1]])), ([c], i32([[0, 1]]).long())):
        with pytest.raises(RuntimeError):
            ops.zentorch_cache_copy_pages(caches, pairs)
    t, n, cu = i32([[0, 1]]), i32([3]), i32([0, 1])
    for args in ((t, n, n, cu, 0, 1), (t, n, n, cu, 16, -1), (t, n, n, n, 16, 1), (t[0], n, n, cu, 16, 1), (t, n.long(), n, cu, 16, 1)):
        with pytest.raises(RuntimeError):
            ops.zentorch_cache_extend(*args)
    for args in ((t, n, n, n, 0), (t, n, n, cu, 16), (t, n, n, n.long(), 16)):
        with pytest.raises(RuntimeError):
            ops.zentorch_cache_fork(*args)
    with pytest.raises(RuntimeError):
        ops.zentorch_cache_compact(t.long(), n)


def test_ops_in_a_graph():
    """A decode step (extend, append, attend, fork, copy, compact) captured
    once; each replay works on what its inputs then hold."""
    torch.manual_seed(0)
    S, H, KV, D, page, pool, width = 6, 8, 2, 64, 16, 90, 12
    kc, vc = (torch.zeros(pool, KV, page, D, device=DEV, dtype=BF) for _ in "kv")
    table_in, cos_sin = torch.full((S, width), -1, dtype=torch.int32, device=DEV), table_of(width * page, D)
    ctx_in, refs_in = torch.zeros(S, dtype=torch.int32, device=DEV), torch.zeros(pool, dtype=torch.int32, device=DEV)
    par, cu = torch.arange(S, dtype=torch.int32, device=DEV), torch.arange(S + 1, dtype=torch.int32, device=DEV)
    x = torch.zeros(S, (H + 2 * KV) * D, device=DEV, dtype=BF)

    def step(kc, vc):
        q, k, v = (s.view(S, -1, D) for s in x.split([H * D, KV * D, KV * D], 1))
        table, ctx, refs, copies = ops.zentorch_cache_fork(table_in, ctx_in, refs_in, par, page)
        ops.zentorch_cache_copy_pages([kc, vc], copies)
        table, refs, copies = ops.zentorch_cache_compact(table, refs)
        ops.zentorch_cache_copy_pages([kc, vc], copies)
        table, ctx, refs, pos, slots = ops.zentorch_cache_extend(table, ctx, refs, cu, page, S)
        q = ops.zentorch_rotary_cache_append(q, k, v, pos, cos_sin, slots, kc, vc)
        return ops.zentorch_paged_attention(q, kc, vc, table, cu, ctx, 1), table, ctx, refs

    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step(kc.clone(), vc.clone())
    torch.cuda.current_stream().wait_stream(warm)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(kc, vc)
    kc.zero_(), vc.zero_()
    ek, ev = kc.clone(), vc.clone()
    r = random.Random(1)
    for i in range(40):
        x.copy_(torch.randn_like(x))
        par.copy_(i32([r.choice([j, j, r.randrange(S)]) for j in range(S)]))
        want = step(ek, ev)  # eager, on caches of its own
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i
        assert torch.equal(kc, ek) and torch.equal(vc, ev), i
        table_in.copy_(out[1]), ctx_in.copy_(out[2]), refs_in.copy_(out[3])
