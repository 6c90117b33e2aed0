"""Attention over the paged cache where queries and keys are not finite, in whole
items and in ones whose keys several workgroups share."""
import math

import pytest
import torch

from test_kv_cache_gpu import BF, F32, call, check, make

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _announce(request):
    print(f"\n[case] {request.node.name}", flush=True)


# (new, all) tokens: few long sequences, whose keys are shared out over dozens
# of workgroups, and many short ones
LONG = {1: [(1, 20011), (1, 9973)], 4: [(4, 6007)], 40: [(40, 9973), (1, 70)], 150: [(150, 6007), (150, 700)]}
KINDS = [(1, False), (1, True), (4, True), (40, False), (40, True), (150, True)]


def lens_of(q, long):
    return LONG[q] if long else [(q, 60 + i % 7) for i in range(90)]


def put(cache, b, seq, tokens, value, column=slice(None)):
    page = cache.size(2)
    for t in tokens:
        cache[b["table"][seq, t // page], :, t % page, column] = value


def same_but(out, want, rows):
    """Every row but those of the mask `rows` has the bits of `want`."""
    return torch.equal(out[~rows], want[~rows])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("q,long", KINDS)
def test_nan_query(q, long, D, dtype):
    """One NaN in a query head: its row is NaN and no other changes."""
    b = make(lens_of(q, long), 8, 2, D, 64, dtype, seed=q)
    want = check(b) if q * D < 10000 else call(b)
    hit = torch.zeros(want.shape[:2], dtype=torch.bool, device=want.device)
    for t, h in ((0, 3), (want.size(0) - 1, 6)):
        b["q"][t, h, D // 2] = math.nan
        hit[t, h] = True
    out = call(b)
    assert out[hit].isnan().all()
    assert same_but(out, want, hit)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("q,long", KINDS)
@pytest.mark.parametrize("share", ["all", "half"])
def test_nan_keys(share, q, long, D, dtype):
    """All keys of the first sequence are NaN, or those of its first half: its
    rows are NaN, the other sequences' keep every bit."""
    lens = lens_of(q, long)
    b = make(lens, 8, 2, D, 64, dtype, seed=q + 1)
    want = call(b)
    n = lens[0][1] if share == "all" else lens[0][1] // 2
    put(b["k"], b, 0, range(n), math.nan)
    out = call(b)
    hit = torch.zeros(want.size(0), dtype=torch.bool, device=want.device)
    hit[:q] = True
    assert out[:q].isnan().all()
    assert same_but(out, want, hit)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("q,long", KINDS)
def test_rows_do_not_feel_each_other(q, long, D, dtype):
    """A row of far larger scores changes no bit of the rows beside it."""
    b = make(lens_of(q, long), 8, 2, D, 64, dtype, seed=q)
    want = call(b)
    hit = torch.zeros(want.shape[:2], dtype=torch.bool, device=want.device)
    for t, h in ((0, 3), (want.size(0) - 1, 6)):
        b["q"][t, h] *= 64
        hit[t, h] = True
    out = call(b)
    assert same_but(out, want, hit) and not torch.equal(out, want)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("q", [4, 12, 40, 200])
def test_keys_of_infinity(q, D, dtype):
    """A key whose score is +inf makes the rows that see it NaN."""
    lens = [(q, 300), (min(q, 9), 9)]
    b = make(lens, 8, 2, D, 16, dtype, seed=D + 2)
    b["q"][..., 5] = b["q"][..., 5].abs() + 0.25
    want = check(b)
    first = 300 - q // 2
    put(b["k"], b, 0, [first], math.inf, 5)
    sees = torch.zeros(want.size(0), dtype=torch.bool, device=want.device)
    sees[first - 300 + q:q] = True
    out = call(b)
    assert out[sees].isnan().all()
    assert same_but(out, want, sees)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("q", [4, 12, 40, 200])
def test_largest_values_unseen(q, D, dtype):
    """The type's largest and lowest finite numbers as values of tokens at the
    chunk's end change no bit of the rows that do not see them."""
    lens = [(q, 300), (min(q, 9), 9)]
    clean, b = (make(lens, 8, 2, D, 16, dtype, seed=D) for _ in "ab")
    want = check(clean)
    top = torch.finfo(dtype).max
    first = 300 - q // 2
    put(b["v"], b, 0, range(first, 300), top, slice(0, D, 2))
    put(b["v"], b, 0, range(first, 300), -top, slice(1, D, 2))
    sees = torch.zeros(want.size(0), dtype=torch.bool, device=want.device)
    sees[first - 300 + q:q] = True
    assert same_but(call(b), want, sees)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("q", [4, 12, 40, 200])
def test_largest_values(q, D, dtype):
    """The type's largest and lowest finite numbers as values of two of the
    chunk's own tokens: rows that do not see them keep every bit, rows that do
    stay finite and within the bound."""
    lens = [(q, 300), (min(q, 9), 9)]
    clean, b = (make(lens, 8, 2, D, 16, dtype, seed=D) for _ in "ab")
    want = check(clean)
    top = torch.finfo(dtype).max
    first = 300 - q // 2
    put(b["v"], b, 0, [first], top, slice(0, D, 2))
    put(b["v"], b, 0, [first], -top, slice(1, D, 2))
    put(b["v"], b, 0, [299], -top, slice(0, D, 3))
    sees = torch.zeros(clean["q"].size(0), dtype=torch.bool, device=want.device)
    sees[first - 300 + q:q] = True
    out = check(b)
    assert sees[:q].any() and not sees[:q].all()
    assert same_but(out, want, sees)
    # no max_query_len makes such a value infinite
    for m in (1, 10 ** 6):
        assert same_but(check(b, max_q=m), call(clean, max_q=m), sees)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("q,long", KINDS)
@pytest.mark.parametrize("size", [1e6, 1e9, 1e12, 1e30, "largest"])
def test_huge_scores(size, q, long, D, dtype):
    """One key's score stands so far above all others that its value is the
    output, bit for bit; a very negative one's weighs nothing."""
    b = make(lens_of(q, long), 8, 2, D, 64, dtype, seed=D + 3)
    # "largest": the key's number is the type's largest, against small queries
    top, by = (torch.finfo(dtype).max, 2.0 ** -20) if size == "largest" else (size, 1)
    b["q"][..., 5] = (b["q"][..., 5].abs() + 0.25) * by
    clean = call(b)
    n, t = lens_of(q, long)[0][1], lens_of(q, long)[0][1] - q
    put(b["k"], b, 0, [t], top, 5)
    out = call(b)
    v = b["v"][b["table"][0, t // 64], :, t % 64].repeat_interleave(4, 0)
    assert torch.equal(out[:q], v.expand_as(out[:q]))
    assert torch.equal(out[q:], clean[q:])
    if long:  # a page of very negative ones, against a cache without that page
        b["k"][b["table"][0, t // 64], :, t % 64, 5] = 0
        put(b["k"], b, 0, range(192, 256), -top, 5)
        out = call(b)
        table = b["table"].clone()
        table[0, 3] = -1
        check(b | dict(table=table), out)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("q,long", KINDS)
def test_small_values(q, long, D, dtype):
    """Values of 2^-100 and less come out as accurate as others."""
    b = make(lens_of(q, long)[:3], 8, 2, D, 64, dtype, seed=D + 5, poison=False)
    b["v"] = b["v"] * 2.0 ** -100
    check(b)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("q", [1, 4, 12, 40, 200])
@pytest.mark.parametrize("all_", [300, 5000])
def test_keys_of_minus_infinity(all_, q, D, dtype):
    """Keys whose scores are -inf weigh nothing: the outputs are those of a
    cache without their pages."""
    lens = [(q, all_), (min(q, 9), 9)]
    b = make(lens, 8, 2, D, 16, dtype, seed=D + 1)
    b["q"][..., 5] = b["q"][..., 5].abs() + 0.25
    gone = [2, 3, 17]
    for p in gone:
        put(b["k"], b, 0, range(16 * p, 16 * p + 16), -math.inf, 5)
    out = call(b)
    table = b["table"].clone()
    table[0, gone] = -1
    check(b | dict(table=table), out)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("q,n,window", [(1, 300, 0), (4, 300, 0), (7, 300, 3), (12, 300, 0), (40, 300, 0), (40, 300, 9),
                                        (200, 300, 70), (150, 6007, 0), (4, 6007, 2000)])
def test_values_that_are_not_finite_by_column(q, n, window, D, dtype):
    """NaN and infinities in some columns of some values: those columns of the
    rows that see them are not finite, wherever they lie; every other output
    keeps its bits."""
    lens = [(q, n), (min(q, 9), 9)]
    clean, b = (make(lens, 8, 2, D, 16, dtype, seed=D + q) for _ in "ab")
    want = call(clean, window=window)
    pos = torch.arange(n - q, n, device=want.device)
    hit = torch.zeros(want.shape, dtype=torch.bool, device=want.device)
    places = [(n - 1, 3, math.inf), (n - q // 2 - 1, 8, math.nan), (n - q // 2 - 1, D - 1, -math.inf),
              (n - q, 9, math.nan), (n - q - 40, 17, math.nan), (100, 18, math.inf), (5, 10, -math.inf)]
    for token, column, value in places:
        put(b["v"], b, 0, [token], value, column)
        sees = (pos >= token) & ((pos - token < window) if window else True)
        hit[:q, :, column] |= sees[:, None]
    out = call(b, window=window)
    assert torch.equal(out[~hit], want[~hit])
    assert not torch.isfinite(out[hit]).any()
