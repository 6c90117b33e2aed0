"""Batches past one round of the kernels' loops over sequences, items and rows
(256 or 512 of the attention's, 1024 of the page ops'), up to the most that
the calls take."""
import random

import pytest
import torch

import kv_ref as R
import zentorch  # noqa: F401
from test_kv_cache_gpu import BF, F32, call, check, i32, make, pages_of

pytestmark = pytest.mark.gpu
ops = torch.ops.zentorch


@pytest.fixture(autouse=True)
def _announce(request):
    print(f"\n[case] {request.node.name}", flush=True)


def lengths(S, most, seed):
    """Short sequences, some without context, some without new tokens, and one
    long one far behind, which several workgroups share."""
    r = random.Random(seed)
    out = []
    for i in range(S):
        n = 0 if r.random() < 0.05 else r.randint(1, 40)
        out.append((0 if r.random() < 0.05 else min(n, r.randint(1, most)), n))
    out[S * 3 // 4] = (most, 3000)
    return out


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("most", [1, 40])
@pytest.mark.parametrize("S,D", [(257, 128), (600, 64), (600, 256), (1024, 128), (1024, 256)])
def test_attn_many_sequences(S, D, most, dtype):
    check(make(lengths(S, most, S + D), 4, 1, D, 16, dtype, seed=S))


@pytest.mark.parametrize("dtype,D", [(BF, 64), (F32, 64), (F32, 128)])
def test_attn_many_items_of_few_sequences(dtype, D):
    """Far more tiles than a round of them, with a window, so that the tiles
    are of like cost and the spans begin in every round."""
    check(make([(5000, 5000), (3, 70), (900, 5000)], 8, 1, D, 16, dtype, seed=D), window=50)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("rows", [16, 17, 32, 33, 40, 48, 49, 64, 65, 80])
def test_attn_tens_of_rows(rows, D, dtype):
    """Chunks around the borders between the kernels for few and for many rows."""
    check(make([(rows, 300), (rows, rows), (1, 90)], 2, 2, D, 16, dtype, seed=rows))
    check(make([(-(-rows // 4), 700)], 8, 2, D, 16, dtype, seed=rows + D), window=333)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D,q", [(64, 1), (64, 40), (128, 40), (256, 40)])
@pytest.mark.parametrize("S", [4, 300])
def test_attn_cu_seqlens_that_descend(S, D, q, dtype):
    """Sequences that would overlap: every row is zero.  Ends outside the batch
    are held to it."""
    b = make([(q, 50)] * S, 4, 1, D, 16, dtype, seed=S)
    good = check(b)
    cu = b["cu"].clone()
    b["cu"][-1], b["cu"][0] = 2 ** 31 - 1, -5
    assert torch.equal(call(b), good)
    for at, value in ((1, 3 * q), (S - 1, 0), (S, -1), (S // 2, -(2 ** 31))):
        b["cu"] = cu.clone()
        b["cu"][at] = value
        assert call(b).eq(0).all(), (at, value)
    b["cu"] = cu.flip(0).contiguous()
    assert call(b).eq(0).all()


@pytest.mark.parametrize("S", [1025, 4096])
def test_extend_many_sequences(S):
    r = random.Random(S)
    lens = [r.randint(0, 30) for _ in range(S)]
    news = [r.randint(0, 3) for _ in range(S)]
    rows, refs = pages_of(lens, 4, S // 3, 10, S)
    cu = [0]
    for k in news:
        cu.append(cu[-1] + k)
    got = ops.zentorch_cache_extend(i32(rows), i32(lens), i32(refs), i32(cu), 4, cu[-1])
    want = R.extend(rows, lens, refs, cu, 4, cu[-1])
    assert [t.tolist() for t in got] == [list(w) for w in want]
    assert -1 in want[3] and max(want[3]) >= 0  # some are granted, some are not


@pytest.mark.parametrize("S", [1025, 4096])
def test_fork_many_rows(S):
    r = random.Random(S)
    lens = [r.randint(0, 30) for _ in range(S)]
    rows, refs = pages_of(lens, 4, S // 9, 10, S)
    par = [r.choice([i, -1, r.randrange(S), r.randrange(S)]) for i in range(S)]
    got = ops.zentorch_cache_fork(i32(rows), i32(lens), i32(refs), i32(par), 4)
    want = R.fork(rows, lens, refs, par, 4)
    assert [t.tolist() for t in got] == [list(w) for w in want]
