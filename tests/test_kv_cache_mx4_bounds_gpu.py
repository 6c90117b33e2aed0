"""How far the numbers that a cache in 4 bits holds are from those written, as the
header states it: by a fifth of their block's largest, where that is from 3.5 2^-125 on
and below 7 2^125; below that by 2^-126; above it 6 2^125 is the most that is held."""
import pytest
import torch

import mx4_ref as M
import test_kv_cache_mx4_gpu as G

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def held(v):
    """What the cache gives back for values [T, 1, 64]."""
    T = v.size(0)
    c = M.cache(T, 1, 1, 64)
    slots = G.i64(list(range(T)))
    zero = torch.zeros_like(v)
    G.ops.zentorch_rotary_cache_append_mxfp4(zero, zero, v, G.i64([-1] * T), G.rope(4, 64), slots, *c)
    return G.ops.zentorch_cache_read_mxfp4(*c, slots, 64, dtype=F32)[1].double()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_bounds(dtype):
    g = torch.Generator().manual_seed(0)
    T = 4000
    x = torch.rand(T, 1, 64, generator=g) * 2 - 1
    x[:, :, 0::32] = x[:, :, 0::32].sign() * (1 + torch.rand(T, 1, 2, generator=g))
    e = torch.randint(-140, 127, (T, 1, 1), generator=g)
    e[:200], e[200:400] = 127, -126
    v = (x.double() * torch.pow(2.0, e.double())).clamp(-3.38e38, 3.38e38).to(dtype).to(G.DEV)
    y, blocks = held(v), v.double().abs().unflatten(2, (2, 32))
    most = blocks.amax(3, keepdim=True).expand_as(blocks).flatten(2)
    off = (y - v.double()).abs()
    low, top = most < 3.5 * 2.0 ** -125, most >= 7 * 2.0 ** 125
    assert low.any() and top.any() and (~low & ~top).any()
    assert (off[~low & ~top] <= most[~low & ~top] / 5).all()
    assert (off[low] <= 2.0 ** -126).all()
    # up to 6 scales as elsewhere, and from there on 6 of them
    past = v.double().abs() > 6 * 2.0 ** 125
    assert (off[top & ~past] <= 2.0 ** 125).all()
    assert (y[top & past].abs() == 6 * 2.0 ** 125).all() and past.any()


def test_the_ends():
    """A fifth is not enough at the ends: fp32's largest number is held as three
    quarters of it, and the smallest ones as 0."""
    v = torch.zeros(3, 1, 64, device=G.DEV)
    v[0], v[1], v[2] = torch.finfo(F32).max, 2.0 ** -127, 5.0
    y = held(v)
    assert (y[0] == 6 * 2.0 ** 125).all() and (y[1] == 0).all() and (y[2] == 4).all()
