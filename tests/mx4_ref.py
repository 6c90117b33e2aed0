"""Plain references of the cache held in 4 bits, in float64, number by number:
a block's scale by the definition's inequality, a code by its distance."""
import torch

import kv_ref

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def power(e):
    """2^e of whole numbers -140 .. 140, exactly (a GPU's pow is not)."""
    return torch.tensor([2.0 ** i for i in range(-140, 141)], dtype=torch.float64, device=e.device)[e.long() + 140]


def blocks(dim):
    return -(-dim // 32)


def quantise(x):
    """(codes uint8 [..., 16 blocks], scales uint8 [..., blocks]) of rows [..., dim]."""
    d = x.size(-1)
    y = torch.nn.functional.pad(x.double(), (0, -d % 32)).unflatten(-1, (-1, 32)).cpu()
    bad = ~torch.isfinite(y).all(-1)
    y = torch.where(bad[..., None], 0.0, y)
    amax = y.abs().amax(-1)
    e = torch.full(amax.shape, -125)
    for k in range(-125, 125):  # the scale grows while the largest is seven of it and more
        e = torch.where((e == k) & (amax >= 7 * 2.0 ** k), k + 1, e)
    v = y.abs() / power(e)[..., None]
    far = (v[..., None] - torch.tensor(GRID, dtype=torch.float64)).abs()
    # of two equally near codes the even one comes first
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7])
    code = order[far[..., order].argmin(-1)]
    code = (code + 8 * torch.signbit(y)).flatten(-2)
    code = torch.where(bad.repeat_interleave(32, -1), 0, code)
    packed = (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8)
    return packed.to(x.device), torch.where(bad, 255, e + 127).to(torch.uint8).to(x.device)


def values(codes, scales, dim):
    """float64 [..., dim]."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    grid = torch.tensor(GRID, dtype=torch.float64, device=codes.device)
    v = grid[c & 7] * (1 - 2 * (c >> 3)).double()
    s = power(scales.int() - 127)
    s = torch.where(scales > 252, float("nan"), s)
    return (v.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)[..., :dim]


def cache(pages, heads, size, dim, device="cuda", fill=0):
    """(key codes, key scales, value codes, value scales)."""
    nb = blocks(dim)
    return tuple(torch.full((pages, heads, size, b), fill, dtype=torch.uint8, device=device)
                 for b in (16 * nb, nb, 16 * nb, nb))


def filled(pages, heads, size, dim, seed=0, device="cuda"):
    """A cache of random numbers, some of whose blocks are large or small."""
    g = torch.Generator(device=device).manual_seed(seed)
    out = []
    for _ in range(2):
        nb = blocks(dim)
        x = torch.randn(pages, heads, size, nb, 32, generator=g, device=device)
        x = x * torch.exp2(torch.randint(-2, 2, (pages, heads, size, nb, 1), generator=g, device=device).float())
        x = x.flatten(-2)
        x[..., dim:] = 0
        out += quantise_fast(x)
    return tuple(out)


def quantise_fast(x):
    """quantise() of finite rows of whole blocks, on the device."""
    y = x.double().unflatten(-1, (-1, 32))
    m, e = torch.frexp(y.abs().amax(-1).clamp(min=2.0 ** -120))
    e = (e + (m >= 0.875) - 3).clamp(-125, 125)
    v = y.abs() * power(-e)[..., None]
    code = sum(((v > t) if i % 2 == 0 else (v >= t)).int()
               for i, t in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)))
    code = (code + 8 * torch.signbit(y).int()).flatten(-2)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), (e + 127).to(torch.uint8)


def attention(q, c, table, cu, ctx, **kw):
    """(out, bound) as kv_ref.attention's over the cache's numbers.

    Its bound is relative to the weights.  Of the numbers held in 4 bits many are
    0, so that a column may be left with weights e^(s - m) below fp32's range
    alone: weights are held times 2^-16 and may vanish below 2^-126, which is
    2^-110 of the largest one, for each of n keys."""
    k, v = values(c[0], c[1], q.size(2)), values(c[2], c[3], q.size(2))
    out, bound = kv_ref.attention(q, k, v, table, cu, ctx, **kw)
    n = int(ctx.max()) if ctx.numel() else 0
    most = torch.where(torch.isfinite(v), v.abs(), 0).max() if v.numel() else 0
    return out, bound + n * 2.0 ** -110 * most
