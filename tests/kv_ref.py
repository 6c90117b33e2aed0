"""Plain references of the paged-cache ops: attention and rotary positions in
float64, the page upkeep as Python lists, row by row."""
import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
U32 = 2.0 ** -24  # a rounding in fp32


def attention(q, k_cache, v_cache, table, cu, ctx, causal=True, window=0, scale=None):
    """(out, bound), float64 [T, H, D]: the definition, and how far a kernel
    with fp32 scores and sums and probabilities rounded to the operands' type
    may be off.  A key whose page is outside the pool is not seen."""
    T, H, D = q.shape
    pages, KV, size, _ = k_cache.shape
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(T, H, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    cu, ctx, table = cu.tolist(), ctx.tolist(), table.long()
    hs = HALF_STEP[q.dtype]
    for i, n in enumerate(ctx):
        a, b = cu[i], cu[i + 1]
        if b <= a or n <= 0:
            continue
        tok = torch.arange(n, device=q.device)
        page, off = table[i][tok // size], tok % size
        held = (page >= 0) & (page < pages)
        page = page.clamp(0, pages - 1)
        pos = torch.arange(n - (b - a), n, device=q.device)[:, None]
        seen = held[None].expand(b - a, n)
        if causal:
            seen = seen & (tok[None] <= pos)
        if window:
            seen = seen & (tok[None] > pos - window)
        used = seen.any(0)
        for h in range(H):
            kv = h // (H // KV)
            # what no row sees may hold anything
            k = torch.where(used[:, None], k_cache[page, kv, off].double(), 0)
            v = torch.where(used[:, None], v_cache[page, kv, off].double(), 0)
            x = q[a:b, h].double()
            s = torch.where(seen, x @ k.t() * scale, -math.inf)
            m = s.amax(1, keepdim=True)
            e = torch.where(seen, torch.exp(s - torch.where(m == -math.inf, 0, m)), 0)
            p = e / e.sum(1, keepdim=True).clamp(min=1e-300)
            o = p @ v
            # a score's error: D products and sums in fp32, the scaling, and
            # exp's argument and value (a few units)
            ds = (D + 8) * U32 * ((x.abs() @ k.abs().t()) * abs(scale)).amax(1, keepdim=True) + 8 * U32
            weight = 2 * ds + (n + 16) * 2 * U32
            if q.dtype == torch.bfloat16:
                weight = weight + 2 * hs  # the weights of the sum and of its norm
            out[a:b, h] = o
            bound[a:b, h] = hs * o.abs() + (1 + hs) * weight * (p @ v.abs())
    return out, bound


def rotary(x, pos, table, interleaved):
    """(out, bound), float64."""
    R, half = table.size(1), table.size(1) // 2
    y = x.double().clone()
    row = table.double()[pos.clamp(0, table.size(0) - 1)][:, None]
    c, s = row[..., :half], row[..., half:]
    i0 = slice(0, R, 2) if interleaved else slice(0, half)
    i1 = slice(1, R, 2) if interleaved else slice(half, R)
    a, b = y[..., i0].clone(), y[..., i1].clone()
    bound = torch.zeros_like(y)
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    hs = HALF_STEP[x.dtype]
    # two products and a sum in fp32, then the rounding
    bound[..., i0] = 3 * U32 * ((a * c).abs() + (b * s).abs()) * (1 + hs) + hs * y[..., i0].abs()
    bound[..., i1] = 3 * U32 * ((b * c).abs() + (a * s).abs()) * (1 + hs) + hs * y[..., i1].abs()
    pad = (pos < 0)[:, None, None]
    y = torch.where(pad, x.double(), y)
    return torch.where((pos >= table.size(0))[:, None, None] & (torch.arange(x.size(2), device=x.device) < R),
                       math.nan, y), torch.where(pad, 0, bound)


def extend(table, ctx, refs, cu, size, T):
    table, ctx, refs = [list(r) for r in table], list(ctx), list(refs)
    pages, W = len(refs), len(table[0]) if table else 0
    free = [p for p in range(pages) if refs[p] == 0]
    pos, slot, taken, short = [-1] * T, [-1] * T, 0, False
    for i, c in enumerate(list(ctx)):
        n = max(0, cu[i + 1] - cu[i])
        have, want = -(-c // size), -(-(c + n) // size)
        if want > W:
            continue
        taken += want - have
        if short or taken > len(free):
            short = True
            continue
        for col in range(have, want):
            table[i][col] = free[taken - (want - have) + col - have]
            refs[table[i][col]] = 1
        for j in range(n):
            p = c + j
            page = table[i][p // size]
            pos[cu[i] + j] = p
            slot[cu[i] + j] = page * size + p % size if 0 <= page < pages else -1
        ctx[i] = c + n
    return table, ctx, refs, pos, slot


def fork(table, ctx, refs, parents, size):
    S, pages, refs = len(table), len(refs), list(refs)
    W = len(table[0]) if S else 0
    par = [p if 0 <= p < S else -1 for p in parents]
    have = [-(-c // size) for c in ctx]
    ok = lambda p: 0 <= p < pages  # noqa: E731
    for i in range(S):
        n = par.count(i)
        for col in range(have[i]):
            if ok(table[i][col]):
                last = ctx[i] % size != 0 and col == have[i] - 1
                refs[table[i][col]] += (min(n, 1) if last else n) - 1
    free = [p for p in range(pages) if refs[p] == 0]
    seen, out, lens, copies, used = set(), [], [], [], 0
    for p in par:
        row, n, copy = [-1] * W, 0, (-1, -1)
        if p >= 0:
            row[:have[p]], n = table[p][:have[p]], ctx[p]
            if ctx[p] % size and p in seen:
                if used < len(free):
                    src = row[have[p] - 1]
                    copy = (src if ok(src) else -1, free[used])
                    row[have[p] - 1] = free[used]
                    refs[free[used]] += 1
                else:
                    for page in row[:have[p] - 1]:
                        if ok(page):
                            refs[page] -= 1
                    row, n = [-1] * W, 0
                used += 1
            seen.add(p)
        out.append(row)
        lens.append(n)
        copies.append(list(copy))
    return out, lens, refs, copies


def compact(table, refs):
    pages = len(refs)
    used = [p for p in range(pages) if refs[p]]
    n = len(used)
    moves = list(zip([p for p in used if p >= n], [p for p in range(n) if not refs[p]]))
    to = dict(moves)
    new = [refs[p] if p < n else 0 for p in range(pages)]
    for s, d in moves:
        new[d] = refs[s]
    copies = [list(m) for m in moves] + [[-1, -1]] * (pages // 2 - len(moves))
    return [[to.get(p, p) for p in row] for row in table], new, copies
