"""Performance cases of the cache path around the quantised linears: rotary
positions, attention of a chunk of new tokens over a paged cache, and the
upkeep of that cache's pages.

A cache of one layer is a pair of tensors ``[pages, kv_heads, page_size, head_dim]``
(or one with a dimension of two after the pages, of which the pair are views).
Sequence i's tokens lie in the pages that row i of ``block_table`` names, in
order; ``context_lens[i]`` counts them, the new ones included, and the new
ones of sequence i are rows ``cu_seqlens[i] .. cu_seqlens[i + 1]`` of the batch.

The kinds of cases:

* ``attn``   ``zentorch_paged_attention``, one call of one layer;
* ``append`` ``zentorch_rotary_cache_append``: the rotated query of one layer,
  and its rotated keys and its values written to the cache;
* ``rotary`` ``zentorch_rotary_embedding`` on one tensor;
* ``extend`` ``zentorch_cache_extend``: a step's new tokens get their pages;
* ``fork``   ``zentorch_cache_fork`` and ``zentorch_cache_copy_pages``: a step
  of a search over several continuations, in every layer's cache;
* ``compact`` ``zentorch_cache_compact`` and the copies it asks for.

Where ``own`` is false ``run`` computes them in elementary torch operations.
Lengths and page plans follow from the case, values from the seed.
"""
import math
import random

import torch

own = False
DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _ops():
    import os
    import sys

    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                      "zendnn-pytorch-plugin_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import zentorch  # noqa: F401

    return torch.ops.zentorch


def listed():
    return [
        # One user's decode step over a short conversation: the smallest call,
        # where launches and latency count.
        dict(name="attn_decode_one", kind="attn", plan=1, batch="same", seqs=1, chunk=1, ctx=777,
             heads=32, kv=8, dim=128, page=16, causal=True, window=0, dtype="bf16"),
        # A serving batch's decode step, contexts of every length.
        dict(name="attn_decode_batch", kind="attn", plan=2, batch="ragged", seqs=64, chunk=1,
             ctx=8192, heads=32, kv=8, dim=128, page=16, causal=True, window=0, dtype="bf16"),
        # Two users deep in long documents: few rows, a long axis.
        dict(name="attn_decode_long", kind="attn", plan=3, batch="same", seqs=2, chunk=1,
             ctx=131072, heads=32, kv=8, dim=128, page=64, causal=True, window=0, dtype="bf16"),
        # A chunk of 2048 prompt tokens behind 6144 that are cached already.
        dict(name="attn_chunk", kind="attn", plan=4, batch="same", seqs=1, chunk=2048, ctx=8192,
             heads=32, kv=8, dim=128, page=16, causal=True, window=0, dtype="bf16"),
        # Decoding sequences and odd prompt chunks in one batch, seven heads to
        # a kv head, a sliding window.
        dict(name="attn_mixed", kind="attn", plan=5, batch="mixed", seqs=33, chunk=1001, ctx=4099,
             heads=28, kv=4, dim=128, page=32, causal=True, window=1024, dtype="bf16"),
        # Bidirectional attention of whole float32 sequences, as an encoder's.
        dict(name="attn_fp32", kind="attn", plan=6, batch="whole", seqs=8, chunk=500, ctx=500,
             heads=16, kv=16, dim=64, page=16, causal=False, window=0, dtype="fp32"),
        # A decode step's new tokens into one layer's cache.
        dict(name="append_decode", kind="append", plan=7, tokens=8, pad=1, heads=32, kv=8, dim=128,
             rot=128, page=16, length=131072, interleaved=False, scaling="by_parts",
             dtype="bf16"),
        # A large prompt batch into one layer's cache.
        dict(name="append_prefill", kind="append", plan=8, tokens=8191, pad=0, heads=32, kv=8,
             dim=128, rot=128, page=16, length=32768, interleaved=False, scaling="none",
             dtype="bf16"),
        # Interleaved pairs over part of a float32 head, far positions.
        dict(name="rotary_partial_fp32", kind="rotary", plan=9, tokens=1000, heads=16, dim=80,
             rot=32, length=131072, interleaved=True, scaling="linear", dtype="fp32"),
        # Page allocation of a serving batch's decode step.
        dict(name="pages_extend", kind="extend", plan=10, seqs=64, chunk=1, ctx=8192, page=16),
        # A search step: rows continue, multiply or end, over a model's caches.
        dict(name="pages_fork", kind="fork", plan=11, seqs=64, ctx=2048, page=16, kv=8, dim=128,
             layers=32, dtype="bf16"),
        # A half-empty pool gathered at its front.
        dict(name="pages_compact", kind="compact", plan=12, pages=2048, share=0.5, page=16, kv=8,
             dim=128, layers=8, dtype="bf16"),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(32, 8), (32, 32), (28, 4), (16, 16), (8, 1), (64, 8), (12, 2)]


def draw(rng):
    kind = rng.choice(["attn"] * 6 + ["append"] * 2 + ["rotary", "extend", "fork", "compact"])
    plan = rng.randrange(1 << 30)
    heads, kv = rng.choice(_HEADS)
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    if kind == "attn":
        batch = rng.choice(["same", "ragged", "mixed", "whole", "long"])
        c = dict(kind="attn", plan=plan, batch="same" if batch == "long" else batch, heads=heads,
                 kv=kv, dim=dim, page=page, causal=True, window=0, dtype=dtype)
        if batch == "long":
            c.update(seqs=rng.randrange(1, 4), chunk=_logint(rng, 1, 16),
                     ctx=_logint(rng, 16384, 131072))
        elif batch == "whole":
            n = _logint(rng, 1, 2048)
            c.update(seqs=_logint(rng, 1, 32), chunk=n, ctx=n, causal=rng.random() < 0.5)
        else:
            c.update(seqs=_logint(rng, 1, 128), ctx=_logint(rng, 64, 16384))
            c["chunk"] = 1 if rng.random() < 0.4 else _logint(rng, 2, min(2048, c["ctx"]))
        if c["causal"] and rng.random() < 0.25:
            c["window"] = _logint(rng, 16, 4096)
        while True:
            w = work(c)
            if w["flops"] <= (2.4e11 if dtype == "bf16" else 1.5e10) and w["bytes"] <= 1.0e9:
                return c
            if c["seqs"] > 1:
                c["seqs"] //= 2
            elif c["chunk"] > 1:
                c["chunk"] = (c["chunk"] + 1) // 2
                if c["batch"] == "whole":
                    c["ctx"] = c["chunk"]
            else:
                c["ctx"] //= 2
    if kind in ("append", "rotary"):
        rot = dim if rng.random() < 0.6 else rng.choice([16, 32, 48])
        c = dict(kind=kind, plan=plan, tokens=_logint(rng, 1, 8192), heads=heads, dim=dim, rot=rot,
                 length=_logint(rng, 4096, 131072), interleaved=rng.random() < 0.4,
                 scaling=rng.choice(["none", "linear", "by_parts"]), dtype=dtype)
        if kind == "append":
            c.update(kv=kv, page=page, pad=rng.choice([0, 0, 1, 5]))
        return c
    if kind == "extend":
        return dict(kind="extend", plan=plan, seqs=_logint(rng, 1, 512),
                    chunk=rng.choice([1, 1, 7, 300]), ctx=_logint(rng, 64, 8192), page=page)
    if kind == "fork":
        return dict(kind="fork", plan=plan, seqs=_logint(rng, 2, 256), ctx=_logint(rng, 64, 2048),
                    page=rng.choice([8, 16, 24, 32]), kv=rng.choice([1, 2, 4, 8]),
                    dim=rng.choice([64, 80, 128]), layers=rng.choice([1, 4, 16, 32]), dtype=dtype)
    return dict(kind="compact", plan=plan, pages=_logint(rng, 64, 2048),
                share=rng.uniform(0.05, 0.95), page=rng.choice([8, 16, 24]),
                kv=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 80, 128]),
                layers=rng.choice([1, 3, 8]), dtype="bf16")


# ------------------------------------------------------------------- plans
def _lengths(c):
    """(new tokens, all tokens) of every sequence of an attn or extend case."""
    r = random.Random(c["plan"])
    out = []
    for i in range(c["seqs"]):
        q, n = c["chunk"], c["ctx"]
        batch = c.get("batch", "ragged")
        if batch in ("ragged", "mixed"):
            n = _logint(r, max(1, c["ctx"] // 32), c["ctx"])
        if batch == "ragged":
            q = r.randint(1, c["chunk"])
        elif batch == "mixed":  # mostly decoding, one chunk in eight
            q = r.randint(1, c["chunk"]) if i % 8 == 0 else 1
        elif batch == "whole":
            q = n = r.randint(max(1, c["ctx"] // 2), c["ctx"])
        out.append((min(q, n), n))
    return out


def _pairs(c):
    """Number of (query, key) pairs the masks of an attn case leave."""
    n = 0
    for q, ctx in _lengths(c):
        if not c["causal"]:
            n += q * ctx
            continue
        for p in (range(ctx - q, ctx) if c["window"] else ()):
            n += min(p + 1, c["window"])
        if not c["window"]:
            n += q * (ctx - q) + q * (q + 1) // 2
    return n


def _read_tokens(c):
    """Cached tokens that at least one query of an attn case sees."""
    return sum(min(n, q - 1 + c["window"]) if c["causal"] and c["window"] else n
               for q, n in _lengths(c))


def _parents(c):
    r = random.Random(c["plan"])
    lens = [_logint(r, max(1, c["ctx"] // 8), c["ctx"]) for _ in range(c["seqs"])]
    # a beam keeps its own row more often than not; some rows end
    par = [i if r.random() < 0.5 else (-1 if r.random() < 0.1 else r.randrange(c["seqs"]))
           for i in range(c["seqs"])]
    return lens, par


def _copied(lens, par, page):
    """Rows that continue a partly filled page which an earlier row keeps."""
    seen, rows = set(), []
    for i, p in enumerate(par):
        if p >= 0 and lens[p] % page != 0 and p in seen:
            rows.append(i)
        seen.add(p)
    return rows


def _used_pages(c):
    r = random.Random(c["plan"])
    return sorted(r.sample(range(c["pages"]), max(1, int(c["pages"] * c["share"]))))


def work(case):
    c = case
    e = 4 if c.get("dtype") == "fp32" else 2
    if c["kind"] == "attn":
        rows = sum(q for q, _ in _lengths(c))
        b = 2 * rows * c["heads"] * c["dim"] * e + 2 * _read_tokens(c) * c["kv"] * c["dim"] * e
        b += 4 * sum(-(-n // c["page"]) for _, n in _lengths(c))
        return {"bytes": b, "flops": 4 * _pairs(c) * c["heads"] * c["dim"]}
    if c["kind"] in ("append", "rotary"):
        t, h = c["tokens"], c["heads"]
        rotated = h + c.get("kv", 0)
        b = 2 * t * (h + 2 * c.get("kv", 0)) * c["dim"] * e + t * (c["rot"] * 4 + 16)
        return {"bytes": b, "flops": 3 * t * rotated * c["rot"]}
    if c["kind"] == "extend":
        held = sum(-(-n // c["page"]) for _, n in _lengths(c))
        t = sum(q for q, _ in _lengths(c))
        return {"bytes": 2 * 4 * held + 8 * 2 * held + 16 * t + 12 * c["seqs"], "flops": 0}
    page = 2 * c["layers"] * c["kv"] * c["page"] * c["dim"] * e
    if c["kind"] == "fork":
        lens, par = _parents(c)
        held = sum(-(-n // c["page"]) for n in lens)
        copies = len(_copied(lens, par, c["page"]))
        return {"bytes": 2 * copies * page + 2 * 4 * held + 2 * 4 * held, "flops": 0}
    used = _used_pages(c)
    moves = sum(p >= len(used) for p in used)
    return {"bytes": 2 * moves * page + 2 * 4 * c["pages"] + 2 * 4 * len(used), "flops": 0}


# ------------------------------------------------------------------ inputs
def _inv_freq(c):
    """Inverse frequencies [rot / 2] in float64 and the factor on cos and sin."""
    f = [10000.0 ** (-2.0 * i / c["rot"]) for i in range(c["rot"] // 2)]
    if c["scaling"] == "linear":
        return [v / 8 for v in f], 1.0
    if c["scaling"] == "by_parts":  # fast pairs keep their angle, slow ones are stretched
        trained, factor, out = 8192.0, 16.0, []
        for v in f:
            turns = trained * v / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - 1.0) / (32.0 - 1.0)))
            out.append(v * keep + v / factor * (1 - keep))
        return out, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _table(c):
    f, m = _inv_freq(c)
    a = torch.arange(c["length"], dtype=torch.float64, device=DEV)[:, None] * \
        torch.tensor(f, dtype=torch.float64, device=DEV)
    return (torch.cat([a.cos(), a.sin()], dim=1) * m).float()


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    pages_rng = random.Random(seed)
    dt = _DT[c.get("dtype", "bf16")]
    st = dict(case=c)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)

    def place(counts, spare):
        """A block table over scattered pages, and the pool's size."""
        total = sum(counts)
        pool = total + spare
        ids = pages_rng.sample(range(pool), total)
        width = max(max(counts), 1) + 1
        rows, at = [], 0
        for n in counts:
            rows.append(ids[at:at + n] + [-1] * (width - n))
            at += n
        return _i32(rows), pool, ids

    if c["kind"] == "attn":
        lens = _lengths(c)
        st["lens"] = lens  # the scheduler's own copy
        st["table"], pool, _ = place([-(-n // c["page"]) for _, n in lens], 8)
        cu = [0]
        for q, _ in lens:
            cu.append(cu[-1] + q)
        st["cu"], st["ctx"] = _i32(cu), _i32([n for _, n in lens])
        st["max_q"] = max(q for q, _ in lens)
        # heads of different sharpness; values with a few strong channels
        sharp = torch.rand(c["heads"], 1, generator=g, device=DEV) * 2 + 0.5
        st["q"] = (randn(cu[-1], c["heads"], c["dim"]) * sharp).to(dt)
        shape = (pool, c["kv"], c["page"], c["dim"])
        strong = 1 + 4 * (torch.rand(c["dim"], generator=g, device=DEV) > 0.95).float()
        st["k"] = torch.empty(shape, dtype=dt, device=DEV)
        st["v"] = torch.empty(shape, dtype=dt, device=DEV)
        for p in range(0, pool, 2048):  # the float32 draws a part at a time
            n = min(2048, pool - p)
            st["k"][p:p + n] = randn(n, *shape[1:]).to(dt)
            st["v"][p:p + n] = (randn(n, *shape[1:]) * strong).to(dt)
        return st
    if c["kind"] in ("append", "rotary"):
        t = c["tokens"]
        st["rope"] = _table(c)
        # chunks of up to 500 neighbours, each at a place of its own
        r, pos = random.Random(c["plan"]), []
        while len(pos) < t:
            n = min(r.randint(1, 500), t - len(pos))
            p = r.randrange(c["length"] - n)
            pos += range(p, p + n)
        st["pos"] = torch.tensor(pos, dtype=torch.int64, device=DEV)
        if c["kind"] == "rotary":
            st["x"] = randn(t, c["heads"], c["dim"]).to(dt)
            return st
        h, k, d = c["heads"], c["kv"], c["dim"]
        # the fused projection's output, of which the three are slices
        qkv = randn(t, (h + 2 * k) * d).to(dt)
        st["q"] = qkv[:, :h * d].view(t, h, d)
        st["key"] = qkv[:, h * d:(h + k) * d].view(t, k, d)
        st["value"] = qkv[:, (h + k) * d:].view(t, k, d)
        pool = -(-t // c["page"]) + 4
        ids = pages_rng.sample(range(pool), pool)
        slots = [ids[i // c["page"]] * c["page"] + i % c["page"] for i in range(t)]
        for i in range(min(c["pad"], t - 1)):
            slots[t - 1 - i] = -1  # the batch is padded to a captured size
        st["slots"] = torch.tensor(slots, dtype=torch.int64, device=DEV)
        st["k"] = torch.zeros(pool, k, c["page"], d, dtype=dt, device=DEV)
        st["v"] = torch.zeros(pool, k, c["page"], d, dtype=dt, device=DEV)
        return st
    if c["kind"] == "extend":
        lens = _lengths(c)
        held = [n - q for q, n in lens]
        st["table"], pool, ids = place([-(-n // c["page"]) for n in held],
                                       sum(-(-n // c["page"]) for _, n in lens) + 16)
        width = max(-(-n // c["page"]) for _, n in lens) + 1
        grown = torch.full((c["seqs"], width), -1, dtype=torch.int32, device=DEV)
        grown[:, :st["table"].size(1)] = st["table"][:, :width]
        st["table"] = grown
        refs = [0] * pool
        for p in ids:
            refs[p] = 1
        cu = [0]
        for q, _ in lens:
            cu.append(cu[-1] + q)
        st.update(cu=_i32(cu), ctx=_i32(held), refs=_i32(refs), tokens=cu[-1])
        return st
    if c["kind"] == "fork":
        lens, par = _parents(c)
        st["table"], pool, ids = place([-(-n // c["page"]) for n in lens], c["seqs"] + 8)
        refs = [0] * pool
        for p in ids:
            refs[p] = 1
        st.update(ctx=_i32(lens), parents=_i32(par), refs=_i32(refs))
        # the scheduler knows which rows need a page of their own
        st["copied"] = _i32(_copied(lens, par, c["page"]))
    else:
        used, pool = _used_pages(c), c["pages"]
        refs = [0] * pool
        order = list(used)
        pages_rng.shuffle(order)
        for p in order:
            refs[p] = 1
        width = 64
        rows = [order[i:i + width] for i in range(0, len(order), width)]
        st["table"] = _i32([r + [-1] * (width - len(r)) for r in rows])
        st["refs"] = _i32(refs)
        st["moves"] = sum(p >= len(used) for p in used)
    # a layer's keys and values beside each other, so that a page moves whole
    st["caches"] = [randn(pool, 2, c["kv"], c["page"], c["dim"]).to(dt)
                    for _ in range(c["layers"])]
    return st


# --------------------------------------------------------------- own calls
def _run_own(st):
    c, ops = st["case"], _ops()
    if c["kind"] == "attn":
        return ops.zentorch_paged_attention(st["q"], st["k"], st["v"], st["table"], st["cu"],
                                            st["ctx"], st["max_q"], causal=c["causal"],
                                            window=c["window"])
    if c["kind"] == "rotary":
        return ops.zentorch_rotary_embedding(st["x"], st["pos"], st["rope"],
                                             interleaved=c["interleaved"])
    if c["kind"] == "append":
        q = ops.zentorch_rotary_cache_append(st["q"], st["key"], st["value"], st["pos"], st["rope"],
                                             st["slots"], st["k"], st["v"],
                                             interleaved=c["interleaved"])
        return q, st["k"], st["v"]
    if c["kind"] == "extend":
        return ops.zentorch_cache_extend(st["table"], st["ctx"], st["refs"], st["cu"], c["page"],
                                         st["tokens"])
    if c["kind"] == "fork":
        table, ctx, refs, copies = ops.zentorch_cache_fork(st["table"], st["ctx"], st["refs"],
                                                           st["parents"], c["page"])
        ops.zentorch_cache_copy_pages(st["caches"], copies)
        return table, ctx, refs, copies, st["caches"]
    table, refs, copies = ops.zentorch_cache_compact(st["table"], st["refs"])
    ops.zentorch_cache_copy_pages(st["caches"], copies)
    return table, refs, copies, st["caches"]


# ------------------------------------------------------------- plain forms
def _plain_attention(st):
    c = st["case"]
    h, kv, d = c["heads"], c["kv"], c["dim"]
    out = torch.empty_like(st["q"])
    at = 0
    for i, (q, n) in enumerate(st["lens"]):
        pages = st["table"][i, :-(-n // c["page"])]
        k = st["k"][pages].float().transpose(0, 1).reshape(kv, -1, d)[:, :n]
        v = st["v"][pages].float().transpose(0, 1).reshape(kv, -1, d)[:, :n]
        x = st["q"][at:at + q].float().view(q, kv, h // kv, d).permute(1, 2, 0, 3)
        s = torch.matmul(x.reshape(kv, -1, d), k.transpose(1, 2).contiguous())
        s = s.view(kv, h // kv, q, n) * (1.0 / math.sqrt(d))
        if c["causal"]:
            pos = torch.arange(n - q, n, device=DEV)[:, None]
            col = torch.arange(n, device=DEV)[None]
            hide = col > pos
            if c["window"]:
                hide = hide | (col <= pos - c["window"])
            s = s.masked_fill(hide, float("-inf"))
        p = torch.exp(s - s.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        o = torch.matmul(p.view(kv, -1, n), v).view(kv, h // kv, q, d)
        out[at:at + q] = o.permute(2, 0, 1, 3).reshape(q, h, d).to(out.dtype)
        at += q
    return out


def _plain_rotary(x, pos, table, interleaved):
    r = table.size(1)
    cos, sin = table[pos][:, None].split(r // 2, dim=-1)
    y = x.float()
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if interleaved else (y[..., :r // 2], y[..., r // 2:r])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    rot = torch.stack([ra, rb], dim=-1).flatten(-2) if interleaved else torch.cat([ra, rb], -1)
    return torch.cat([rot, y[..., r:]], dim=-1).to(x.dtype)


def _plain_append(st):
    c = st["case"]
    q = _plain_rotary(st["q"], st["pos"], st["rope"], c["interleaved"])
    key = _plain_rotary(st["key"], st["pos"], st["rope"], c["interleaved"])
    held = c["tokens"] - min(c["pad"], c["tokens"] - 1)  # the padding is at the end
    slots = st["slots"][:held]
    page, off = slots // c["page"], slots % c["page"]
    st["k"][page, :, off] = key[:held]
    st["v"][page, :, off] = st["value"][:held]
    return q, st["k"], st["v"]


def _free_pages(refs):
    """Page ids, the free ones first and ascending, and their number."""
    return torch.argsort((refs != 0).int(), stable=True), (refs == 0).sum()


def _plain_extend(st):
    c = st["case"]
    size, t = c["page"], st["tokens"]
    table, ctx, refs = st["table"].long(), st["ctx"].long(), st["refs"].clone()
    cu, pool, width = st["cu"].long(), st["refs"].numel(), st["table"].size(1)
    new = cu[1:] - cu[:-1]
    have, want = (ctx + size - 1) // size, (ctx + new + size - 1) // size
    need = torch.where(want <= width, want - have, 0)
    end = need.cumsum(0)
    order, free = _free_pages(refs)
    granted = (want <= width) & (end <= free)
    col = torch.arange(width, device=DEV)[None]
    fresh = granted[:, None] & (col >= have[:, None]) & (col < want[:, None])
    rank = (end - need)[:, None] + col - have[:, None]
    page = order[rank.clamp(0, pool - 1)]
    table = torch.where(fresh, page, table)
    refs.scatter_add_(0, page.flatten(), fresh.flatten().int())
    tok = torch.arange(t, device=DEV)
    row = torch.searchsorted(cu, tok, right=True) - 1
    pos = ctx[row] + tok - cu[row]
    ok = granted[row]
    held = table[row, (pos // size).clamp(max=width - 1)]
    slot = torch.where(ok & (held >= 0), held * size + pos % size, -1)
    return (table.int(), torch.where(granted, ctx + new, ctx).int(), refs,
            torch.where(ok, pos, -1), slot)


def _copy_pages(caches, copies):
    src, dst = copies.unbind(1)
    for cache in caches:
        cache[dst] = cache[src]


def _plain_fork(st):
    c = st["case"]
    size, rows = c["page"], c["seqs"]
    table, ctx, refs = st["table"].long(), st["ctx"].long(), st["refs"].long()
    par, pool, width = st["parents"].long(), st["refs"].numel(), st["table"].size(1)
    alive = par >= 0
    p = par.clamp(min=0)
    idx = torch.arange(rows, device=DEV)
    children = torch.zeros(rows, dtype=torch.int64, device=DEV).scatter_add_(0, p, alive.long())
    first = torch.full((rows,), rows, device=DEV).scatter_reduce_(
        0, p, torch.where(alive, idx, rows), "amin")
    have = (ctx + size - 1) // size
    part = ctx % size != 0
    col = torch.arange(width, device=DEV)[None]
    last = part[:, None] & (col == have[:, None] - 1)
    gain = torch.where(last, (children > 0).long()[:, None], children[:, None]) - 1
    in_use = col < have[:, None]
    refs = refs.scatter_add(0, table.clamp(min=0).flatten(),
                            torch.where(in_use, gain, 0).flatten())
    order, free = _free_pages(refs)
    need = alive & part[p] & (first[p] != idx)
    rank = need.cumsum(0) - 1
    lost = need & (rank >= free)
    page = order[rank.clamp(0, pool - 1)]
    fresh = need & ~lost
    keep = alive & ~lost
    new = torch.where(keep[:, None] & in_use[p], table[p], -1)
    source = table[p].gather(1, (have[p] - 1).clamp(min=0)[:, None])[:, 0]
    new = torch.where(fresh[:, None] & last[p], page[:, None], new)
    refs = refs.scatter_add(0, page, fresh.long())
    gone = lost[:, None] & in_use[p] & ~last[p]
    refs = refs.scatter_add(0, table[p].clamp(min=0).flatten(), -gone.flatten().long())
    copies = torch.where(fresh[:, None], torch.stack([source, page], 1), -1).int()
    _copy_pages(st["caches"], copies[st["copied"]].long())
    return new.int(), torch.where(keep, ctx[p], 0).int(), refs.int(), copies, st["caches"]


def _plain_compact(st):
    c = st["case"]
    table, refs = st["table"].long(), st["refs"]
    pool = refs.numel()
    idx = torch.arange(pool, device=DEV)
    used = refs != 0
    n = used.sum()
    moves, holes = used & (idx >= n), ~used & (idx < n)
    src = torch.argsort((~moves).int(), stable=True)[:pool // 2]
    dst = torch.argsort((~holes).int(), stable=True)[:pool // 2]
    real = torch.arange(pool // 2, device=DEV) < moves.sum()
    copies = torch.where(real[:, None], torch.stack([src, dst], 1), -1).int()
    to = idx.clone().scatter_(0, src, torch.where(real, dst, src))
    table = torch.where(table >= 0, to[table.clamp(min=0)], table)
    new_refs = torch.where(idx < n, refs, 0)
    new_refs = new_refs.scatter(0, torch.where(real, dst, idx[:pool // 2]),
                                torch.where(real, refs[src], new_refs[:pool // 2]))
    new_refs = torch.where(holes, torch.zeros_like(refs).scatter(0, to, refs), new_refs)
    _copy_pages(st["caches"], copies[:st["moves"]].long())
    return table.int(), new_refs.int(), copies, st["caches"]


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "attn":
        return _plain_attention(state)
    if kind == "rotary":
        return _plain_rotary(state["x"], state["pos"], state["rope"], state["case"]["interleaved"])
    return {"append": _plain_append, "extend": _plain_extend, "fork": _plain_fork,
            "compact": _plain_compact}[kind](state)


# ------------------------------------------------------------------- exact
def _exact_attention(c, st):
    """o_r = sum_j exp(s_rj) v_j / sum_j exp(s_rj) over the j that row r sees."""
    group = c["heads"] // c["kv"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    row = 0
    for i, (q, n) in enumerate(_lengths(c)):
        tok = torch.arange(n, device=DEV)
        page, off = st["table"][i].long()[tok // c["page"]], tok % c["page"]
        for h in range(c["kv"]):
            k, v = st["k"][page, h, off].double(), st["v"][page, h, off].double()
            step = max(1, 2 ** 26 // n)  # rows at a time: 0.5 GB of scores
            for head in range(h * group, (h + 1) * group):
                for a in range(0, q, step):
                    b = min(q, a + step)
                    s = st["q"][row + a:row + b, head].double() @ k.t() / math.sqrt(c["dim"])
                    if c["causal"]:
                        back = torch.arange(n - q + a, n - q + b, device=DEV)[:, None] - tok[None]
                        seen = back >= 0
                        if c["window"]:
                            seen &= back < c["window"]
                        s = torch.where(seen, s, -torch.inf)
                    e = torch.exp(s - s.max(dim=1, keepdim=True).values)
                    out[row + a:row + b, head] = (e @ v) / e.sum(dim=1, keepdim=True)
        row += q
    return out


def _exact_rotary(c, x, pos):
    """Pair (a, b) as the complex number a + ib, times m exp(i pos f)."""
    f, m = _inv_freq(c)
    angle = pos.double()[:, None] * torch.tensor(f, dtype=torch.float64, device=DEV)
    turn = torch.polar(torch.full_like(angle, m), angle)[:, None]
    y, r = x.double().clone(), c["rot"]
    if c["interleaved"]:
        z = torch.complex(y[..., 0:r:2], y[..., 1:r:2]) * turn
        y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
    else:
        z = torch.complex(y[..., :r // 2], y[..., r // 2:r]) * turn
        y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
    return y


def _moved(caches, pairs):
    out = [x.double() for x in caches]
    for x in out:
        for src, dst in pairs:
            x[dst] = x[src]
    return out


def _exact_fork(c, st):
    """Row by row, page by page: which pages end up copied where."""
    lens, par = _parents(c)
    table, size = st["table"].tolist(), c["page"]
    live, kept, wants = set(), set(), []
    for p in par:
        if p < 0:
            continue
        pages = table[p][:-(-lens[p] // size)]
        if lens[p] % size and p in kept:
            wants.append(pages[-1])
            pages = pages[:-1]
        kept.add(p)
        live.update(pages)
    free = (i for i in range(st["refs"].numel()) if i not in live)
    return [None] * 4 + [_moved(st["caches"], [(w, next(free)) for w in wants])]


def _exact_compact(c, st):
    used = _used_pages(c)
    n, held = len(used), set(used)
    holes = [p for p in range(n) if p not in held]
    return [None] * 3 + [_moved(st["caches"], list(zip([p for p in used if p >= n], holes)))]


def exact(case, seed):
    c = case
    if c["kind"] == "extend":
        return None  # whole numbers
    st = prepare(c, seed)
    if c["kind"] == "fork":
        return _exact_fork(c, st)
    if c["kind"] == "compact":
        return _exact_compact(c, st)
    if c["kind"] == "attn":
        return _exact_attention(c, st)
    if c["kind"] == "rotary":
        return _exact_rotary(c, st["x"], st["pos"])
    size = c["page"]
    k, v = st["k"].double(), st["v"].double()
    held = torch.nonzero(st["slots"] >= 0)[:, 0]
    page, off = st["slots"][held] // size, st["slots"][held] % size
    for head in range(c["kv"]):
        k[page, head, off] = _exact_rotary(c, st["key"], st["pos"])[held, head]
        v[page, head, off] = st["value"].double()[held, head]
    return _exact_rotary(c, st["q"], st["pos"]), k, v
