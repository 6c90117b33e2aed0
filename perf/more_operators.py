"""Performance cases of the key / value cache held in 4 bits: quantising a
step's keys and values as they are written, reading them back, and attention
over them.

The format (MXFP4): a head row of ``dim`` numbers is cut into blocks of 32, the
last one filled with zeros.  A block has a scale 2^E, kept as the byte E + 127,
and 32 codes of 4 bits, the element of even index in a byte's low half: bit 3
is the sign, the others name one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.  E is such that
the largest magnitude is at least 3.5 and less than 7 scales, held to -125 ..
125.  A layer's cache is four uint8 tensors, codes ``[pages, kv_heads,
page_size, 16 blocks]`` and scales ``[pages, kv_heads, page_size, blocks]`` of
keys and of values.  Tables, lengths and slots are the paged cache's: sequence
i's tokens lie in the pages that row i of ``block_table`` names, in order;
``context_lens[i]`` counts them, the new ones included, and the new ones of
sequence i are rows ``cu_seqlens[i] .. cu_seqlens[i + 1]`` of the batch.

The kinds of cases:

* ``attn``    ``zentorch_paged_attention_mxfp4``, one call of one layer;
* ``append``  ``zentorch_rotary_cache_append_mxfp4``: the rotated query of one
  layer, its rotated keys and its values quantised into the cache; and
  ``zentorch_cache_read_mxfp4``, which gives what the cache now holds for them;
* ``read``    ``zentorch_cache_read_mxfp4`` of tokens that are there already.

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
        # A float32 decode step with heads that blocks of 32 do not divide.
        dict(name="attn_decode_fp32", kind="attn", plan=7, batch="ragged", seqs=16, chunk=1,
             ctx=4096, heads=32, kv=32, dim=80, page=24, causal=True, window=0, dtype="fp32"),
        # A decode step's new tokens into one layer's cache.
        dict(name="append_decode", kind="append", plan=8, tokens=8, pad=1, heads=32, kv=8, dim=128,
             rot=128, page=16, length=131072, interleaved=False, scaling="by_parts",
             dtype="bf16"),
        # A large prompt batch into one layer's cache.
        dict(name="append_prefill", kind="append", plan=9, tokens=8191, pad=0, heads=32, kv=8,
             dim=128, rot=128, page=16, length=32768, interleaved=False, scaling="none",
             dtype="bf16"),
        # Interleaved pairs over part of a float32 head, far positions.
        dict(name="append_partial_fp32", kind="append", plan=10, tokens=1000, pad=5, heads=16,
             kv=4, dim=80, rot=32, page=24, length=131072, interleaved=True, scaling="linear",
             dtype="fp32"),
        # The last page of a sequence, looked at.
        dict(name="read_page", kind="read", plan=11, tokens=16, pad=0, kv=8, dim=128, page=16,
             dtype="bf16"),
        # A long prefix that goes to a program without the 4-bit format.
        dict(name="read_prefix", kind="read", plan=12, tokens=65536, pad=3, kv=8, dim=128, page=64,
             dtype="bf16"),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(32, 8), (32, 32), (28, 4), (16, 16), (8, 1), (64, 8), (12, 2)]


def draw(rng):
    kind = rng.choice(["attn"] * 6 + ["append"] * 2 + ["read"])
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
            if w["flops"] <= (2.4e11 if dtype == "bf16" else 1.5e10) and w["bytes"] <= 2.8e8:
                return c
            if c["seqs"] > 1:
                c["seqs"] //= 2
            elif c["chunk"] > 1:
                c["chunk"] = (c["chunk"] + 1) // 2
                if c["batch"] == "whole":
                    c["ctx"] = c["chunk"]
            else:
                c["ctx"] //= 2
    pad = rng.choice([0, 0, 1, 5])
    if kind == "append":
        return dict(kind=kind, plan=plan, tokens=_logint(rng, 1, 8192), pad=pad, heads=heads,
                    kv=kv, dim=dim, rot=dim if rng.random() < 0.6 else rng.choice([16, 32, 48]),
                    page=page, length=_logint(rng, 4096, 131072),
                    interleaved=rng.random() < 0.4,
                    scaling=rng.choice(["none", "linear", "by_parts"]), dtype=dtype)
    most = 134217728 // (kv * dim * (2 if dtype == "fp32" else 1))
    return dict(kind="read", plan=plan, tokens=_logint(rng, 1, min(65536, most)), pad=pad, kv=kv,
                dim=dim, page=page, dtype=dtype)


# ------------------------------------------------------------------- plans
def _lengths(c):
    """(new tokens, all tokens) of every sequence of an attn case."""
    r = random.Random(c["plan"])
    out = []
    for i in range(c["seqs"]):
        q, n = c["chunk"], c["ctx"]
        if c["batch"] in ("ragged", "mixed"):
            n = _logint(r, max(1, c["ctx"] // 32), c["ctx"])
        if c["batch"] == "ragged":
            q = r.randint(1, c["chunk"])
        elif c["batch"] == "mixed":  # mostly decoding, one chunk in eight
            q = r.randint(1, c["chunk"]) if i % 8 == 0 else 1
        elif c["batch"] == "whole":
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


def _held(c):
    """Tokens of an append or read case that are not padding."""
    return c["tokens"] - min(c["pad"], c["tokens"] - 1)


def _blocks(c):
    return -(-c["dim"] // 32)


def work(case):
    c = case
    e = 4 if c["dtype"] == "fp32" else 2
    row = 17 * _blocks(c)  # bytes of a head row in the cache
    if c["kind"] == "attn":
        rows = sum(q for q, _ in _lengths(c))
        b = 2 * rows * c["heads"] * c["dim"] * e + 2 * _read_tokens(c) * c["kv"] * row
        b += 4 * sum(-(-n // c["page"]) for _, n in _lengths(c))
        return {"bytes": b, "flops": 4 * _pairs(c) * c["heads"] * c["dim"]}
    t, n, kv, d = c["tokens"], _held(c), c["kv"], c["dim"]
    if c["kind"] == "append":  # the keys and values go in, and come back as they are held
        b = 2 * t * c["heads"] * d * e + 2 * n * kv * (d * e + row) + t * (c["rot"] * 4 + 16)
        b += 2 * n * kv * row + 2 * t * kv * d * e
        return {"bytes": b, "flops": 3 * t * (c["heads"] + kv) * c["rot"] + 4 * n * kv * d}
    return {"bytes": 2 * n * kv * row + 2 * t * kv * d * e + 8 * t, "flops": 2 * n * kv * d}


# --------------------------------------------------------------- the format
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _powers():
    """2^E for the scale bytes 0 .. 254, in 64 bits."""
    return torch.tensor([2.0 ** (b - 127) for b in range(255)], dtype=torch.float64, device=DEV)


def _quantise(x):
    """(codes, scales, values) of head rows [..., dim] that are finite.  Whole
    numbers and comparisons in 64 bits decide, so that nothing is rounded
    before a code is."""
    d = x.size(-1)
    y = torch.nn.functional.pad(x.double(), (0, -d % 32)).unflatten(-1, (-1, 32))
    part, exponent = torch.frexp(y.abs().amax(-1))  # amax = part * 2^exponent, 0.5 <= part < 1
    exponent = exponent + (part >= 0.875) - 3
    scale = torch.where(part > 0, exponent, -125).clamp(-125, 125) + 127
    unit = _powers()[scale][..., None]
    v = y.abs() / unit
    code = torch.zeros_like(scale)[..., None].expand(v.shape).clone()
    # halfway between two values the even code is taken
    for i, (a, b) in enumerate(zip(_GRID, _GRID[1:])):
        code += (v > (a + b) / 2) if i % 2 == 0 else (v >= (a + b) / 2)
    sign = (y < 0) & (code > 0)
    grid = torch.tensor(_GRID, dtype=torch.float64, device=DEV)
    values = grid[code.long()] * unit * torch.where(sign, -1.0, 1.0)
    code = (code + 8 * (y < 0)).flatten(-2)
    packed = (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8)
    return packed, scale.to(torch.uint8), values.flatten(-2)[..., :d]


def _values(codes, scales, d):
    """The numbers of head rows, in float32 (which holds them all)."""
    grid = torch.tensor([*_GRID, *(-g for g in _GRID)], dtype=torch.float32, device=DEV)
    both = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).int()
    unit = _powers().float()[scales.int()]
    return (grid[both].unflatten(-1, (-1, 32)) * unit[..., None]).flatten(-2)[..., :d]


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
    dt = _DT[c["dtype"]]
    st = dict(case=c)
    nb = _blocks(c)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)

    def pool_of(pages):
        for x in "kv":
            st[x] = torch.zeros(pages, c["kv"], c["page"], 16 * nb, dtype=torch.uint8, device=DEV)
            st[x + "_sc"] = torch.zeros(pages, c["kv"], c["page"], nb, dtype=torch.uint8, device=DEV)

    def fill():
        """Every page from numbers of a cache's kind: some strong channels."""
        pages = st["k"].size(0)
        strong = 1 + 4 * (torch.rand(c["dim"], generator=g, device=DEV) > 0.95).float()
        step = max(1, (1 << 25) // (c["kv"] * c["page"] * c["dim"]))
        for p in range(0, pages, step):  # the wide draws a part at a time
            n = min(step, pages - p)
            for x in "kv":
                y = randn(n, c["kv"], c["page"], c["dim"]) * (strong if x == "v" else 1)
                st[x][p:p + n], st[x + "_sc"][p:p + n], _ = _quantise(y.to(dt))

    def slots_of(tokens, held, pool):
        ids = pages_rng.sample(range(pool), pool)
        slots = [ids[i // c["page"]] * c["page"] + i % c["page"] for i in range(tokens)]
        slots[held:] = [-1] * (tokens - held)  # the batch is padded to a captured size
        return torch.tensor(slots, dtype=torch.int64, device=DEV)

    if c["kind"] == "attn":
        lens = _lengths(c)
        st["lens"] = lens  # the scheduler's own copy
        counts = [-(-n // c["page"]) for _, n in lens]
        total, width = sum(counts), max(counts) + 1
        ids = pages_rng.sample(range(total + 8), total)
        rows, at = [], 0
        for n in counts:
            rows.append(ids[at:at + n] + [-1] * (width - n))
            at += n
        st["table"] = _i32(rows)
        cu = [0]
        for q, _ in lens:
            cu.append(cu[-1] + q)
        st["cu"], st["ctx"] = _i32(cu), _i32([n for _, n in lens])
        st["max_q"] = max(q for q, _ in lens)
        # heads of different sharpness
        sharp = torch.rand(c["heads"], 1, generator=g, device=DEV) * 2 + 0.5
        st["q"] = (randn(cu[-1], c["heads"], c["dim"]) * sharp).to(dt)
        pool_of(total + 8)
        fill()
        return st
    t, pool = c["tokens"], -(-c["tokens"] // c["page"]) + 4
    pool_of(pool)
    st["slots"] = slots_of(t, _held(c), pool)
    if c["kind"] == "read":
        fill()
        return st
    st["rope"] = _table(c)
    # chunks of up to 500 neighbours, each at a place of its own
    r, pos = random.Random(c["plan"]), []
    while len(pos) < t:
        n = min(r.randint(1, 500), t - len(pos))
        p = r.randrange(c["length"] - n)
        pos += range(p, p + n)
    st["pos"] = torch.tensor(pos, dtype=torch.int64, device=DEV)
    h, k, d = c["heads"], c["kv"], c["dim"]
    # the fused projection's output, of which the three are slices
    qkv = randn(t, (h + 2 * k) * d).to(dt)
    st["q"] = qkv[:, :h * d].view(t, h, d)
    st["key"] = qkv[:, h * d:(h + k) * d].view(t, k, d)
    st["value"] = qkv[:, (h + k) * d:].view(t, k, d)
    return st


# --------------------------------------------------------------- own calls
def _run_own(st):
    c, ops = st["case"], _ops()
    cache = st["k"], st["k_sc"], st["v"], st["v_sc"]
    if c["kind"] == "attn":
        return ops.zentorch_paged_attention_mxfp4(st["q"], *cache, st["table"], st["cu"],
                                                  st["ctx"], st["max_q"], causal=c["causal"],
                                                  window=c["window"])
    if c["kind"] == "append":
        q = ops.zentorch_rotary_cache_append_mxfp4(st["q"], st["key"], st["value"], st["pos"],
                                                   st["rope"], st["slots"], *cache,
                                                   interleaved=c["interleaved"])
    k, v = ops.zentorch_cache_read_mxfp4(*cache, st["slots"], c["dim"], dtype=_DT[c["dtype"]])
    return (q, k, v) if c["kind"] == "append" else (k, v)


# ------------------------------------------------------------- plain forms
def _plain_attention(st):
    c = st["case"]
    h, kv, d = c["heads"], c["kv"], c["dim"]
    out = torch.empty_like(st["q"])
    at = 0
    for i, (q, n) in enumerate(st["lens"]):
        pages = st["table"][i, :-(-n // c["page"])]
        k, v = (_values(st[x][pages], st[x + "_sc"][pages], d).transpose(0, 1)
                .reshape(kv, -1, d)[:, :n] for x in "kv")
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
        o = torch.matmul(p.view(kv, -1, n), v.contiguous()).view(kv, h // kv, q, d)
        out[at:at + q] = o.permute(2, 0, 1, 3).reshape(q, h, d).to(out.dtype)
        at += q
    return out


def _turn(y, pos, table, interleaved):
    r = table.size(1)
    cos, sin = table[pos][:, None].to(y.dtype).split(r // 2, dim=-1)
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if interleaved else (y[..., :r // 2], y[..., r // 2:r])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    rot = torch.stack([ra, rb], dim=-1).flatten(-2) if interleaved else torch.cat([ra, rb], -1)
    return torch.cat([rot, y[..., r:]], dim=-1)


def _plain_append(st):
    c = st["case"]
    dt, held = _DT[c["dtype"]], _held(c)  # the padding is at the end
    q = _turn(st["q"].float(), st["pos"], st["rope"], c["interleaved"]).to(dt)
    # a key next to a border takes its side by the exact products
    key = _turn(st["key"].double(), st["pos"], st["rope"], c["interleaved"])
    slots = st["slots"][:held]
    page, off = slots // c["page"], slots % c["page"]
    out = [q]
    for x, y in (("k", key), ("v", st["value"])):
        st[x][page, :, off], st[x + "_sc"][page, :, off], values = _quantise(y[:held])
        back = torch.zeros(y.shape, dtype=dt, device=DEV)
        back[:held] = values.to(dt)
        out.append(back)
    return tuple(out)


def _plain_read(st):
    c = st["case"]
    held = (st["slots"] >= 0)[:, None, None]
    slots = st["slots"].clamp(min=0)
    page, off = slots // c["page"], slots % c["page"]
    return tuple((_values(st[x][page, :, off], st[x + "_sc"][page, :, off], c["dim"]) * held)
                 .to(_DT[c["dtype"]]) for x in "kv")


def run(state):
    if own:
        return _run_own(state)
    return {"attn": _plain_attention, "append": _plain_append,
            "read": _plain_read}[state["case"]["kind"]](state)


# ------------------------------------------------------------------- exact
def _number(codes, scales):
    """What 4-bit codes [...] and their scale bytes stand for, bit by bit:
    s eem is (-1)^s 2^(ee - 1) (1 + m / 2), or (-1)^s m / 2 where ee is 0."""
    codes, sign = codes & 7, 1 - 2 * ((codes >> 3) & 1).double()
    e, m = (codes >> 1).double(), (codes & 1).double() / 2
    return sign * torch.where(e == 0, m, (1 + m) * torch.exp2(e - 1)) * \
        torch.exp2(scales.double() - 127)


def _rows(c, codes, scales):
    """Head rows [n, dim] of codes [n, 16 blocks] and scales [n, blocks]."""
    i = torch.arange(c["dim"], device=DEV)
    byte = codes[:, i // 2].int()
    return _number(torch.where(i % 2 == 0, byte, byte >> 4) & 15, scales[:, i // 32])


def _exact_attention(c, st):
    """o_r = sum_j exp(s_rj) v_j / sum_j exp(s_rj) over the j that row r sees."""
    group = c["heads"] // c["kv"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    row = 0
    for i, (q, n) in enumerate(_lengths(c)):
        tok = torch.arange(n, device=DEV)
        page, off = st["table"][i].long()[tok // c["page"]], tok % c["page"]
        for h in range(c["kv"]):
            k, v = (_rows(c, st[x][page, h, off], st[x + "_sc"][page, h, off]) for x in "kv")
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


def _exact_turn(c, st, x):
    """Pair (a, b) as the complex number a + ib, times the table's cos + i sin."""
    t = st["rope"].double()[st["pos"]]
    turn = torch.complex(t[:, :c["rot"] // 2], t[:, c["rot"] // 2:])[:, None]
    y, r = x.double().clone(), c["rot"]
    at = (slice(0, r, 2), slice(1, r, 2)) if c["interleaved"] else \
        (slice(0, r // 2), slice(r // 2, r))
    z = torch.complex(y[..., at[0]], y[..., at[1]]) * turn
    y[..., at[0]], y[..., at[1]] = z.real, z.imag
    return y


def _exact_held(c, x):
    """What a cache holds of rows x: the nearest number of the block's sixteen,
    by their distances."""
    n = _held(c)
    out = torch.zeros_like(x)
    for at in range(0, c["dim"], 32):
        y = x[:n, :, at:at + 32]
        top = y.abs().amax(-1, keepdim=True)
        # the least power of two of which seven are more than the largest
        e = torch.ceil(torch.log2(top / 7))
        e = torch.where(7 * torch.exp2(e) <= top, e + 1, e)
        e = torch.where(7 * torch.exp2(e - 1) > top, e - 1, e).clamp(-125, 125)
        unit = torch.exp2(e)
        near, best = torch.full_like(y, torch.inf), torch.zeros_like(y)
        for code in (0, 2, 4, 6, 1, 3, 5, 7):  # of two equally near ones an even code
            value = _number(torch.tensor(code, device=DEV), torch.tensor(127, device=DEV)) * unit
            far = (y.abs() - value).abs()
            best = torch.where(far < near, value, best)
            near = torch.minimum(near, far)
        out[:n, :, at:at + 32] = torch.copysign(best, y)
    return out


def exact(case, seed):
    c = case
    st = prepare(c, seed)
    if c["kind"] == "attn":
        return _exact_attention(c, st)
    if c["kind"] == "append":
        return (_exact_turn(c, st, st["q"]), _exact_held(c, _exact_turn(c, st, st["key"])),
                _exact_held(c, st["value"].double()))
    out = []
    for x in "kv":
        y = torch.zeros(c["tokens"], c["kv"], c["dim"], dtype=torch.float64, device=DEV)
        slots = st["slots"][:_held(c)]
        for h in range(c["kv"]):
            at = slots // c["page"], h, slots % c["page"]
            y[:_held(c), h] = _rows(c, st[x][at], st[x + "_sc"][at])
        out.append(y)
    return tuple(out)
