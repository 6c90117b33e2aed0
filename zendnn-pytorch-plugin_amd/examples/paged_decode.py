"""A small int4 decoder served from a paged key / value cache.

Prompts of different lengths are prefilled in one batch, every sequence is
continued by a few decode steps, some sequences then branch into several
continuations (sharing their pages) while others end, and the pool is compacted
before the last steps.  The linears are zentorch's int4 ops, and between them
run the cache's: extend -> rotary + append -> attention in every layer, fork
and compact with the page copies between steps.

Weights are random.  ``python paged_decode.py`` prints the continuations and
how far the last logits are from those of a cacheless recomputation of every
whole sequence in plain torch operations.
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import zentorch  # noqa: E402,F401

ops = torch.ops.zentorch


class Decoder:
    """Pre-norm decoder layers with grouped-query attention and a gated MLP."""

    def __init__(self, layers=2, hidden=512, heads=8, kv_heads=2, dim=64, inter=1024, vocab=1000,
                 device="cuda", seed=0):
        self.g = torch.Generator().manual_seed(seed)
        self.device, self.heads, self.kv, self.dim = device, heads, kv_heads, dim
        self.embed = (torch.randn(vocab, hidden, generator=self.g) * 0.5).bfloat16().to(device)
        self.layers = [dict(qkv=self._int4((heads + 2 * kv_heads) * dim, hidden),
                            o=self._int4(hidden, heads * dim), gate_up=self._int4(2 * inter, hidden),
                            down=self._int4(hidden, inter)) for _ in range(layers)]

    def _int4(self, n, k, group=128):
        q = torch.randint(-8, 8, (n, k), generator=self.g, dtype=torch.int8)
        s = ((torch.rand(k // group, n, generator=self.g) * 0.5 + 0.75) / (4.6 * math.sqrt(k))).bfloat16()
        dense = (q.float().view(n, k // group, group) * s.float().t()[:, :, None]).view(n, k).bfloat16()
        return dict(w=ops.zentorch_woq_repack_weight(q.to(self.device)).t(), s=s.to(self.device),
                    dense=dense.to(self.device))

    @staticmethod
    def norm(x):
        return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)

    def rope(self, length):
        f = 10000.0 ** (-torch.arange(0, self.dim, 2, dtype=torch.float64) / self.dim)
        a = torch.arange(length, dtype=torch.float64)[:, None] * f
        return torch.cat([a.cos(), a.sin()], 1).float().to(self.device)

    def step(self, tokens, cache, cu, max_query_len):
        """Logits of every sequence's last new token; `tokens` are the new ones
        of all sequences, sequence i's being cu[i] .. cu[i + 1]."""
        pos, slots = cache.extend(cu, tokens.numel())
        x = self.embed[tokens]
        for p, (k_cache, v_cache) in zip(self.layers, cache.views):
            h = ops.zentorch_woq_linear(self.norm(x), p["qkv"]["w"], p["qkv"]["s"], None)
            q, k, v = (t.view(tokens.numel(), -1, self.dim) for t in h.split(
                [self.heads * self.dim, self.kv * self.dim, self.kv * self.dim], dim=1))
            q = ops.zentorch_rotary_cache_append(q, k, v, pos, cache.cos_sin, slots, k_cache, v_cache)
            a = ops.zentorch_paged_attention(q, k_cache, v_cache, cache.table, cu, cache.lens, max_query_len)
            x = ops.zentorch_woq_linear_add(a.flatten(1), p["o"]["w"], p["o"]["s"], None, x)
            m = ops.zentorch_woq_linear_gate_up_silu_mul(self.norm(x), p["gate_up"]["w"], p["gate_up"]["s"], None)
            x = ops.zentorch_woq_linear_add(m, p["down"]["w"], p["down"]["s"], None, x)
        return self.norm(x[cu[1:].long() - 1]).float() @ self.embed.float().t()

    def whole(self, tokens):
        """Logits after one whole sequence, in plain operations without a cache."""
        n = tokens.numel()
        cos, sin = self.rope(n)[:, None].chunk(2, -1)
        x = self.embed[tokens].float()

        def turn(y):
            a, b = y.chunk(2, -1)
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

        for p in self.layers:
            w = {k: t["dense"].float() for k, t in p.items()}
            h = self.norm(x) @ w["qkv"].t()
            q, k, v = (t.view(n, -1, self.dim) for t in h.split(
                [self.heads * self.dim, self.kv * self.dim, self.kv * self.dim], dim=1))
            q, k = turn(q), turn(k)
            rep = self.heads // self.kv
            q, k, v = q.transpose(0, 1), k.repeat_interleave(rep, 1).transpose(0, 1), v.repeat_interleave(rep, 1).transpose(0, 1)
            s = (q @ k.transpose(1, 2).contiguous()) / math.sqrt(self.dim)
            s = s.masked_fill(torch.ones(n, n, device=self.device).triu(1).bool(), -math.inf)
            x = x + (torch.softmax(s, -1) @ v).transpose(0, 1).reshape(n, -1) @ w["o"].t()
            g, u = (self.norm(x) @ w["gate_up"].t()).chunk(2, -1)
            x = x + (torch.nn.functional.silu(g) * u) @ w["down"].t()
        return self.norm(x[-1]).float() @ self.embed.float().t()


class PagedCache:
    """Every layer's pages, one block table for all of them, and its upkeep."""

    def __init__(self, model, rows, pages=96, page_size=16, width=16):
        dev, self.size = model.device, page_size
        self.layers = [torch.zeros(pages, 2, model.kv, page_size, model.dim, dtype=torch.bfloat16, device=dev)
                       for _ in model.layers]
        self.views = [c.unbind(1) for c in self.layers]
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(rows, dtype=torch.int32, device=dev)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=dev)
        self.cos_sin = model.rope(width * page_size)

    def extend(self, cu, tokens):
        self.table, self.lens, self.refs, pos, slots = ops.zentorch_cache_extend(
            self.table, self.lens, self.refs, cu, self.size, tokens)
        return pos, slots

    def fork(self, parents):
        self.table, self.lens, self.refs, copies = ops.zentorch_cache_fork(
            self.table, self.lens, self.refs, parents, self.size)
        ops.zentorch_cache_copy_pages(self.layers, copies)

    def compact(self):
        self.table, self.refs, copies = ops.zentorch_cache_compact(self.table, self.refs)
        ops.zentorch_cache_copy_pages(self.layers, copies)


def run(prompt_lens=(37, 5, 64, 18), steps=6, device="cuda"):
    """(sequences, the last step's logits, the plain ones, the cache)."""
    model = Decoder(device=device)
    rows = len(prompt_lens)
    cache = PagedCache(model, rows)
    g = torch.Generator().manual_seed(1)
    seqs = [torch.randint(0, 1000, (n,), generator=g).to(device) for n in prompt_lens]

    def i32(v):
        return torch.tensor(v, dtype=torch.int32, device=device)

    cu = i32([sum(prompt_lens[:i]) for i in range(rows + 1)])
    logits = model.step(torch.cat(seqs), cache, cu, max(prompt_lens))
    one = i32(list(range(rows + 1)))
    for i in range(steps):
        rank = torch.zeros(rows, dtype=torch.int64, device=device)
        if i == steps // 2:  # row 0 goes on three times (its best three tokens), row 1 ends
            parents = [0, 0, 2, 0] + list(range(4, rows))
            cache.fork(i32(parents))
            seqs, logits = [seqs[p] for p in parents], logits[parents]
            rank[1], rank[3] = 1, 2
            cache.compact()
        new = logits.topk(3, dim=1).indices.gather(1, rank[:, None])[:, 0]
        seqs = [torch.cat([s, t[None]]) for s, t in zip(seqs, new)]
        logits = model.step(new, cache, one, 1)
    return seqs, logits, torch.stack([model.whole(s) for s in seqs]), cache


if __name__ == "__main__":
    seqs, got, want, cache = run()
    for s in seqs:
        print(len(s), s[-8:].tolist())
    rel = ((got - want).norm() / want.norm()).item()
    print(f"logits off by {rel:.4f} of their norm; {int((cache.refs > 0).sum())} pages in use")
