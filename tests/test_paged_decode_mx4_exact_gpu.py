"""The paged decoding example over a cache held in 4 bits, against the same steps
with append and attention computed from their definitions in 64 bits (mx4_ref.py,
kv_ref.py); the linears between them are the same calls.

The runs differ where attention's outputs round differently: by bf16's 2^-8 of a number
and 0.0022 of their norm at most, in each of two layers.  What follows differs by as
much, some 0.4 %, until it is quantised: a number off by d takes another code, a step s
away, once in s / d times, so by sqrt(d s) in the mean.  With numbers of two scales and
steps of a half that is 0.03 of a key or value, of which a score sums 64 and an output
some 40: less than 0.01 of each.  Two layers and the sums with the residual stay within
0.05 of the logits' norm; keys and values exchanged pass that."""
import importlib.util
import os

import pytest
import torch

import kv_ref as R
import mx4_ref as M

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "zendnn-pytorch-plugin_amd", "examples", "paged_decode.py")


def example(plain=False, swapped=False):
    spec = importlib.util.spec_from_file_location("paged_decode", PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)

    class Plain(mod.PagedCache):
        def __init__(self, *args, **kw):
            super().__init__(*args, **kw)
            self.append, self.attention = self.plain_append, self.plain_attention

        def plain_append(self, q, k, v, pos, cos_sin, slots, kc, ks, vc, vs):
            held = slots >= 0
            at = slots[held] // self.size, slice(None), slots[held] % self.size
            rows = [R.rotary(k, pos, cos_sin, False)[0][held], v[held]]
            for x, codes, scales in zip(rows[::-1] if swapped else rows, (kc, vc), (ks, vs)):
                codes[at], scales[at] = M.quantise(x)
            return R.rotary(q, pos, cos_sin, False)[0].to(q.dtype)

        def plain_attention(self, q, kc, ks, vc, vs, table, cu, lens, max_query_len):
            return M.attention(q, (kc, ks, vc, vs), table, cu, lens)[0].to(q.dtype)

    if plain:
        mod.PagedCache = Plain
    return mod.run(mxfp4=True)


def test_the_example_in_4_bits_computes_its_definition():
    seqs, got, _, cache = example()
    same, want, _, other = example(plain=True)
    assert all(torch.equal(a, b) for a, b in zip(seqs, same))
    assert torch.equal(cache.table, other.table) and torch.equal(cache.lens, other.lens)
    rel = (got - want).norm(dim=1) / want.norm(dim=1)
    assert (rel < 0.05).all(), rel
    print("off by", rel.tolist())
    # the bound tells keys from values: with them exchanged in the definition it is passed
    _, wrong, _, _ = example(plain=True, swapped=True)
    assert ((got - wrong).norm(dim=1) / wrong.norm(dim=1) > 0.05).all()
