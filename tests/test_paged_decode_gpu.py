"""The paged decoding example: quantised linears with the paged cache between
them, against a cacheless recomputation in fp32.  Activations are bf16 (half a
step 2^-8) at some ten places of two layers, so the logits may be off by 2^-8
times the root of those roundings, 3 %; a wrong page, position or mask gives
logits of another sequence, off by more than their norm."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "zendnn-pytorch-plugin_amd", "examples", "paged_decode.py")


def test_paged_decode_example():
    spec = importlib.util.spec_from_file_location("paged_decode", PATH)
    M = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(M)
    seqs, got, want, cache = M.run()
    assert [len(s) for s in seqs] == [43, 43, 70, 43]
    assert len({tuple(s.tolist()) for s in seqs}) == 4  # three continuations of row 0
    rel = (got - want).norm(dim=1) / want.norm(dim=1)
    assert (rel < 0.03).all(), rel
    assert torch.equal(cache.lens.cpu(), torch.tensor([43, 43, 70, 43], dtype=torch.int32))
    # 37 + 3 tokens at the fork: two full pages are shared by three rows; each
    # has a last page of its own, and row 2 has five
    assert sorted(cache.refs[cache.refs > 0].tolist()) == [1] * 8 + [3] * 2
