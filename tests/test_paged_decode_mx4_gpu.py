"""The paged decoding example over a cache held in 4 bits: that it runs, and that
its pages are where the other cache's are.  (What the ops compute is checked in
test_kv_cache_mx4_gpu.py; the logits' distance from exact ones is the format's.)"""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "zendnn-pytorch-plugin_amd", "examples", "paged_decode.py")


def test_paged_decode_example_in_4_bits():
    spec = importlib.util.spec_from_file_location("paged_decode", PATH)
    M = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(M)
    seqs, got, want, cache = M.run(mxfp4=True)
    assert [len(s) for s in seqs] == [43, 43, 70, 43]
    assert got.shape == want.shape and torch.isfinite(got).all()
    assert torch.equal(cache.lens.cpu(), torch.tensor([43, 43, 70, 43], dtype=torch.int32))
    assert sorted(cache.refs[cache.refs > 0].tolist()) == [1] * 8 + [3] * 2
    print("logits off by", ((got - want).norm() / want.norm()).item(), "of their norm")
