"""Attention over the cache held in 4 bits where items are whole and have several
tiles, the first or last of which a window or the causal border cuts: against the
references and bounds of test_kv_cache_mx4_gpu.py, again and again with the same bits."""
import pytest
import torch

import test_kv_cache_mx4_gpu as G

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 96, 104, 128, 256])
@pytest.mark.parametrize("window", [0, 1, 2, 16, 31, 65, 100])
def test_cut_tiles_of_whole_items(window, D, dtype):
    for i, lens in enumerate(([(130, 130)], [(1, 300), (40, 300), (130, 130), (1, 5)], [(130, 1300)], [(200, 200)] * 3)):
        b = G.make(lens, 8, 2, D, 16, dtype, seed=window + i)
        out = G.check(b, window=window)
        for _ in range(4):
            assert torch.equal(G.call(b, window=window), out)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [64, 129, 300, 513])
def test_whole_sequences(n, D, dtype):
    for causal in (True, False):
        for kv in (1, 4):
            b = G.make([(n, n)] * 2, kv, kv, D, 16, dtype, seed=n)
            out = G.check(b, causal=causal)
            assert torch.equal(G.call(b, causal=causal), out)
