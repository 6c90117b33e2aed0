"""Outputs of the paged-cache ops that overlap an input or another output are
refused by the C-ABI, before anything is launched.  No GPU is needed: a call
whose arrays are apart fails only at its launch here."""
import ctypes

import pytest
import torch

import zt_kv as K

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="the calls' addresses are made up")
MB = 1 << 20
S, W, PAGES, T = 8, 16, 64, 12


def err(rc):
    return rc, K.lib().zt_last_error_string().decode()


def extend(p):
    return err(K.lib().zt_cache_extend(*p[:4], S, W, PAGES, 16, T, *p[4:], None))


def fork(p):
    return err(K.lib().zt_cache_fork(*p[:4], S, W, PAGES, 16, *p[4:], None))


def compact(p):
    return err(K.lib().zt_cache_compact(p[0], S * W, p[1], PAGES, p[2], p[3], p[4], p[5], PAGES * 4, None))


# bytes of each array, and how many of them are inputs
OPS = [(extend, [S * W * 4, S * 4, PAGES * 4, (S + 1) * 4, S * W * 4, S * 4, PAGES * 4, T * 8, T * 8], 4),
       (fork, [S * W * 4, S * 4, PAGES * 4, S * 4, S * W * 4, S * 4, PAGES * 4, S * 8], 4),
       (compact, [S * W * 4, PAGES * 4, S * W * 4, PAGES * 4, PAGES * 4, PAGES * 4], 2)]


@pytest.mark.parametrize("op,sizes,inputs", OPS, ids=["extend", "fork", "compact"])
def test_page_ops(op, sizes, inputs):
    apart = [(i + 1) * MB for i in range(len(sizes))]
    rc, msg = op(apart)
    assert rc != 1, msg
    close = [MB + sum(sizes[:i]) for i in range(len(sizes))]  # end to end
    assert op(close)[0] != 1
    for out in range(inputs, len(sizes)):
        for other in range(out):
            for at in (apart[other], apart[other] + sizes[other] - 4, apart[other] - sizes[out] + 4):
                p = list(apart)
                p[out] = at
                rc, msg = op(p)
                assert rc == 1 and "overlap" in msg, (out, other, at - apart[other], rc, msg)
            for at in (apart[other] + sizes[other], apart[other] - sizes[out]):
                p = list(apart)
                p[out] = at
                assert op(p)[0] != 1


def attend(q, out, ws, T=4, H=4, D=64, ld=None):
    st = (ctypes.c_int64 * 3)(2 * 16 * D, 16 * D, D)
    c = K.KvCache(64 * MB, 96 * MB, 1, 4, 2, 16, D, st, st)
    ld = ld or (H * D, D)
    n = K.lib().zt_paged_attention_workspace_size(T, H, ctypes.byref(c), 1, 4, 4)
    return err(K.lib().zt_paged_attention(q, T, H, ld[0], ld[1], ctypes.byref(c), 256, 1, 4, 512, 1024, 4, 1, 0, 0.1,
                                          out, ws, n, None)) + (n,)


def test_attention():
    row = 4 * 64 * 2
    assert attend(16 * MB, 17 * MB, 32 * MB)[0] != 1
    n = attend(16 * MB, 17 * MB, 32 * MB)[2]
    for q, out, ws in ((16 * MB, 16 * MB, 32 * MB), (16 * MB, 16 * MB + 3 * row, 32 * MB),
                       (16 * MB, 16 * MB - 4 * row + 16, 32 * MB), (16 * MB, 32 * MB, 32 * MB),
                       (32 * MB, 17 * MB, 32 * MB), (32 * MB + n - 256, 17 * MB, 32 * MB)):
        rc, msg, _ = attend(q, out, ws)
        assert rc == 1 and "overlap" in msg, (q, out, ws, rc, msg)
    for out in (16 * MB + 4 * row, 16 * MB - 4 * row):
        assert attend(16 * MB, out, 32 * MB)[0] != 1
    # a slice of a wider buffer: the output may lie between two tokens' queries
    assert attend(16 * MB, 16 * MB + row, 32 * MB, T=2, ld=(3 * 4 * 64, 64))[0] != 1
    assert attend(16 * MB, 16 * MB + row + 16, 32 * MB, T=2, ld=(3 * 4 * 64, 64))[0] == 1
    assert attend(16 * MB, 16 * MB + row, 32 * MB, T=3, ld=(3 * 4 * 64, 64))[0] == 1
