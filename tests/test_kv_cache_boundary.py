"""CPU checks of the paged-cache ops: what the C-ABI and the torch ops refuse,
and the Meta kernels.  No GPU compute is called here."""
import ctypes

import pytest
import torch

import zentorch  # noqa: F401
import zt_kv as K

ops = torch.ops.zentorch
I32 = torch.int32


def err(rc):
    return rc, K.lib().zt_last_error_string().decode()


def cache(dtype=1, pages=4, heads=2, size=16, dim=64, k=None, v=None, strides=None):
    st = strides or (heads * size * dim, size * dim, dim)
    return K.KvCache(k, v, dtype, pages, heads, size, dim, (ctypes.c_int64 * 3)(*st),
                     (ctypes.c_int64 * 3)(*st))


def attn(c, T=4, H=4, S=1, W=4, max_q=4, causal=1, window=0, scale=0.1, ptr=256, ld=(256, 64), ws=None):
    return err(K.lib().zt_paged_attention(ptr, T, H, ld[0], ld[1], ctypes.byref(c), ptr, S, W, ptr, ptr,
                                          max_q, causal, window, scale, ptr, ws, 0, None))


@pytest.mark.parametrize("kw,code,word", [
    (dict(H=3), 1, "multiple of the cache's"), (dict(window=-1), 1, "window"),
    (dict(causal=0, window=4), 1, "window"), (dict(max_q=-1), 1, "max_query_len"),
    (dict(T=-1), 1, "T, S, W"), (dict(scale=float("nan")), 1, "finite"),
    (dict(ptr=None), 1, "null"), (dict(S=5000), 2, "sequences"), (dict(W=1 << 27), 2, "table of"),
    (dict(ld=(255, 64)), 2, "16-byte"),
])
def test_attention_refusals(kw, code, word):
    rc, msg = attn(cache(k=256, v=256), **kw)
    assert rc == code and word in msg, (rc, msg)


@pytest.mark.parametrize("c,code,word", [
    (dict(dtype=2), 1, "bf16 or fp32"), (dict(dim=60), 2, "multiple of 8"),
    (dict(dim=264), 2, "up to 256"), (dict(size=0), 1, "page_size"), (dict(pages=-1), 1, "pages"),
    (dict(strides=(1, -1, 1)), 1, "negative"), (dict(k=None, v=None), 1, "null"),
    (dict(k=260), 2, "16-byte"), (dict(strides=(2048, 1024, 60)), 2, "16-byte"),
])
def test_attention_cache_refusals(c, code, word):
    rc, msg = attn(cache(**dict(dict(k=256, v=256), **c)))
    assert rc == code and word in msg, (rc, msg)


def test_attention_of_no_tokens_is_nothing():
    assert attn(cache(), T=0, ptr=None)[0] == 0


def test_rotary_refusals():
    L = K.lib()

    def call(dtype=1, T=4, H=2, D=64, R=64, ld=64, length=10, ptr=256):
        return err(L.zt_rotary_embedding(ptr, dtype, T, H, D, 128, 64, ptr, ptr, length, R, ld, 0, ptr, None))

    for kw, word in ((dict(dtype=2), "bf16 or fp32"), (dict(R=63), "even"), (dict(R=66), "at most"),
                     (dict(R=0), "even"), (dict(ld=32), "row stride"), (dict(T=-1), "T >= 0"),
                     (dict(ptr=None), "null"), (dict(H=0), "heads")):
        rc, msg = call(**kw)
        assert rc == 1 and word in msg, (kw, rc, msg)
    assert call(T=1 << 40)[0] == 2
    assert call(T=0, ptr=None)[0] == 0


def test_page_refusals():
    L = K.lib()
    p = 256

    def extend(S=2, W=4, pages=8, size=16, T=2, ptr=p):
        return err(L.zt_cache_extend(ptr, ptr, ptr, ptr, S, W, pages, size, T, ptr, ptr, ptr, ptr, ptr, None))

    assert extend(size=0)[0] == 1 and extend(S=-1)[0] == 1 and extend(ptr=None)[0] == 1
    assert extend(S=5000)[0] == 2 and extend(W=1 << 24, size=1 << 12)[0] == 2

    def fork(S=2, W=4, pages=8, size=16, ptr=p):
        return err(L.zt_cache_fork(ptr, ptr, ptr, ptr, S, W, pages, size, ptr, ptr, ptr, ptr, None))

    assert fork(size=0)[0] == 1 and fork(pages=-1)[0] == 1 and fork(ptr=None)[0] == 1
    assert fork(S=5000)[0] == 2
    rc, msg = err(L.zt_cache_compact(p, 4, p, 8, p, p, p, None, 0, None))
    assert rc == 1 and "workspace" in msg
    assert L.zt_cache_compact_workspace_size(0) == 0
    arr = (ctypes.c_void_p * 1)(p)
    assert err(L.zt_cache_copy_pages(arr, 1, 8, 1024, 512, p, 2, None))[0] == 1   # pages overlap
    assert err(L.zt_cache_copy_pages(arr, 1, 8, 1024, 1024, None, 2, None))[0] == 1
    arr[0] = None
    assert err(L.zt_cache_copy_pages(arr, 1, 8, 1024, 1024, p, 2, None))[0] == 1
    assert err(L.zt_cache_copy_pages(None, 0, 8, 1024, 1024, None, 2, None))[0] == 0


def test_cpu_tensors_are_refused():
    x, t = torch.randn(2, 2, 64).bfloat16(), torch.randn(8, 64)
    with pytest.raises(NotImplementedError):
        ops.zentorch_rotary_embedding(x, torch.zeros(2, dtype=torch.int64), t)
    kv = torch.zeros(4, 2, 16, 64).bfloat16()
    one = torch.zeros(1, dtype=I32)
    with pytest.raises(NotImplementedError):
        ops.zentorch_paged_attention(x, kv, kv, torch.zeros(1, 4, dtype=I32), torch.zeros(2, dtype=I32), one, 2)
    with pytest.raises(NotImplementedError):
        ops.zentorch_cache_extend(torch.zeros(1, 4, dtype=I32), one, one, torch.zeros(2, dtype=I32), 16, 0)


def test_meta():
    m = dict(device="meta")
    q = torch.empty(5, 8, 64, dtype=torch.bfloat16, **m)
    kv = torch.empty(9, 2, 16, 64, dtype=torch.bfloat16, **m)
    table, ctx = torch.empty(3, 4, dtype=I32, **m), torch.empty(3, dtype=I32, **m)
    cu, pos = torch.empty(4, dtype=I32, **m), torch.empty(5, dtype=torch.int64, **m)
    cs = torch.empty(100, 32, **m)
    k = torch.empty(5, 2, 64, dtype=torch.bfloat16, **m)
    assert ops.zentorch_rotary_embedding(q, pos, cs).shape == q.shape
    assert ops.zentorch_rotary_cache_append(q, k, k, pos, cs, pos, kv, kv).shape == q.shape
    o = ops.zentorch_paged_attention(q, kv, kv, table, cu, ctx, 3)
    assert o.shape == q.shape and o.dtype == q.dtype
    refs = torch.empty(9, dtype=I32, **m)
    got = ops.zentorch_cache_extend(table, ctx, refs, cu, 16, 5)
    assert [tuple(t.shape) for t in got] == [(3, 4), (3,), (9,), (5,), (5,)]
    assert got[3].dtype == torch.int64
    got = ops.zentorch_cache_fork(table, ctx, refs, ctx, 16)
    assert [tuple(t.shape) for t in got] == [(3, 4), (3,), (9,), (3, 2)]
    got = ops.zentorch_cache_compact(table, refs)
    assert [tuple(t.shape) for t in got] == [(3, 4), (9,), (4, 2)]
    assert ops.zentorch_cache_copy_pages([kv, kv], got[2]) is None
