"""CPU checks of the cache held in 4 bits: what the C-ABI and the torch ops
refuse, and the Meta kernels.  No GPU compute is called here."""
import ctypes

import pytest
import torch

import zentorch  # noqa: F401
import zt_mx4 as K

ops = torch.ops.zentorch
I32, U8 = torch.int32, torch.uint8
FAR = 1 << 40  # an address nothing else here is near


def err(rc):
    return rc, K.lib().zt_last_error_string().decode()


def cache(pages=4, heads=2, size=16, dim=64, ptr=256, k=None, scales=256, strides=None, sc_strides=None):
    b, nb = (dim + 31) // 32 * 16, (dim + 31) // 32
    st = (ctypes.c_int64 * 3)(*(strides or (heads * size * b, size * b, b)))
    sc = (ctypes.c_int64 * 3)(*(sc_strides or (heads * size * nb, size * nb, nb)))
    return K.KvCacheMxfp4(ptr if k is None else k, ptr, scales, scales, pages, heads, size, dim, st, st, sc, sc)


def attn(c, dtype=1, T=4, H=4, S=1, W=4, max_q=4, causal=1, window=0, scale=0.1, ptr=256, ld=(256, 64), ws=None,
         out=None, ws_bytes=0):
    return err(K.lib().zt_paged_attention_mxfp4(ptr, dtype, T, H, ld[0], ld[1], ctypes.byref(c) if c else None, ptr,
                                                S, W, ptr, ptr, max_q, causal, window, scale,
                                                ptr if out is None else out, ws, ws_bytes, None))


@pytest.mark.parametrize("kw,code,word", [
    (dict(H=3), 1, "multiple of the cache's"), (dict(window=-1), 1, "window"),
    (dict(causal=0, window=4), 1, "window"), (dict(max_q=-1), 1, "max_query_len"),
    (dict(T=-1), 1, "T, S, W"), (dict(scale=float("nan")), 1, "finite"), (dict(scale=float("inf")), 1, "finite"),
    (dict(ptr=None), 1, "null"), (dict(S=5000), 2, "sequences"), (dict(W=1 << 27), 2, "table of"),
    (dict(ld=(255, 64)), 2, "16-byte"), (dict(ptr=260), 2, "16-byte"), (dict(dtype=2), 1, "bf16 or fp32"),
    (dict(), 1, "workspace"), (dict(ws=FAR + 8, ws_bytes=1 << 40), 1, "aligned workspace"),
    (dict(ws=FAR, ws_bytes=100), 1, "workspace"), (dict(ws=FAR, ws_bytes=1 << 40), 1, "overlap"),
    (dict(out=FAR, ws=FAR, ws_bytes=1 << 40), 1, "overlap"), (dict(out=256 + 512, ws=FAR, ws_bytes=1 << 40), 1, "overlap"),
])
def test_attention_refusals(kw, code, word):
    rc, msg = attn(cache(), **kw)
    assert rc == code and word in msg, (rc, msg)


CACHES = [
    (dict(dim=60), 2, "multiple of 8"), (dict(dim=264), 2, "up to 256"), (dict(size=0), 1, "page_size"),
    (dict(pages=-1), 1, "pages"), (dict(heads=0), 1, "heads"), (dict(heads=1 << 17), 2, "65535"),
    (dict(strides=(1, -1, 1)), 1, "negative"), (dict(sc_strides=(1, 1, -1)), 1, "negative"),
    (dict(ptr=None), 1, "null"), (dict(scales=None), 1, "null"), (dict(k=264), 2, "16-byte"),
    (dict(strides=(1024, 512, 24)), 2, "16-byte"), (dict(pages=1 << 40), 2, "32 bits"),
]


@pytest.mark.parametrize("c,code,word", CACHES)
def test_cache_refusals(c, code, word):
    L, p = K.lib(), 256
    bad = cache(**c)
    rc, msg = attn(bad, H=2 * max(1, bad.heads))
    assert rc == code and word in msg, (rc, msg)
    st = (ctypes.c_int64 * 2)(512, 64)
    rc, msg = err(L.zt_rotary_cache_append_mxfp4(p, 1, 4, 4, st, p, st, p, st, p, p, 8, 8, 8, 0, p,
                                                 ctypes.byref(bad), FAR, None))
    assert rc == code and word in msg, (rc, msg)
    rc, msg = err(L.zt_cache_read_mxfp4(ctypes.byref(bad), p, 4, 1, FAR, 2 * FAR, None))
    assert rc == code and word in msg, (rc, msg)


def test_far_rows_are_refused():
    rc, msg = attn(cache(pages=1 << 20, strides=(1 << 20, 512, 32)))
    assert rc == 2 and "64 GB" in msg, (rc, msg)


def test_null_cache():
    L, st = K.lib(), (ctypes.c_int64 * 2)(512, 64)
    assert attn(None)[0] == 1
    assert err(L.zt_cache_read_mxfp4(None, 256, 4, 1, FAR, 2 * FAR, None))[0] == 1
    assert err(L.zt_rotary_cache_append_mxfp4(256, 1, 4, 4, st, 256, st, 256, st, 256, 256, 8, 8, 8, 0, 256, None,
                                              FAR, None))[0] == 1
    assert L.zt_paged_attention_mxfp4_workspace_size(4, 4, 1, None, 1, 4, 4) == 0


def test_append_refusals():
    L, p = K.lib(), 256

    def call(dtype=1, T=4, H=4, R=64, ld=64, length=10, ptr=p, out=FAR, strides=(512, 64), c=None):
        st = (ctypes.c_int64 * 2)(*strides) if strides else None
        c = c or cache()
        return err(L.zt_rotary_cache_append_mxfp4(ptr, dtype, T, H, st, ptr, st, ptr, st, ptr, ptr, length, R, ld, 0,
                                                  ptr, ctypes.byref(c), out, None))

    for kw, code, word in ((dict(dtype=2), 1, "bf16 or fp32"), (dict(R=63), 1, "even"), (dict(R=66), 1, "at most"),
                           (dict(R=0), 1, "even"), (dict(ld=32), 1, "row stride"), (dict(T=-1), 1, "T >= 0"),
                           (dict(ptr=None), 1, "null"), (dict(H=0), 1, "heads"), (dict(strides=None), 1, "strides"),
                           (dict(H=1 << 20), 2, "heads"), (dict(T=1 << 62), 2, "too many"), (dict(out=p + 512), 1, "overlaps")):
        rc, msg = call(**kw)
        assert rc == code and word in msg, (kw, rc, msg)
    assert call(T=0, ptr=None, out=None)[0] == 0


def test_read_refusals():
    L, c = K.lib(), cache()

    def call(n=4, dtype=1, slots=256, k=FAR, v=2 * FAR):
        return err(L.zt_cache_read_mxfp4(ctypes.byref(c), slots, n, dtype, k, v, None))

    for kw, code, word in ((dict(n=-1), 1, "n >= 0"), (dict(dtype=3), 1, "bf16 or fp32"), (dict(slots=None), 1, "null"),
                           (dict(k=None), 1, "null"), (dict(v=None), 1, "null"), (dict(k=FAR + 8), 2, "alignment"),
                           (dict(v=FAR + 16), 1, "overlap"), (dict(slots=FAR + 8), 1, "overlaps an input"),
                           (dict(n=1 << 62), 2, "too many")):
        rc, msg = call(**kw)
        assert rc == code and word in msg, (kw, rc, msg)
    assert call(n=0, slots=None, k=None, v=None)[0] == 0


def test_attention_of_no_tokens_is_nothing():
    assert attn(cache(ptr=None, scales=None), T=0, ptr=None)[0] == 0


def test_cpu_tensors_are_refused():
    x = torch.randn(2, 2, 64).bfloat16()
    kc, ks = torch.zeros(4, 2, 16, 32, dtype=U8), torch.zeros(4, 2, 16, 2, dtype=U8)
    one, pos = torch.zeros(1, dtype=I32), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(NotImplementedError):
        ops.zentorch_paged_attention_mxfp4(x, kc, ks, kc, ks, torch.zeros(1, 4, dtype=I32),
                                           torch.zeros(2, dtype=I32), one, 2)
    with pytest.raises(NotImplementedError):
        ops.zentorch_rotary_cache_append_mxfp4(x, x, x, pos, torch.randn(8, 64), pos, kc, ks, kc.clone(), ks.clone())
    with pytest.raises(NotImplementedError):
        ops.zentorch_cache_read_mxfp4(kc, ks, kc, ks, pos, 64)


def test_meta():
    m = dict(device="meta")
    q = torch.empty(5, 8, 80, dtype=torch.bfloat16, **m)
    k = torch.empty(5, 2, 80, dtype=torch.bfloat16, **m)
    c = [torch.empty(9, 2, 16, n, dtype=U8, **m) for n in (48, 3, 48, 3)]
    table, ctx = torch.empty(3, 4, dtype=I32, **m), torch.empty(3, dtype=I32, **m)
    cu, pos = torch.empty(4, dtype=I32, **m), torch.empty(5, dtype=torch.int64, **m)
    out = ops.zentorch_rotary_cache_append_mxfp4(q, k, k, pos, torch.empty(100, 32, **m), pos, *c)
    assert out.shape == q.shape and out.dtype == q.dtype
    out = ops.zentorch_paged_attention_mxfp4(q, *c, table, cu, ctx, 3)
    assert out.shape == q.shape and out.dtype == q.dtype
    for dtype in (torch.bfloat16, torch.float32):
        got = ops.zentorch_cache_read_mxfp4(*c, pos, 80, dtype=dtype)
        assert [(tuple(t.shape), t.dtype) for t in got] == [((5, 2, 80), dtype)] * 2
    assert ops.zentorch_cache_read_mxfp4(*c, pos, 80)[0].dtype == torch.bfloat16
