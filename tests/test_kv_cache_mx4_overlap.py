"""Outputs and workspaces that lie on the cache, on its table or on another input are
refused by the C-ABI before anything is launched, and those between two rows of an
array are not.  No GPU is needed: a call whose arrays are apart fails only at its
launch here."""
import ctypes
import itertools
import random

import pytest
import torch

import zt_kv
import zt_mx4 as K

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="the calls' addresses are made up")
MB = 1 << 20
PAGES, KV, SIZE, D, T, H, S, W = 3, 2, 4, 32, 2, 4, 2, 3
SCALES, VALUES, INPUTS, FAR = 64 * MB, 128 * MB, 256 * MB, 1 << 40
LAYOUTS = {  # strides of page, head and token for rows of 16 bytes
    "hnd": (128, 64, 16), "nhd": (128, 16, 32), "holes": (1024, 256, 48), "tokens outermost": (32, 16, 96),
    "one page": (0, 64, 16), "pages on each other": (32, 64, 16)}


def rows(at, row, strides):
    return {at + p * strides[0] + h * strides[1] + t * strides[2] + b for p, h, t, b in
            itertools.product(range(PAGES), range(KV), range(SIZE), range(row))}


def err(rc):
    return rc, K.lib().zt_last_error_string().decode()


def c3(x):
    return (ctypes.c_int64 * 3)(*x)


def cache(strides, scale_strides):
    return K.KvCacheMxfp4(MB, VALUES, SCALES, SCALES + VALUES, PAGES, KV, SIZE, D, c3(strides), c3((128, 64, 16)),
                          c3(scale_strides), c3((8, 4, 1)))


def append(c, out):
    st, p = (ctypes.c_int64 * 2)(H * D, D), INPUTS
    return err(K.lib().zt_rotary_cache_append_mxfp4(p, 1, T, H, st, p + MB, st, p + 2 * MB, st, p + 3 * MB, p + 4 * MB, 8,
                                                    D, D, 0, p + 5 * MB, ctypes.byref(c), out, None))


def read(c, k_out, v_out):
    return err(K.lib().zt_cache_read_mxfp4(ctypes.byref(c), INPUTS, T, 1, k_out, v_out, None))


def attend(c, out, ws):
    p, L = INPUTS, K.lib()
    n = L.zt_paged_attention_mxfp4_workspace_size(T, H, 1, ctypes.byref(c), S, W, 1)
    return err(L.zt_paged_attention_mxfp4(p, 1, T, H, H * D, D, ctypes.byref(c), p + MB, S, W, p + 2 * MB, p + 3 * MB, 1,
                                          1, 0, 0.1, out, ws, n, None)) + (n,)


def attend16(strides, out, ws):
    """Over the cache in bf16: rows of 8 numbers, 16 bytes."""
    p, L = INPUTS, zt_kv.lib()
    e = c3([s // 2 for s in strides])
    c = zt_kv.KvCache(MB, VALUES, 1, PAGES, KV, SIZE, 8, e, e)
    n = L.zt_paged_attention_workspace_size(T, H, ctypes.byref(c), S, W, 1)
    return err(L.zt_paged_attention(p, T, H, H * 8, 8, ctypes.byref(c), p + MB, S, W, p + 2 * MB, p + 3 * MB, 1, 1, 0,
                                    0.1, out, ws, n, None)) + (n,)


def verdicts(call, at, nbytes, held, r):
    """call(address) is refused exactly where [address, + nbytes) meets a byte of held."""
    seen = set()
    lo, hi = min(held) - nbytes - 64, max(held) + 64
    for a in [16 * r.randint(lo // 16, hi // 16) for _ in range(60)] + [min(held) - nbytes, max(held) // 16 * 16 + 16]:
        rc, msg = call(a)[:2]
        meets = any(a <= x < a + nbytes for x in held)
        seen.add(meets)
        assert (rc == 1) == meets and (not meets or "overlap" in msg), (a - at, nbytes, rc, msg)
    assert seen == {False, True}


@pytest.mark.parametrize("name", LAYOUTS)
def test_outputs_on_codes(name):
    st, r = LAYOUTS[name], random.Random(1)
    c, held = cache(st, (8, 4, 1)), rows(MB, 16, st)
    n = T * KV * D * 2
    verdicts(lambda a: append(c, a), MB, T * H * D * 2, held, r)
    verdicts(lambda a: read(c, a, FAR), MB, n, held, r)
    verdicts(lambda a: read(c, FAR, a), MB, n, held, r)
    verdicts(lambda a: attend(c, a, FAR), MB, T * H * D * 2, held, r)
    verdicts(lambda a: attend(c, FAR, a), MB, attend(c, FAR, 2 * FAR)[2], held, r)
    verdicts(lambda a: attend16(st, a, FAR), MB, T * H * 8 * 2, held, r)
    verdicts(lambda a: attend16(st, FAR, a), MB, attend16(st, FAR, 2 * FAR)[2], held, r)


@pytest.mark.parametrize("st", [(8, 4, 1), (512, 256, 64), (2, 1, 1000)])
def test_outputs_on_scales(st):
    r = random.Random(2)
    c, held = cache((128, 64, 16), st), rows(SCALES, 1, st)
    verdicts(lambda a: append(c, a), SCALES, T * H * D * 2, held, r)
    verdicts(lambda a: read(c, FAR, a), SCALES, T * KV * D * 2, held, r)
    verdicts(lambda a: attend(c, a, FAR), SCALES, T * H * D * 2, held, r)


def test_outputs_on_values_and_their_scales():
    c = cache((128, 64, 16), (8, 4, 1))
    for at in (VALUES, SCALES + VALUES):
        assert append(c, at)[0] == read(c, at, FAR)[0] == read(c, FAR, at)[0] == attend(c, at, FAR)[0] == 1
        assert attend(c, FAR, at)[0] == 1
    assert attend16((128, 64, 16), VALUES, FAR)[0] == attend16((128, 64, 16), FAR, VALUES)[0] == 1


@pytest.mark.parametrize("at,nbytes", [(3, T * 8), (4, 8 * D * 4), (5, T * 8)])
def test_append_output_on_another_input(at, nbytes):
    c, at = cache((128, 64, 16), (8, 4, 1)), INPUTS + at * MB
    verdicts(lambda a: append(c, a), at, T * H * D * 2, range(at, at + nbytes), random.Random(3))


@pytest.mark.parametrize("at,nbytes", [(1, S * W * 4), (2, (S + 1) * 4), (3, S * 4)])
def test_attention_output_on_another_input(at, nbytes):
    c, at, r = cache((128, 64, 16), (8, 4, 1)), INPUTS + at * MB, random.Random(4)
    held = range(at, at + nbytes)
    verdicts(lambda a: attend(c, a, FAR), at, T * H * D * 2, held, r)
    verdicts(lambda a: attend(c, FAR, a), at, attend(c, FAR, 2 * FAR)[2], held, r)
    verdicts(lambda a: attend16((128, 64, 16), a, FAR), at, T * H * 8 * 2, held, r)
    verdicts(lambda a: attend16((128, 64, 16), FAR, a), at, attend16((128, 64, 16), FAR, 2 * FAR)[2], held, r)


def test_large_strides():
    """Sizes whose products pass 64 bits end in an answer, not in a wrapped one."""
    big = (1 << 61, 1 << 60, 16)
    c = K.KvCacheMxfp4(MB, VALUES, SCALES, SCALES + VALUES, 1 << 30, 1 << 10, 1 << 20, D, c3(big), c3(big), c3(big),
                       c3(big))
    n = T * 1024 * D * 2  # of an output
    assert read(c, 2 * MB, FAR)[0] == read(c, MB - 256, FAR)[0] == 1 and read(c, MB - n, FAR)[0] != 1
