"""What the ops of the cache held in 4 bits ask of the runtime, without a GPU (see
test_kv_cache_launch.py): LDS sizes and launches are recorded, and nothing runs."""
import json
import os
import subprocess
import sys
import textwrap

import test_kv_cache_launch as T

pytestmark = T.pytestmark

CALLS = """
import ctypes
import zt_mx4 as K
L, p = K.lib(), 256

def cache(dim, pages=4, heads=2, size=16, far=False):
    nb = (dim + 31) // 32
    st = (ctypes.c_int64 * 3)(heads * size * 16 * nb, size * 16 * nb, 16 * nb)
    sc = (ctypes.c_int64 * 3)(heads * size * nb, size * nb, nb)
    other = (ctypes.c_int64 * 3)(2 * heads * size * nb, size * nb, nb)
    return K.KvCacheMxfp4(p, p, p, p, pages, heads, size, dim, st, st, sc, other if far else sc)

def attend(dtype, dim, S, max_q, far=False, T=4000, H=8, W=500):
    c = cache(dim, far=far)
    ws = L.zt_paged_attention_mxfp4_workspace_size(T, H, dtype, ctypes.byref(c), S, W, max_q)
    rc = L.zt_paged_attention_mxfp4(p, dtype, T, H, H * dim, dim, ctypes.byref(c), p, S, W, p, p, max_q, 1, 0, 0.1,
                                    p << 20, p << 24, ws, None)
    assert rc == 0, L.zt_last_error_string()
"""


def record(tmp_path, calls):
    src, lib = tmp_path / "recorder.c", tmp_path / "recorder.so"
    src.write_text(T.RECORDER)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-o", lib, src], check=True)
    preload = ":".join(x for x in (str(lib), os.environ.get("LD_PRELOAD")) if x)
    out = subprocess.run([sys.executable, "-c", CALLS + textwrap.dedent(calls)], stdout=subprocess.PIPE,
                         stderr=subprocess.PIPE, text=True, timeout=120,
                         env=dict(os.environ, PYTHONPATH=T.HERE, LD_PRELOAD=preload))
    assert out.returncode == 0, out.stderr
    return [json.loads(line) for line in out.stdout.splitlines() if line.startswith("[")]


def test_lds_sizes_do_not_depend_on_the_call(tmp_path):
    got = record(tmp_path, """
        for dtype in (0, 1):
            for dim in (64, 80, 128, 256):
                for max_q in (1, 500):
                    for far in (False, True):
                        for S in (1, 1024, 700, 1):
                            attend(dtype, dim, S, max_q, far)
    """)
    allowed, largest, last = {}, {}, {}
    for kind, f, *rest in got:
        if kind == "allow":
            allowed.setdefault(f, set()).add(rest[1])
            last[f] = rest[1]
        else:
            largest[f] = max(largest.get(f, 0), rest[4])
            assert rest[4] <= 64 * 1024 or rest[4] <= last[f]
            assert rest[4] <= 160 * 1024
    assert len(allowed) >= 4 and all(len(v) == 1 for v in allowed.values()), allowed
    assert all(largest[f] == max(v) for f, v in allowed.items())


def test_launches_stay_below_two_to_the_31_threads(tmp_path):
    """A thread's number is divided in 31 bits, so longer calls are several launches."""
    got = record(tmp_path, """
        T, c = (1 << 20) + 5, cache(128, heads=16)
        for rot in (128, 32, 2):
            st = (ctypes.c_int64 * 2)(64 * 128, 128)
            rc = L.zt_rotary_cache_append_mxfp4(p, 1, T, 32, st, p, st, p, st, p, p, 2, rot, 128, 0, p,
                                                ctypes.byref(c), 1 << 50, None)
            assert rc == 0, L.zt_last_error_string()
        rc = L.zt_cache_read_mxfp4(ctypes.byref(c), p, (1 << 23) + 3, 1, 1 << 50, 1 << 51, None)
        assert rc == 0, L.zt_last_error_string()
    """)
    threads = {}
    for kind, f, x, y, z, block, lds in got:
        assert kind == "launch" and x * block < 1 << 31
        threads.setdefault(f, []).append(x * block)
    T_ = (1 << 20) + 5
    pair = T_ * (32 * 8 + 16 * 8 + 16 * 16)   # a thread to eight elements of each half
    wide = T_ * (32 * 16 + 2 * 16 * 16)       # or to eight elements
    read = ((1 << 23) + 3) * 16 * 16
    for got_, want in zip(threads.values(), (pair, wide, wide, read)):
        assert want <= sum(got_) < want + 256 * len(got_)
