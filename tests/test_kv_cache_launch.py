"""What the paged-cache ops ask of the runtime, without a GPU: a small library in
the runtime's place (LD_PRELOAD, in a process of its own) records the LDS sizes
and the launches, and runs nothing."""
import json
import os
import shutil
import subprocess
import sys
import textwrap

import pytest
import torch

pytestmark = [pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc"),
              pytest.mark.skipif(torch.cuda.is_available(), reason="the calls' addresses are made up")]
HERE = os.path.dirname(os.path.abspath(__file__))

RECORDER = r"""
#include <stddef.h>
#include <stdint.h>
#include <stdio.h>
typedef struct { uint32_t x, y, z; } dim3_t;
int hipFuncSetAttribute(const void *f, int attr, int value) {
  printf("[\"allow\", %zu, %d, %d]\n", (size_t)f, attr, value);
  fflush(stdout);
  return 0;
}
int hipLaunchKernel(const void *f, dim3_t g, dim3_t b, void **args, size_t lds, void *stream) {
  printf("[\"launch\", %zu, %u, %u, %u, %u, %zu]\n", (size_t)f, g.x, g.y, g.z, b.x * b.y * b.z, lds);
  fflush(stdout);
  return 0;
}
static struct { dim3_t g, b; size_t lds; void *stream; } call;
int __hipPushCallConfiguration(dim3_t g, dim3_t b, size_t lds, void *stream) {
  call.g = g, call.b = b, call.lds = lds, call.stream = stream;
  return 0;
}
int __hipPopCallConfiguration(dim3_t *g, dim3_t *b, size_t *lds, void **stream) {
  *g = call.g, *b = call.b, *lds = call.lds, *stream = call.stream;
  return 0;
}
int hipGetLastError(void) { return 0; }
"""

CALLS = """
import ctypes
import zt_kv as K
L, p = K.lib(), 256

def cache(dtype, dim, pages=4, heads=2, size=16):
    st = (ctypes.c_int64 * 3)(heads * size * dim, size * dim, dim)
    return K.KvCache(p, p, dtype, pages, heads, size, dim, st, st)

def attend(dtype, dim, S, max_q, T=4000, H=8, W=500):
    c = cache(dtype, dim)
    ws = L.zt_paged_attention_workspace_size(T, H, ctypes.byref(c), S, W, max_q)
    rc = L.zt_paged_attention(p, T, H, H * dim, dim, ctypes.byref(c), p, S, W, p, p, max_q, 1, 0, 0.1, p << 20,
                              p << 24, ws, None)
    assert rc == 0, L.zt_last_error_string()

def fork(S):
    rc = L.zt_cache_fork(p, p, p, p, S, 4, 8, 16, p << 20, p << 21, p << 22, p << 23, None)
    assert rc == 0, L.zt_last_error_string()
"""


def record(tmp_path, calls):
    src, lib = tmp_path / "recorder.c", tmp_path / "recorder.so"
    src.write_text(RECORDER)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-o", lib, src], check=True)
    # the recorder's functions stand in front of the runtime's
    preload = ":".join(p for p in (str(lib), os.environ.get("LD_PRELOAD")) if p)
    p = subprocess.run([sys.executable, "-c", CALLS + textwrap.dedent(calls)], stdout=subprocess.PIPE,
                       stderr=subprocess.PIPE, text=True, timeout=120,
                       env=dict(os.environ, PYTHONPATH=HERE, LD_PRELOAD=preload))
    assert p.returncode == 0, p.stderr
    return [json.loads(line) for line in p.stdout.splitlines() if line.startswith("[")]


def test_lds_sizes_do_not_depend_on_the_call(tmp_path):
    """A kernel that needs more than 64 KB of LDS is allowed one size, its
    largest: two threads' calls of different sizes cannot take it from each other."""
    got = record(tmp_path, """
        for dtype in (0, 1):
            for dim in (64, 80, 128, 256):
                for max_q in (1, 500):
                    for S in (1, 1024, 700, 1):
                        attend(dtype, dim, S, max_q)
        for S in (4096, 1, 3000):
            fork(S)
    """)
    allowed, largest, last = {}, {}, {}
    for kind, f, *rest in got:
        if kind == "allow":
            allowed.setdefault(f, set()).add(rest[1])
            last[f] = rest[1]
        else:
            largest[f] = max(largest.get(f, 0), rest[4])
            assert rest[4] <= 64 * 1024 or rest[4] <= last[f]
    assert len(allowed) >= 8 and all(len(v) == 1 for v in allowed.values()), allowed
    assert all(largest[f] == max(v) for f, v in allowed.items())


def test_launches_stay_below_two_to_the_32_threads(tmp_path):
    """The runtime leaves out what is past 2^32 threads of a launch, so longer
    calls are several launches."""
    got = record(tmp_path, """
        rc = L.zt_rotary_embedding(p, 1, (1 << 20) + 5, 32, 130, 32 * 130, 130, p, p, 2, 2, 2, 0, p << 20, None)
        assert rc == 0, L.zt_last_error_string()
        c = cache(1, 130, heads=16)
        st = (ctypes.c_int64 * 2)(64 * 130, 130)
        rc = L.zt_rotary_cache_append(p, (1 << 20) + 5, 32, st, p, st, p, st, p, p, 2, 2, 2, 1, p, ctypes.byref(c),
                                      p << 20, None)
        assert rc == 0, L.zt_last_error_string()
        caches = (ctypes.c_void_p * 70)(*[p] * 70)
        for n, size in (((1 << 24) + 3, 64), (1 << 20, 1 << 20)):
            rc = L.zt_cache_copy_pages(caches, 70, 1 << 25, size, size, p, n, None)
            assert rc == 0, L.zt_last_error_string()
    """)
    threads = {}  # by kernel, in the order of the calls
    for kind, f, x, y, z, block, lds in got:
        assert kind == "launch" and x * block < 1 << 32
        threads[f] = threads.get(f, 0) + x * y * z * block
    T, row = (1 << 20) + 5, 129  # a head row is a pair and 128 single elements
    rotary, append = T * 32 * row, T * (48 * row + 16 * 130)
    copies = 256 * 70 * ((1 << 24) + 3 + 64 * (1 << 20))  # 64 workgroups copy a page of 2^20 bytes
    got = list(threads.values())
    assert rotary <= got[0] < rotary + 3 * 256 and append <= got[1] < append + 5 * 256 and got[2:] == [copies]
