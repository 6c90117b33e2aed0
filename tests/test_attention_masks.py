"""The attention kernels' listings: where the lanes that a branch left out return, no
vector instruction of the same block stands before that.  The compiler has put a
move there (of a register that overflowed into an accumulation register) that then
was made for some lanes only, and the others went on with what was there before.
It showed in fp32 at head_dim 128 where a whole item has several tiles and the first
is cut by a window (test_kv_cache_mx4_windows_gpu.py).  No GPU is needed."""
import concurrent.futures
import os
import re
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "zendnn-pytorch-plugin_amd"))
import build  # noqa: E402

SOURCES = ["paged_attn.hip", "paged_attn_tile.hip", "paged_attn_split.hip", "paged_attn_mx4.hip",
           "paged_attn_mx4_tile.hip"]
VECTOR = re.compile(r"(v_(?!readlane|writelane|readfirstlane|nop)|ds_|global_|buffer_|scratch_|flat_)")
ENDS = re.compile(r"s_(cbranch|branch|and_saveexec|andn2_saveexec|endpgm|setpc)|s_\w+\s+exec,")
BACK = re.compile(r"s_or_b64\s+exec,\s*exec,")


def early(listing):
    """(kernel, instruction) of every one before its block's lanes return."""
    kernel, found, before = None, [], []
    for line in listing.split("\n"):
        name = re.match(r"([A-Za-z_]\w*):", line)
        if name or re.match(r"\.LBB\d+_\d+:|;\s*%bb\.\d+:", line):
            kernel, before = name[1] if name else kernel, []
            continue
        ins = line.split(";")[0].strip()
        if not ins or ins.startswith(".") or before is None:
            continue
        if BACK.match(ins):
            found += [(kernel, i) for i in before if VECTOR.match(i)]
            before = None
        elif ENDS.match(ins):
            before = None
        else:
            before.append(ins)
    return found


def test_the_search_finds_it():
    good = "k:\n\ts_and_saveexec_b64 s[2:3], vcc\n; %bb.1:\n\tv_mov_b32 v1, v2\n.LBB0_2:\n\ts_or_b64 exec, exec, s[2:3]\n"
    bad = good.replace("\ts_or", "\tv_accvgpr_write_b32 a3, v7 ; copy\n\ts_mov_b64 s[4:5], 0\n\ts_or")
    assert early(good) == [] and early(bad) == [("k", "v_accvgpr_write_b32 a3, v7")]


@pytest.fixture(scope="module")
def listings(tmp_path_factory):
    out = tmp_path_factory.mktemp("listings")

    def one(src):
        to = str(out / (src + ".s"))
        build._run([build.HIPCC] + build.HIP_FLAGS + ["-S", "--cuda-device-only", os.path.join(build.CSRC, src), "-o", to],
                   False)
        return open(to).read()

    with concurrent.futures.ThreadPoolExecutor(len(SOURCES)) as ex:
        return dict(zip(SOURCES, ex.map(one, SOURCES)))


@pytest.mark.parametrize("source", SOURCES)
def test_lanes_are_back_first(source, listings):
    text = listings[source]
    assert len(re.findall(r"^_Z\w+:", text, re.M)) >= 2 and "s_or_b64 exec" in text
    assert early(text) == []
