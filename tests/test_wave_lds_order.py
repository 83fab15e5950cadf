"""Where lanes of a wave hand values to one another through LDS without a barrier, wave_lds_fence() stands between the
writes and the reads, and where they do so again between the reads and the next writes.

The hardware runs a wave's own LDS operations in order, but the compiler sees the addresses of one lane: in store_groups a
lane writes 8 bytes at 32 lane + 8 t and reads them at 8 lane + 512 t, which never meet within a lane for most t, so that
it may put such a read ahead of the writes of other lanes that it is there for."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lockstep_amd", "csrc")

# file, the function, its last write, its first read, whether it writes again
PLACES = [("norm_fp8.hip", "store_groups", r"mine\[t\] = ", r"\(const uint64_t\*\)strip\)\[u\]", True),
          ("fp8.hip", "fp8_tile_out", r"\*\(v4f\*\)\(strip ", r"\*\(const v4f\*\)\(strip ", True),
          ("fp4.hip", "fp4_tile_kernel", r"\*\(v4f\*\)\(strip ", r"\*\(const v4f\*\)\(strip ", True),
          ("route.hip", "route_kernel", r"values\[wave\]\[lane \+ 64 \* j\] = ", r"kept_groups\(p, values\[wave\]\)", False)]


@pytest.mark.parametrize("name,function,write,read,again", PLACES, ids=[p[1] for p in PLACES])
def test_fences(name, function, write, read, again):
    src = open(os.path.join(CSRC, name)).read()
    start = re.search(r"\bvoid %s\(" % function, src)
    body = src[start.end():src.index("\n}\n", start.end())]
    w, r = re.search(write, body), re.search(read, body)
    assert w and r and w.end() < r.start()
    assert body.count("wave_lds_fence();", w.end(), r.start()) == 1
    assert body.count("wave_lds_fence();", r.end()) == (1 if again else 0)


def test_the_fence_is_one_for_the_compiler():
    src = open(os.path.join(CSRC, "lsk_common.h")).read()
    assert 'void wave_lds_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }' in src
