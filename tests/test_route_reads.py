"""The choice of experts reads its logits and its bias, and nothing that it has not written: of its two outputs neither is
ever read, not even for a value that is thrown away (other blocks are writing them)."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lockstep_amd", "csrc")


def test_outputs_are_only_written():
    src = open(os.path.join(CSRC, "route.hip")).read()
    kernel = src[src.index("void route_kernel("):src.index('extern "C" int lsk_route_experts')]
    assert re.findall(r"[^\n]*\bp\.idx\b[^\n]*", kernel) == ["    p.idx[o] = expert;"]
    assert all("[o] = " in line or "store_out(p.w" in line for line in re.findall(r"[^\n]*\bp\.w\b[^\n]*", kernel))
