"""The .aligned forms of the warp-wide instructions need the whole warp at them, together.
Which lanes get there first is the compiler's choice after a branch of some of them (one
thread sets the barriers up, lanes wait or load different numbers of times), so the
wrappers of these instructions join the warp themselves."""
import os
import re

import pytest

from conftest import REPO

CSRC = os.path.join(REPO, "parakeet-streaming_b200", "csrc")
WIDE = re.compile(r"tcgen05\.(alloc|dealloc|ld|st)\.|bar\.red\.")


def wrappers():
    for name in ("pk_umma.cuh", "pk_tree_attn_tc.cu"):
        text = open(os.path.join(CSRC, name)).read()
        for m in re.finditer(r"__device__ __forceinline__ [\w ]+?\b(\w+)\([^)]*(?:\([^)]*\))?[^{;]*\) ?\{", text):
            body = text[m.end():text.index("\n}", m.end())]
            if WIDE.search(body):
                yield name, m.group(1), body


def test_there_are_wrappers():
    assert {n for _, n, _ in wrappers()} >= {
        "tmem_alloc", "tmem_dealloc", "tmem_alloc_pair", "tmem_dealloc_pair", "tmem_ld32",
        "tmem_st32", "tmem_ld_scores", "group_any"}


@pytest.mark.parametrize("file,name,body", list(wrappers()), ids=lambda x: x if len(x) < 40 else "")
def test_the_warp_is_joined_before(file, name, body):
    at = WIDE.search(body).start()
    assert "__syncwarp();" in body[:at], f"{file}: {name}"


def test_no_kernel_has_its_own():
    for name in sorted(os.listdir(CSRC)):
        text = open(os.path.join(CSRC, name)).read()
        for m in re.finditer(r"tcgen05\.(alloc|dealloc)\.", text):
            assert name == "pk_umma.cuh", name
