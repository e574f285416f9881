"""What the kernels' sources have to keep to, checked without a GPU."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lfm3-1.7b-mi50_amd", "csrc")


@pytest.mark.parametrize("name", sorted(f for f in os.listdir(CSRC) if f.endswith((".hip", ".h"))))
def test_barriers_are_fenced(name):
    """The bare barrier builtin orders no memory access for the compiler and waits for no LDS read in flight: a hand-over of
    LDS between waves goes through common.h's ring_barrier / lds_barrier (or __syncthreads)."""
    text = open(os.path.join(CSRC, name)).read()
    text = re.sub(r"//[^\n]*", "", text)
    allowed = 1 if name == "common.h" else 0
    assert text.count("__builtin_amdgcn_s_barrier") == allowed
    if allowed:
        body = text[text.index("ring_barrier()"):]
        assert re.search(r's_waitcnt\(vmcnt_imm\(N\) & ~0x0F00\);\s*asm volatile\("" ::: "memory"\);\s*'
                         r'__builtin_amdgcn_s_barrier\(\);\s*asm volatile\("" ::: "memory"\);', body)


def helpers(text, param):
    """Bodies of the device functions that take `param`, by name."""
    for at in re.finditer(r"\b(\w+)\(([^()]*\b%s[^()]*)\) \{\n" % re.escape(param), text):
        depth, end = 1, at.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        yield at.group(1), text[at.end():end]


def test_sampling_helpers_return_behind_a_barrier():
    """What a wave reads of the words that the sampler's helpers share it has read before any wave returns: the caller's next helper writes
    the same words at once (a wave that is late would take another way through the barriers than the rest)."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "sample.hip")).read())
    seen = 0
    for name, body in helpers(text, "SampleShared& sh"):
        for at in re.finditer(r"return false;", body):
            seen += 1
            since = body[:at.start()].rsplit("__syncthreads();", 1)[-1]
            assert not re.search(r"\bsh\.", since), (name, since)
    assert seen >= 5
