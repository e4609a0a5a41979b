"""CPU checks of the token mixers' source, for what no run can show: a kernel that reads past its shared memory or leaves
out an ordering fence may give the right answer all the same."""
from __future__ import annotations

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wzy-flash-serve_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name,kernels", [("gdn_delta.cu", 2), ("kv_attn.cu", 1)])
def test_dynamic_shared_memory_is_one_struct(name, kernels):
    """A kernel's dynamic shared memory is one struct at its start, and a launch asks for the size of such a struct: then
    nothing of the layout can lie outside what was asked for."""
    text = source(name)
    buffers = re.findall(r"extern __shared__ [^;]*?(\w+)\[\];", text)
    assert len(buffers) == kernels
    for buffer in set(buffers):
        uses = [line.strip() for line in text.splitlines() if re.search(rf"\b{buffer}\b", line) and "extern" not in line]
        assert len(uses) == buffers.count(buffer), uses
        for line in uses:
            assert re.fullmatch(rf"(.+)& sm = \*reinterpret_cast<\1\*>\({buffer}\);", line), line
    for size in re.findall(r"\w+_smem = (.{40})", text):
        assert re.match(r"\(int\)sizeof\(\w+<T, HD>\)[,;]", size), size
