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


def test_tensor_memory_changes_hands_between_fences():
    """Tensor memory that one warp read or wrote and another writes or reads next: every hand-over through an mbarrier has
    tcgen05's fence before the arrival and the other one after the wait. The score columns go from the MMA to the softmax
    warps (s_full), among these (x_full) and back as weights (p_full)."""
    text = re.sub(r"\s+", " ", source("kv_attn.cu"))
    loop = text[text.index("float s[kKeys];"):text.index("sm.x_max[0][part][r] = l;")]
    assert "tc_fence_before(); warp_arrive(&sm.x_full[warp & 3], lane);" in loop
    assert "ok = tc_wait_warp(&sm.x_full[warp & 3], b); if (!ok) break; tc_fence_after();" in loop
    assert "tc_wait_st(); tc_fence_before(); warp_arrive(&sm.p_full[g / 2], lane);" in loop
    for wait in re.findall(r"tc_wait_warp\(&sm\.(?:s|x|o)_full[^;]*; if \(!ok\) break; (.{16})", loop):
        assert wait == "tc_fence_after()"


def test_scan_stops_copying_after_a_lost_wait():
    """A chunk's copies that did not arrive in time: the fetching warp starts no more copies into the buffers and waits
    (bounded) for those in flight before the block's shared memory goes."""
    text = re.sub(r"\s+", " ", source("gdn_delta.cu"))
    fetch = text[text.index("if (role == 2) {"):text.index("if (role == 1) {")]
    assert "if (lost < 0 && !mbar_wait(&full[(ch - 1) & 1], ((ch - 1) >> 1) & 1)) lost = ch - 1;" in fetch
    assert fetch.count("bulk_load(") == 2 and fetch.index("if (lane == 0 && lost < 0) {") < fetch.index("bulk_load(")
    end = fetch[fetch.index("cp_async_commit();"):]
    assert "if (lost >= 0) mbar_wait_until(&full[lost & 1], (lost >> 1) & 1, globaltimer_ns() + kWaitLimitNs); return;" in end
