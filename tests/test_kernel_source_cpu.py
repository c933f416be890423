"""Rules that the kernels' source keeps and no run can show broken."""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "forgetune_b200", "csrc")
FILES = sorted(f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")))


def code(name):
    """The file without comments."""
    with open(os.path.join(CSRC, name), encoding="utf-8") as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name", FILES)
def test_tensor_memory_loads_follow_a_warp_barrier(name):
    """tcgen05.ld is .aligned: all lanes of a converged warp.  Lanes that went apart before (a lane that arrived
    on a barrier or sent a copy) meet again only where the program says so."""
    lines = [s for s in code(name).splitlines() if s.strip()]
    for i, s in enumerate(lines):
        if "FTB_TMEM_LD32(" in s and "#define" not in s:
            assert any("__syncwarp();" in t for t in lines[max(0, i - 2):i]), "%s: %s" % (name, s.strip())


def test_cluster_barriers_begin_with_a_warp_barrier():
    """barrier.cluster.arrive and .wait are .aligned too, and in one place."""
    text = {name: code(name) for name in FILES}
    assert [n for n in FILES if "barrier.cluster" in text[n]] == ["tc_ptx.cuh"]
    assert len(re.findall(r"barrier\.cluster\.arrive", text["tc_ptx.cuh"])) == 1
    assert re.search(r"cluster_sync_all\(\)\s*\{\s*__syncwarp\(\);\s*asm volatile\(\"barrier\.cluster\.arrive",
                     text["tc_ptx.cuh"])


def test_a_box_stored_by_rows_is_fenced_before_the_copy_engine_writes_it():
    """Ordinary accesses to shared memory and a TMA load into the same bytes are ordered by a proxy fence of the
    lanes that made them, then the warp barrier before the lane that sends the load."""
    body = re.search(r"void store_box_rows\(.*?\n\}", code("fp8_pair.cuh"), re.S).group(0)
    assert re.search(r"fence_proxy_async_smem\(\);\s*__syncwarp\(\);\s*\}$", body)


# of a model, written when it is made
CONSTANTS = {"tc_conv.cuh": ["__ldg(p.ktab + k)", "__ldg(p.bias + co)"]}


@pytest.mark.parametrize("name", [n for n in FILES if "grid_dep_wait();" in code(n)])
def test_programmatic_launches_read_by_plain_loads(name):
    """A kernel that may begin before the one in front of it is done: what that one writes is written during this one's
    life, which the read-only loads do not allow."""
    text = code(name)
    for constant in CONSTANTS.get(name, []):
        assert constant in text
        text = text.replace(constant, "")
    assert not re.search(r"__ldg|ld\.global\.nc", text)


def test_every_macro_is_used():
    text = "\n".join(code(f) for f in sorted(os.listdir(CSRC)) if f.endswith((".cu", ".cuh", ".cpp", ".h", ".hpp")))
    made = set(re.findall(r"#define (FTB_TMEM_\w+)", text))
    assert made and not [m for m in made if len(re.findall(r"\b%s\b" % m, text)) < 2]
