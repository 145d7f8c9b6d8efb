"""What the serving operators do on the host, and rules of their kernels that only the source shows (CPU)."""
import os
import re

from spruce_research_b200 import build

CSRC = build.CSRC


def test_a_warpgroup_gives_up_registers_by_one_instruction():
    """setmaxnreg is defined only where all warps of a warpgroup execute the same one: once for each side of the split,
    under a condition on the warpgroup, before the roles of its warps part."""
    with open(os.path.join(CSRC, "paged_chunk_sm100.cu")) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert len(re.findall(r"setmaxnreg\.dec", code)) == 1 and len(re.findall(r"setmaxnreg\.inc", code)) == 1
    assert re.search(r"if \(warp >= kChunkMma\) \{\s*asm volatile\(\"setmaxnreg\.dec", code)
    assert re.search(r"\} else \{\s*asm volatile\(\"setmaxnreg\.inc", code)
    roles = {k: int(v) for k, v in re.findall(r"constexpr int kChunk(Mma|Threads) = (\d+);", code)}
    assert roles["Mma"] % 4 == 0 and roles["Threads"] == 32 * (roles["Mma"] + 4)   # whole warpgroups either side
