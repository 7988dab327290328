"""What hipcc makes of the batch attention, read from the assembly that it writes for this source: no kernel spills.  And the one-row-tile form asks for a block
in one place: a second load whose values nothing uses is dropped without a word, and the source then says something that is not done."""
import os
import re
import shlex
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quickvideo_amd", "csrc")


def source():
    with open(os.path.join(CSRC, "qp_batch.hip")) as f:
        return f.read()


@pytest.mark.skipif(shutil.which("/opt/rocm/bin/hipcc") is None, reason="no hipcc")
def test_nothing_spills(tmp_path):
    plan = subprocess.run(["make", "-Bn", "-C", CSRC, "qp_batch.o"], capture_output=True, text=True, check=True).stdout
    words = shlex.split(next(line for line in plan.splitlines() if " qp_batch.hip " in line and " -c " in line))
    words.remove("-c")
    words[words.index("-o") + 1] = str(tmp_path / "out.s")
    subprocess.run(words + ["--cuda-device-only", "-S"], cwd=CSRC, check=True, capture_output=True)
    asm = (tmp_path / "out.s").read_text()
    kernels = re.findall(r"\.name:\s+(\S*batch_\S*)\n(?:.*\n)*?.*\.vgpr_spill_count: (\d+)", asm)
    assert len(kernels) >= 8 and all(spills == "0" for _, spills in kernels), kernels
    assert "scratch_" not in asm


def test_a_block_is_asked_for_in_one_place():
    text = source()
    start = text.index("__device__ __forceinline__ void walk_alone(")
    body = text[start:text.index("\n}\n", start)]
    assert len(re.findall(r"(?<![\w.])load\(", body)) == 1
