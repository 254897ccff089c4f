"""Properties of the attention kernels' code that no run shows reliably."""
import os
import re
import subprocess

import pytest

from lazyweights_amd.build import COMMON, CSRC, HIP_DEVICE, HIPCC


@pytest.mark.parametrize("source, kernel", [("lw_attn_decode.hip", "k_attn_decode")])
def test_no_path_reads_a_variable_that_was_not_set(tmp_path, source, kernel):
    """In the optimised IR a variable that some path leaves unset is an undefined operand of the phi where the paths meet: with 65
    to 192 sequences a block's later waves hold none of them, and what they compare with the wanted 64 must be set all the same."""
    out = tmp_path / "k.ll"
    subprocess.run([HIPCC, "-x", "hip", "--cuda-device-only", "-S", "-emit-llvm", os.path.join(CSRC, source), "-o", str(out)] +
                   COMMON + HIP_DEVICE, check=True, stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    bodies = re.findall(r"^define [^\n]*%s[^\n]*\{\n(.*?)^\}" % kernel, out.read_text(), re.M | re.S)
    assert bodies
    unset = [line.strip() for body in bodies for line in body.splitlines() if re.search(r"= phi .*\b(undef|poison)\b", line)]
    assert not unset, unset[:8]
