"""Properties of the 8-bit attention kernels' code that no run shows reliably."""
import os
import re
import subprocess

import pytest

from lazyweights_amd.build import COMMON, CSRC, HIP_DEVICE, HIPCC


@pytest.mark.parametrize("source, kernel", [("lw_attn8_decode.hip", "k_attn8_decode"), ("lw_kv8_append.hip", "k_kv8_append"),
                                            ("lw_pages.hip", "k_pages")])
def test_no_path_reads_a_variable_that_was_not_set(tmp_path, source, kernel):
    """In the optimised IR a variable that some path leaves unset is an undefined operand of the phi where the paths meet. Whole
    numbers: indices, lengths, counts (the compiler itself leaves sums unset in threads that store nothing)."""
    out = tmp_path / "k.ll"
    subprocess.run([HIPCC, "-x", "hip", "--cuda-device-only", "-S", "-emit-llvm", os.path.join(CSRC, source), "-o", str(out)] +
                   COMMON + HIP_DEVICE, check=True, stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    bodies = re.findall(r"^define [^\n]*%s[^\n]*\{\n(.*?)^\}" % kernel, out.read_text(), re.M | re.S)
    assert bodies
    unset = [line.strip() for body in bodies for line in body.splitlines() if re.search(r"= phi i\d+ .*\b(undef|poison)\b", line)]
    assert not unset, unset[:8]
