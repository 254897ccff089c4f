"""Registers of the built 8-bit attention kernels, and variables that a path leaves unset in the prompt kernel's: what their figures rest on and no
run shows reliably. Reads the build's own gfx950 code objects."""
import os
import re
import subprocess

import pytest
from test_build_checks import kernels  # noqa: F401

from lazyweights_amd.build import ARCH, COMMON, CSRC, HIP_DEVICE, HIPCC, OBJDUMP


def notes(obj):
    """Kernel -> its metadata's numbers."""
    text = subprocess.run([os.path.join(os.path.dirname(OBJDUMP), "llvm-readelf"), "--notes", obj], check=True, text=True,
                          stdout=subprocess.PIPE).stdout
    found = {}
    for part in text.split("- .agpr_count:")[1:]:
        name = re.search(r"\.name:\s+(\S+)", part).group(1)
        found[name] = {k: int(v) for k, v in re.findall(r"\.(vgpr_count|vgpr_spill_count|private_segment_fixed_size):\s+(\d+)", part)}
    return found


def of(kernels, pattern):  # noqa: F811
    found, read = kernels(pattern), {}
    for obj in set(found.values()):
        read.update(notes(obj))
    return {name: dict(read[name], obj=obj) for name, obj in found.items()}


def test_decode_append_and_pages_stay_in_registers(kernels):  # noqa: F811
    """Nothing goes to memory, and decode of one row tile in parts takes 128 registers at most: four waves a SIMD."""
    decode = of(kernels, "k_attn8_decode")
    assert len(decode) == 2 * (3 * 3 + 1)
    for name, n in decode.items():
        size, tiles, runs = re.search(r"ILi(\d+)ELb[01]ELi(\d)ELi[48]ELb([01])E", name).groups()
        assert n["vgpr_count"] <= (128 if tiles == "1" and runs == "0" else 256), name
        assert runs == "0" or size == "128", name
    rest = {**of(kernels, "k_kv8_append"), **of(kernels, "k_pages")}
    assert len(rest) == 18 + 2
    for name, n in {**decode, **rest}.items():
        assert n["vgpr_spill_count"] == 0 and n["private_segment_fixed_size"] == 0, name


def loops(obj, name):
    """(instructions' names) of every loop of a kernel: from a branch back to where it goes."""
    text = subprocess.run([OBJDUMP, "-d", "--mcpu=" + ARCH, "--disassemble-symbols=" + name, obj], check=True, text=True,
                          stdout=subprocess.PIPE).stdout
    base, rows = 0, []
    for line in text.splitlines():
        head, row = re.match(r"([0-9a-f]+) <", line), re.match(r"\s+(\S+)\s*(.*?)\s*//\s*([0-9A-F]+):", line)
        if head:
            base = int(head.group(1), 16)
        if row:
            to = re.search(r"<\S+\+0x([0-9a-f]+)>", line)
            rows.append((int(row.group(3), 16), row.group(1), base + int(to.group(1), 16) if to and "branch" in row.group(1) else None))
    return [[op for at, op, _ in rows if to <= at <= end] for end, _, to in rows if to is not None and to <= end]


def test_prompt_loops_stay_in_registers(kernels):  # noqa: F811
    """No loop over tiles moves registers to memory or back (a reload would wait for the tile that is on its way), but for the forms of
    long runs with fp32 outputs, whose additional sums do not all fit."""
    found = {name: n for name, n in of(kernels, "k_attn_prompt").items() if "Attn8Args" in name}
    assert len(found) == 2 * 3 * (2 + 2 * 2)
    seen = 0
    for name, n in found.items():
        if re.search(r"ELi\dELi[48]ELb1E", name):
            continue
        with_products = [ops for ops in loops(n["obj"], name) if any("mfma" in op for op in ops)]
        assert with_products, name
        seen += 1
        assert not any(op.startswith("scratch") for ops in with_products for op in ops), name
    assert seen == 2 * 3 * (2 + 2)


@pytest.mark.parametrize("form", ("128, true, 1, 4, false", "96, false, 2, 8, false", "64, true, 2, 4, true", "128, false, 2, 8, true"))
def test_no_path_of_a_prompt_reads_a_variable_that_was_not_set(tmp_path, form):
    """As of the other kernels in test_attention8_build.py, of some of the prompt kernel's forms."""
    source, out = tmp_path / "k.hip", tmp_path / "k.ll"
    source.write_text('#include "lw_attn_prompt.h"\nnamespace lw {\nvoid launch(const Attn8Args& a) { k_attn_prompt<%s, Attn8Args><<<1, 64>>>(a); }\n}\n'
                      % form)
    subprocess.run([HIPCC, "-x", "hip", "--cuda-device-only", "-S", "-emit-llvm", str(source), "-o", str(out), "-I", CSRC] + COMMON + HIP_DEVICE,
                   check=True, stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    bodies = re.findall(r"^define [^\n]*k_attn_prompt[^\n]*\{\n(.*?)^\}", out.read_text(), re.M | re.S)
    assert len(bodies) == 1
    assert not [line for line in bodies[0].splitlines() if re.search(r"= phi i\d+ .*\b(undef|poison)\b", line)]
