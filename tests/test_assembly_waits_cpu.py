"""What the many-row kernels ask of the compiler, checked in the gfx950 assembly of
this library's own sources.

Products written as inline assembly (mla_flash.hpp: MLA_MFMA_CHAIN) accumulate in
ordinary registers, and the compiler does not know that they are products:
  * a product's result may be read 11 issue slots after an 8-pass product at the
    earliest (every instruction is a slot, s_nop n is n + 1), except as the accumulator of
    the next product of its chain;
  * an operand that a vector instruction wrote may be read 2 slots later.
stream_to_lds16 leaves m0 changed: nothing outside inline assembly may use m0.
"""
import os
import re
import subprocess
import sys

import pytest

from conftest import PKG

sys.path.insert(0, PKG)
import build as pkg_build  # noqa: E402  -- ada-mla_amd/build.py

RESULT_SLOTS, OPERAND_SLOTS = 11, 2


def _registers(text):
    out = set()
    for kind, lo, hi, one in re.findall(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+))", text):
        first, last = int(lo or one), int(hi or one)
        out |= {(kind, i) for i in range(first, last + 1)}
    return out


class _Line:
    def __init__(self, function, text, inline):
        self.function, self.text, self.inline = function, text, inline
        self.op = text.split()[0]
        self.args = [a.strip() for a in text[len(self.op):].split(",")]
        self.product = self.op.startswith("v_mfma")
        self.slots = int(self.args[0]) + 1 if self.op == "s_nop" else 1


def _lines(asm):
    function, inline, out = "", False, []
    for raw in asm.splitlines():
        if m := re.match(r"(\w+):", raw):
            if not m.group(1).startswith("."):
                function = m.group(1)
        if "ASMSTART" in raw or "ASMEND" in raw:
            inline = "ASMSTART" in raw
        text = raw.split(";")[0].strip()
        if raw[:1] in " \t" and text and not text.startswith((".", "#", "//")) and not text.endswith(":"):
            out.append(_Line(function, text, inline))
    return out


def _faults(lines):
    products, faults = 0, []
    for i, line in enumerate(lines):
        if not line.product or not line.args[0].startswith("v["):
            continue
        products += 1
        result, operands = _registers(line.args[0]), _registers(line.args[1]) | _registers(line.args[2])
        slots, j = 0, i + 1
        while j < len(lines) and slots < RESULT_SLOTS and lines[j].function == line.function:
            other = lines[j]
            if other.op == "s_endpgm":
                break
            if _registers(other.text) & result:
                chain = (other.product and _registers(other.args[0]) == result == _registers(other.args[3])
                         and not (_registers(other.args[1]) | _registers(other.args[2])) & result)
                if not chain:
                    faults.append(f"{line.text} read {slots} slots later by {other.text}")
                break
            slots += other.slots
            j += 1
        slots, j = 0, i - 1
        while j >= 0 and slots < OPERAND_SLOTS and lines[j].function == line.function:
            other = lines[j]
            if (other.op.startswith("v_") and not other.product and not other.op.startswith("v_cmp")
                    and _registers(other.args[0]) & (operands | _registers(line.args[3]))):
                faults.append(f"{line.text} reads what {other.text} wrote {slots} slots before")
                break
            slots += other.slots
            j -= 1
    return products, faults


def test_the_check_sees_faults():
    good = "f:\n\tv_mfma_f32_32x32x16_f16 v[0:15], v[16:19], v[20:23], 0\n" \
           "\tv_mfma_f32_32x32x16_f16 v[0:15], v[24:27], a[0:3], v[0:15]\n\ts_nop 15\n\tv_add_f32 v30, v0, v1\n"
    assert _faults(_lines(good)) == (2, [])
    early = good.replace("s_nop 15", "s_nop 1")
    assert len(_faults(_lines(early))[1]) == 1
    moved = "f:\n\tv_accvgpr_read_b32 v20, a9\n" + good[3:]
    assert len(_faults(_lines(moved))[1]) == 1
    assert _faults(_lines(moved.replace("a9\n", "a9\n\ts_nop 1\n")))[1] == []


@pytest.mark.parametrize("source,products", [("mla_tree.hip", 100), ("mla_prefill.hip", 100)])
def test_waits_around_inline_products_and_m0(source, products, tmp_path):
    out = tmp_path / "kernels.s"
    hipcc = os.path.join(pkg_build.ROCM, "bin", "hipcc")
    subprocess.run([hipcc, *pkg_build.HIPCC_FLAGS, "--cuda-device-only", "-S", os.path.join(pkg_build.CSRC, source),
                    "-o", str(out)], check=True, capture_output=True)
    lines = _lines(out.read_text())
    found, faults = _faults(lines)
    assert found >= products and not faults, faults[:5]
    streams = {l.function for l in lines if l.inline and l.op == "s_add_u32" and l.args[0] == "m0"}
    assert streams
    others = [l.text for l in lines if l.function in streams and not l.inline and re.search(r"\bm0\b", l.text)]
    assert not others, others[:5]
