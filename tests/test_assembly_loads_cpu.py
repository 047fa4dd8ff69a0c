"""What the direct loads to LDS (mla_ring.hpp, mla_flash.hpp: inline assembly that the
compiler does not know to be loads) need around them, checked in the gfx950 assembly of
every source of the library. Every instruction is a slot, s_nop n is n + 1:
  * m0, which carries the LDS address, may be read by the load one slot after a scalar
    instruction wrote it;
  * the scalar base may be read 5 slots after a vector instruction (v_readfirstlane) wrote it;
  * m0 is left changed, so nothing outside inline assembly may use it.
And of the products in inline assembly: a result may be read 12 slots after an
8-pass product on gfx950, the distance that the compiler keeps for its own.
All paths to a load count, jumps among them.
"""
import os
import re
import subprocess
import sys

import pytest

from conftest import PKG

sys.path.insert(0, PKG)
import build as pkg_build  # noqa: E402  -- ada-mla_amd/build.py
import test_assembly_waits_cpu as products  # noqa: E402

M0_SLOTS, BASE_SLOTS, RESULT_SLOTS = 1, 5, 12


class _Code:
    """The instructions of one file: (text, inline, label) with label for a jump's target."""

    def __init__(self, asm):
        self.lines, self.jumps, inline = [], {}, False
        for raw in asm.splitlines():
            if m := re.match(r"([\w.$]+):", raw):
                self.lines.append((m.group(1), inline, True))
            if "ASMSTART" in raw or "ASMEND" in raw:
                inline = "ASMSTART" in raw
            text = raw.split(";")[0].strip()
            if raw[:1] in (" ", "\t") and text and not text.startswith((".", "#", "//")) and not text.endswith(":"):
                if m := re.match(r"s_c?branch\w*\s+(\S+)", text):
                    self.jumps.setdefault(m.group(1), []).append(len(self.lines))
                self.lines.append((text, inline, False))

    def before(self, i, slots, seen=None):
        """(instruction, slots between it and line i) on every path to line i, less than `slots` away."""
        seen = {} if seen is None else seen
        stack = [(i - 1, 0)]
        while stack:
            j, away = stack.pop()
            while j >= 0 and away < slots and seen.get(j, slots) > away:
                seen[j] = away
                text, _, label = self.lines[j]
                if label:
                    stack += [(k, away) for k in self.jumps.get(text, [])]
                    if not text.startswith("."):
                        break  # the function's start
                else:
                    if re.match(r"s_branch|s_endpgm|s_setpc", text) and away > 0 and self.lines[j + 1][2]:
                        break  # the line above does not run into the label below
                    yield text, away
                    m = re.match(r"s_nop\s+(\d+)", text)
                    away += int(m.group(1)) + 1 if m else 1
                j -= 1


def _scalars(text):
    out = set()
    for lo, hi, one in re.findall(r"\bs(?:\[(\d+):(\d+)\]|(\d+)\b)", text):
        out |= set(range(int(lo or one), int(hi or one) + 1))
    return out


def _faults(code):
    loads, faults = 0, []
    for i, (text, inline, label) in enumerate(code.lines):
        if label:
            continue
        if not inline and re.search(r"\bm0\b", text):
            faults.append(f"m0 outside inline assembly: {text}")
        if not re.match(r"global_load_lds|buffer_load\w* .*\blds\b", text):
            continue
        loads += 1
        base = _scalars(text)
        for other, away in code.before(i, BASE_SLOTS):
            target = other.split(None, 1)[1].split(",")[0] if " " in other or "\t" in other else ""
            if away < M0_SLOTS and other.startswith("s_") and target.strip() == "m0":
                faults.append(f"{text} reads m0 {away} slots after {other}")
            if other.startswith("v_") and _scalars(target) & base:
                faults.append(f"{text} reads its base {away} slots after {other}")
    return loads, faults


def test_the_check_sees_faults():
    load = "\tglobal_load_lds_dwordx4 v1, s[4:5]\n"
    wrap = lambda s: "f:\n\t;;#ASMSTART\n" + s + "\t;;#ASMEND\n\ts_endpgm\n"  # noqa: E731
    assert _faults(_Code(wrap("\ts_mov_b32 m0, s2\n\ts_nop 0\n" + load))) == (1, [])
    assert _faults(_Code(wrap("\ts_add_u32 m0, s2, 64\n\tv_add_u32 v1, 4, v0\n" + load))) == (1, [])
    assert len(_faults(_Code(wrap("\ts_mov_b32 m0, s2\n" + load)))[1]) == 1
    assert len(_faults(_Code("f:\n\ts_mov_b32 m0, s2\n\ts_nop 0\n" + load))[1]) == 1  # the compiler's own m0
    base = "\tv_readfirstlane_b32 s5, v9\n"
    assert len(_faults(_Code(wrap(base + "\ts_mov_b32 m0, s2\n\ts_nop 0\n" + load)))[1]) == 1
    assert _faults(_Code(wrap(base + "\ts_nop 2\n\ts_mov_b32 m0, s2\n\ts_nop 0\n" + load))) == (1, [])
    assert _faults(_Code(wrap(base.replace("s5", "s6") + "\ts_mov_b32 m0, s2\n\ts_nop 0\n" + load))) == (1, [])
    # over a jump: the write stands behind the load in the text
    jump = "f:\n\ts_branch .L2\n.L1:\n\t;;#ASMSTART\n\ts_mov_b32 m0, s2\n\ts_nop 0\n" + load + \
           "\t;;#ASMEND\n.L2:\n" + base + "\ts_cbranch_scc1 .L1\n\ts_endpgm\n"
    assert len(_faults(_Code(jump))[1]) == 1


@pytest.mark.parametrize("source", pkg_build.HIP_SOURCES)
def test_waits_of_direct_loads(source, tmp_path):
    out = tmp_path / "kernels.s"
    hipcc = os.path.join(pkg_build.ROCM, "bin", "hipcc")
    subprocess.run([hipcc, *pkg_build.HIPCC_FLAGS, "--cuda-device-only", "-S", os.path.join(pkg_build.CSRC, source),
                    "-o", str(out)], check=True, capture_output=True)
    asm = out.read_text()
    loads, faults = _faults(_Code(asm))
    with open(os.path.join(pkg_build.CSRC, source)) as f:
        assert (loads > 0) == bool(re.search(r"global_to_lds16|stream_to_lds16", f.read()))
    assert not faults, (len(faults), faults[:5])


def test_the_compiler_keeps_12_slots_itself(tmp_path):
    # the distance that the inline products below are held to, from a product the compiler knows
    src, out = tmp_path / "product.hip", tmp_path / "product.s"
    src.write_text("""#include <hip/hip_runtime.h>
typedef float f16x __attribute__((ext_vector_type(16)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
__global__ void k(const h8 *p, float *o, float n)
{
    f16x c = {};
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[threadIdx.x], p[threadIdx.x + 64], c, 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
    o[0] = c[0] * n;
}
""")
    hipcc = os.path.join(pkg_build.ROCM, "bin", "hipcc")
    subprocess.run([hipcc, *pkg_build.HIPCC_FLAGS, "--cuda-device-only", "-S", str(src), "-o", str(out)], check=True,
                   capture_output=True)
    lines = products._lines(out.read_text())
    at = next(i for i, l in enumerate(lines) if l.product)
    result, slots = products._registers(lines[at].args[0]), 0
    for other in lines[at + 1:]:
        if products._registers(other.text) & result:
            break
        slots += other.slots
    assert slots == RESULT_SLOTS


@pytest.mark.parametrize("source", ["mla_tree.hip", "mla_prefill.hip"])
def test_results_of_inline_products(source, tmp_path, monkeypatch):
    out = tmp_path / "kernels.s"
    hipcc = os.path.join(pkg_build.ROCM, "bin", "hipcc")
    subprocess.run([hipcc, *pkg_build.HIPCC_FLAGS, "--cuda-device-only", "-S", os.path.join(pkg_build.CSRC, source),
                    "-o", str(out)], check=True, capture_output=True)
    monkeypatch.setattr(products, "RESULT_SLOTS", RESULT_SLOTS)
    found, faults = products._faults(products._lines(out.read_text()))
    assert found >= 100 and not faults, faults[:5]
