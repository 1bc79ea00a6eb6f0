"""CPU: the loops over a sum's rounds in the built 16-bit products (matmul.hip) use no scratch memory. The tiles of 256 x 256 spill some registers
around those loops, once a tile; a spill inside one would cost every round, and nothing else would tell."""
import os
import re
import subprocess

import pytest

import loki_amd
from tests.test_isa import OBJDUMP, code_objects

LINE = re.compile(r"^\s+(\S.*?)\s*// ([0-9A-F]{12}):")
TARGET = re.compile(r"<\S+?\+0x([0-9a-f]+)>\s*$")


def kernels(listing):
    """(name, [(offset in the kernel, instruction, a branch's target or None)]) of a disassembly"""
    name, start, code = None, 0, []
    for l in listing.splitlines():
        m = re.match(r"^([0-9a-f]{16}) <(\S+)>:", l)
        if m:
            if name:
                yield name, code
            name, start, code = m.group(2), int(m.group(1), 16), []
            continue
        m = LINE.match(l)
        if m and name:
            t = TARGET.search(l) if m.group(1).startswith(("s_cbranch", "s_branch")) else None
            code.append((int(m.group(2), 16) - start, m.group(1), int(t.group(1), 16) if t else None))
    if name:
        yield name, code


def product_loops(code):
    """(matrix instructions, scratch instructions) of the innermost loops that hold a matrix instruction"""
    spans = [(t, o) for o, _, t in code if t is not None and t <= o]
    for a, b in spans:
        if any((c, d) != (a, b) and a <= c and d <= b for c, d in spans):
            continue
        body = [i for o, i, _ in code if a <= o <= b]
        mfma = sum(i.startswith("v_mfma") for i in body)
        if mfma:
            yield mfma, sum(i.startswith("scratch_") for i in body)


@pytest.mark.skipif(OBJDUMP is None, reason="llvm-objdump not found")
@pytest.mark.skipif(not os.path.exists(loki_amd.LIB_PATH), reason="libloki_moe.so not built")
def test_no_scratch_in_a_products_loop(tmp_path):
    seen = set()
    for k, co in enumerate(code_objects(loki_amd.LIB_PATH)):
        f = tmp_path / ("co%d.o" % k)
        f.write_bytes(co)
        out = subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", str(f)], capture_output=True, text=True, check=True).stdout
        if "k_mm_dx" not in out and "k_mm_few" not in out:
            continue
        for name, code in kernels(out):
            kind = re.search(r"k_mm(_dx|_dw_few|_dw|_few)?(?=I)", name)
            if not kind:
                continue
            loops = list(product_loops(code))
            assert loops, name
            assert all(s == 0 for _, s in loops), (name, loops)
            seen.add(kind.group(0))
    assert seen == {"k_mm", "k_mm_dx", "k_mm_dw", "k_mm_dw_few", "k_mm_few"}


def test_a_planted_spill_is_found():
    listing = "%016x <k>:\n" % 0x100 + "".join("\t%s // %012X: 00\n" % (i, 0x100 + 4 * n) for n, i in enumerate(
        ["scratch_store_dword off, v1, off", "v_mfma_f32_16x16x32_bf16 a", "%s", "s_cbranch_scc1 9", "scratch_load_dword v1, off, off"]))
    back = listing.replace("s_cbranch_scc1 9 // 00000000010C: 00", "s_cbranch_scc1 9 // 00000000010C: 00 <k+0x4>")
    assert [list(product_loops(c)) for _, c in kernels(back % "s_nop 0")] == [[(1, 0)]]
    assert [list(product_loops(c)) for _, c in kernels(back % "scratch_load_dword v2, off, off")] == [[(1, 1)]]
