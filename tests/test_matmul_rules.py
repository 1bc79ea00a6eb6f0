"""CPU: the rules that give a 16-bit product its tiles and the parts of its sums (loki_amd/csrc/launch_rules.h), compiled as they are:
what they answer can be launched, and the sizes of the GPU test of all kernels reach every one of them."""
import ctypes
import os
import subprocess

import pytest

from tests import _mm_cases as cases

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "loki_amd", "csrc", "launch_rules.h")
SMALL, WIDE, LARGE, FEW = range(4)


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("mm_rules")
    src, so = d / "rules.cpp", d / "rules.so"
    src.write_text('#include "%s"\n' % HEADER +
                   'extern "C" int mm(int n, int ne, int cols, int terms, int fwd) { auto p = lk::mm_plan(n, ne, cols, terms, fwd != 0); return 100 * p.shape + p.parts; }\n'
                   'extern "C" int dw(int n, int ne, int R, int K, int mats) { auto p = lk::dw_plan(n, ne, R, K, mats); return 100 * p.shape + p.parts; }\n')
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    return lambda which, *a: divmod(getattr(lib, which)(*a), 100)


def test_the_cases_reach_every_kernel(rules):
    seen = set()
    for n, ne, R, K in [(n, 1, R, K) for n, R, K in cases.DENSE] + cases.EXPERTS:
        g = "dense" if ne == 1 else "experts"
        for name, (shape, parts) in (("forward", rules("mm", n, ne, R, K, 1)), ("gated", rules("mm", n, ne, 2 * R, K, 1)), ("dx", rules("mm", n, ne, K, R, 0)),
                                     ("dx2", rules("mm", n, ne, K, 2 * R, 0)), ("dW", rules("dw", n, ne, R, K, 1)), ("dW2", rules("dw", n, ne, R, K, 2))):
            seen.add((name, g, shape, parts > 1))
    for g in ("dense", "experts"):
        for name in ("forward", "gated", "dx", "dx2"):
            for want in [(SMALL, False), (SMALL, True), (WIDE, False), (WIDE, True), (LARGE, False)] + ([(FEW, False)] if name in ("forward", "gated") else []):
                assert (name, g) + want in seen, (name, g, want)
        for want in [(SMALL, False), (SMALL, True), (LARGE, False), (FEW, False)]:
            assert ("dW", g) + want in seen, (g, want)
    assert any(("dW", "dense", LARGE, True) == s for s in seen) and any(s[0] == "forward" and s[2:] == (LARGE, True) for s in seen)


def test_plans_can_be_launched(rules):
    """Few rows' kernel is the forward pass's alone and never splits; a part has two rounds at least on average; the parts' workspace stays below
    1 GiB up to 2^20 rows or 16384 columns, and experts that could have all rows count as one."""
    sizes = (8, 72, 264, 1032, 2048, 7168, 16384, 65536)
    for ne in (1, 2, 8, 64, 256):
        for n in (1, 2, 7, 16, 31, 64, 129, 500, 1001, 4096, 8192, 65536, 1 << 20, 1 << 24):
            for R in sizes:
                for K in sizes:
                    for fwd in (0, 1):
                        shape, parts = rules("mm", n, ne, R, K, fwd)
                        assert shape in (SMALL, WIDE, LARGE) or (fwd and shape == FEW and parts == 1 and n <= 1 << 15)
                        assert parts == 1 or (parts <= 16 and parts * 128 <= K)
                        assert parts == 1 or parts * n * R * 4 <= 1 << 30, (n, ne, R, K, shape, parts)
                    shape, parts = rules("dw", n, ne, R, K, 2)
                    assert shape in (SMALL, LARGE, FEW)
                    assert parts == 1 or (parts <= 16 and parts * 128 * ne <= n and parts * ne * R * K * 8 <= 1 << 30), (n, ne, R, K, shape, parts)
