"""CPU: how the router's backward products are cut into workgroups (loki_amd/csrc/launch_rules.h), compiled as it is and checked over the
sizes that the entry point takes."""
import ctypes
import os
import subprocess

import pytest

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "loki_amd", "csrc", "launch_rules.h")
NS = [1, 31, 127, 128, 129, 255, 256, 257, 512, 1000, 2048, 4096, 8192, 20000, 65536]
ES = [1024 * k for k in (1, 2, 4, 5, 6, 7, 8, 16, 32, 33, 63, 64)]


@pytest.fixture(scope="module")
def cut(tmp_path_factory):
    d = tmp_path_factory.mktemp("route")
    src, so = d / "rules.cpp", d / "rules.so"
    src.write_text('#include "%s"\nusing namespace lk;\n' % HEADER +
                   'extern "C" int splits(int n, int E, int w, int x) { return route_cut(n, E, w, x).splits; }\n'
                   'extern "C" int parts(int n, int E, int w, int x) { return route_cut(n, E, w, x).parts; }\n')
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    return lambda n, E, w, x: (lib.splits(n, E, w, x), lib.parts(n, E, w, x))


def test_every_run_and_part_has_rows(cut):
    for n in NS:
        for E in ES:
            for w, x in ((1, 1), (1, 0), (0, 1)):
                s, p = cut(n, E, w, x)
                steps = -(-n // 32)
                assert 1 <= s <= max(1, n // 128) and 1 <= p <= max(1, -(-n // 256))
                bounds = [steps * r // s for r in range(s + 1)]
                assert all(b > a for a, b in zip(bounds, bounds[1:]))
                assert E // 128 * (s + p) <= 1024 + 256 + 2 * (E // 128)


def test_one_workgroup_a_cu_where_it_fills_them(cut):
    assert cut(5000, 4096, 1, 1) == (5, 3) and cut(3000, 6144, 1, 1) == (3, 2) and cut(700, 7168, 1, 1) == (2, 2)
    assert cut(8192, 7168, 1, 1) == (4, 18) and cut(8192, 7168, 1, 0)[0] == 4 and cut(8192, 7168, 0, 1)[1] == 4
    assert cut(48, 7168, 1, 1) == (1, 1) and cut(65536, 65536, 1, 1)[0] == 1
