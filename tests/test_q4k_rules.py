"""CPU: which Q4_K kernel a product gets (loki_amd/csrc/launch_rules.h), compiled as it is and checked over the sizes that the entry
point takes."""
import ctypes
import os
import subprocess

import pytest

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "loki_amd", "csrc", "launch_rules.h")
NS = [1, 2, 3, 8, 16, 17, 32, 33, 48, 49, 64, 100, 128, 129, 500, 2048, 65536]
RS = [1, 15, 16, 17, 64, 512, 1024, 1025, 2048, 7168, 24576, 24577, 131072, 1 << 22]
KS = [256, 512, 2048, 7168, 16384, 65536]


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("q4")
    src, so = d / "rules.cpp", d / "rules.so"
    src.write_text('#include "%s"\nusing namespace lk;\n' % HEADER +
                   'extern "C" int pick(int n, int64_t R, int K, int tiles) { return q4k_kernel(n, R, K, tiles); }\n'
                   'extern "C" int tiled(int k) { return q4k_tiled(k); }\n'
                   'extern "C" int count() { return Q4_KERNELS; }\n'
                   'extern "C" int toks(int k) { return Q4_KERNEL[k].toks; }\n'
                   'extern "C" int rows(int k) { return Q4_KERNEL[k].rows; }\n'
                   'extern "C" float us(int k, int n, int64_t R, int K) { return q4k_us(Q4_KERNEL[k], n, R, K); }\n')
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.pick.argtypes = [ctypes.c_int, ctypes.c_int64, ctypes.c_int, ctypes.c_int]
    lib.us.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_int64, ctypes.c_int]
    lib.us.restype = ctypes.c_float
    return lib


def test_every_size_gets_a_kernel_that_may_be_taken(rules):
    vec = rules.count()
    seen = set()
    for n in NS:
        for R in RS:
            for K in KS:
                for tiles in (0, 1):
                    k = rules.pick(n, R, K, tiles)
                    assert 0 <= k <= vec
                    assert k != vec or n == 1
                    assert tiles or not rules.tiled(k)
                    seen.add(k)
                    if k < vec:   # the least estimate of those allowed
                        assert all(rules.us(k, n, R, K) <= rules.us(j, n, R, K) for j in range(vec) if (tiles and n > 16) or not rules.tiled(j))
    assert seen == set(range(vec + 1)), "a kernel that no size reaches"


def test_estimates_grow_with_the_work(rules):
    for k in range(rules.count()):
        for R in RS:
            for K in KS:
                t = [rules.us(k, n, R, K) for n in NS]
                assert t == sorted(t)
        assert all(rules.us(k, n, 7168, K1) < rules.us(k, n, 7168, K2) for n in NS for K1, K2 in zip(KS, KS[1:]))


def test_few_tokens_do_not_take_many_token_tiles(rules):
    for R in RS:
        for K in KS:
            k = rules.pick(1, R, K, 1)
            assert k == rules.count() or rules.toks(k) == 16
            assert not rules.tiled(rules.pick(16, R, K, 1))


# rows, columns, tokens of the device tests that go through each kernel (test_gpu_q4k.py), ragged in rows and tokens: 1 to 28 blocks a row
SIZES = {"ks_32_16": [(7001, 512, 12), (7001, 7168, 13)], "ks_32_32": [(1001, 1024, 200), (7001, 512, 20)],
         "ks_32_48": [(7001, 768, 40), (2049, 768, 130)], "mm_64_32": [(2049, 1024, 200), (8200, 768, 40), (1001, 3328, 403)],
         "mm_64_64": [(4100, 256, 257), (7001, 768, 130), (1001, 3328, 601)], "mm_128_64": [(4100, 2048, 257), (7001, 3328, 130)],
         "mm_256_64": [(8200, 256, 403), (8200, 2048, 403), (33000, 768, 130)], "mm_128_128_8": [(2049, 256, 1000), (7001, 768, 403), (4100, 3328, 601)],
         "mm_128_128": [(8200, 256, 601), (16000, 768, 333), (7001, 1280, 1000)]}
KERNELS = ["ks_16_16", *SIZES]


@pytest.mark.parametrize("name", SIZES)
def test_sizes_that_reach_each_kernel(rules, name):
    assert [KERNELS[rules.pick(n, R, K, 1)] for R, K, n in SIZES[name]] == [name] * len(SIZES[name])


def test_launches_fit_a_grid(rules):
    """workgroups of 256 or 512 lanes along x below 2^32 lanes, along z (16 .. 48 tokens each) at most 65535, at every size that the
    entry point takes (2^26 rows, 2^19 tokens) and 300 GB hold"""
    n = 1
    while n <= 1 << 19:
        R = 1
        while R <= 1 << 26:
            for K in KS:
                if max(4.0 * n * R, 0.5625 * R * K, 1.0 * n * K) < 3e11:
                    k = rules.pick(n, R, K, 1)
                    t, r = (rules.toks(k), rules.rows(k)) if k < rules.count() else (n, 1)
                    tt, rt = -(-n // t), -(-R // r)
                    if rules.tiled(k):
                        assert rt * tt * 512 < 1 << 32, (n, R, K, k)
                    else:
                        assert tt <= 65535 and rt * (512 if k < rules.count() else 32) < 1 << 32, (n, R, K, k)
            R = R + 1 if R < 16 else min(R * 3 // 2 + 1, 1 << 26) if R < 1 << 26 else R + 1
        n = n + 1 if n < 20 else min(n * 4 // 3 + 1, 1 << 19) if n < 1 << 19 else n + 1
