"""Whether two sets of rows share a float (csrc/row_overlap.h), against sets of addresses."""
import ctypes as C
import os
import random
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def overlap(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("rows") / "host_row_overlap.so")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-static-libubsan", "-shared", "-fPIC", "-Wall", "-Wextra", "-Werror",
                           os.path.join(HERE, "host_row_overlap.cpp"), "-o", so])
    f = C.CDLL(so).host_rows_overlap
    f.argtypes = [C.c_uint64, C.c_int64, C.c_int64, C.c_uint64, C.c_int64, C.c_int64, C.c_int64]
    return f


def floats(a, ld, w, n):
    return {a + 4 * (i * ld + e) + byte for i in range(n) for e in range(w) for byte in range(4)}


@pytest.mark.parametrize("same_ld", [True, False])
def test_against_sets_of_addresses(overlap, same_ld):
    rng = random.Random(7 + same_ld)
    seen = [0, 0]
    for _ in range(6000):
        n, w_a, w_b = rng.randint(0, 5), rng.randint(0, 4), rng.randint(0, 4)
        ld_a = max(1, w_a, w_b) + rng.randint(0, 5)
        ld_b = ld_a if same_ld else max(1, w_b) + rng.randint(0, 5)
        a = 4096
        b = a + rng.choice([4, 4, 4, 1]) * rng.randint(-40, 40)
        want = bool(floats(a, ld_a, w_a, n) & floats(b, ld_b, w_b, n))
        assert bool(overlap(a, ld_a, w_a, b, ld_b, w_b, n)) == want, (a, ld_a, w_a, b, ld_b, w_b, n)
        seen[want] += 1
    assert min(seen) > 500


def test_the_largest_rows(overlap):
    big = (1 << 62) - 1
    assert not overlap(4096, big, 8, 4096 + 32, big, 8, 1 << 24)
    assert overlap(4096, big, 9, 4096 + 32, big, 8, 1 << 24)
    assert not overlap(0, 1 << 40, 8, (1 << 63), 1 << 41, 8, 1 << 20)
    assert not overlap(4096, 8, 8, 4096, 8, 8, 0)
