"""Whether two sets of rows share a float (csrc/row_overlap.h), and whether a layer's pages have a row for every place (csrc/paged_plan.h), against sets of addresses."""
import ctypes as C
import os
import random
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("rows") / "host_row_overlap.so")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-static-libubsan", "-shared", "-fPIC", "-Wall", "-Wextra", "-Werror",
                           os.path.join(HERE, "host_row_overlap.cpp"), "-o", so])
    l = C.CDLL(so)
    l.host_rows_overlap.argtypes = [C.c_uint64, C.c_int64, C.c_int64, C.c_uint64, C.c_int64, C.c_int64, C.c_int64]
    l.host_rows_apart.argtypes = [C.c_int] * 4 + [C.c_int64] * 3
    return l


@pytest.fixture(scope="module")
def overlap(lib):
    return lib.host_rows_overlap


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


def test_strides_of_pages_whose_rows_lie_on_one_another(lib):
    """Never taken where two rows share an element; always where a dense order of the three with any gaps made them."""
    rng, taken = random.Random(5), 0
    for _ in range(4000):
        hs, n = rng.randint(1, 4), [rng.randint(1, 4) for _ in range(3)]  # pages, heads, places
        strides = [rng.randint(hs, 40) for _ in range(3)]
        rows = [sum(i * s for i, s in zip((p, h, t), strides)) for p in range(n[0]) for h in range(n[1]) for t in range(n[2])]
        shared = len({r + e for r in rows for e in range(hs)}) < hs * len(rows)
        apart = lib.host_rows_apart(hs, *n, *strides)
        assert not (apart and shared), (hs, n, strides)
        taken += apart
        order, span, dense = rng.sample(range(3), 3), hs, [0, 0, 0]
        for d in order:
            dense[d] = span + rng.choice([0, 0, 1, 5])
            span = n[d] * dense[d]
        assert lib.host_rows_apart(hs, *n, *dense), (hs, n, dense)
    assert taken > 300
    assert lib.host_rows_apart(256, 1 << 30, 1, 1, 1 << 61, 256, 256) and not lib.host_rows_apart(128, 11, 2, 64, 1 << 12, 64 * 128, 128)
