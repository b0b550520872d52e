"""Orders of work inside the paged chunk kernels (csrc/paged_order.h), on the host."""
import ctypes as C
import os
import random
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("order") / "host_paged_order.so")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-Wall", "-Wextra", "-Werror", os.path.join(HERE, "host_paged_order.cpp"), "-o", so])
    l = C.CDLL(so)
    l.host_chunk_products.restype = C.c_char_p
    return l


@pytest.mark.parametrize("units", [[1], [2], [3], [4], [17], [1, 1, 1], [1, 2, 3, 4], [5, 1, 2], [random.Random(1).randint(1, 9) for _ in range(60)]])
def test_scores_wait_for_the_product_that_reads_what_they_overwrite(lib, units):
    """Two products of different shapes have no order but the one that a wait gives them."""
    assert lib.host_chunk_products((C.c_int * len(units))(*units), len(units)).decode() == ""


@pytest.mark.parametrize("rounds", range(0, 9))
@pytest.mark.parametrize("reads", range(0, 9))
def test_the_last_fill_of_a_slot_is_waited_for_when_a_wait_gave_up(lib, rounds, reads):
    assert lib.host_settles_wrongly(rounds, reads) == 0
