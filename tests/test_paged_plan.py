"""The host's side of a step over a paged cache: refusals, and that the blocks' shares cover every (tile, head, unit) once."""
import ctypes as C
import os
import subprocess
import time

import numpy as np
import pytest

COST = 2  # places of the line in front of a pair
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("paged") / "host_paged.so")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-static-libubsan", "-shared", "-fPIC", "-Wall", "-Wextra", "-Werror",
                           os.path.join(HERE, "host_paged.cpp"), "-o", so])
    l = C.CDLL(so)
    l.host_paged_create.restype = C.c_void_p
    l.host_paged_destroy.argtypes = [C.c_void_p]
    l.host_paged_layout.argtypes = [C.c_void_p, C.c_void_p]
    l.host_paged_plan.restype = C.c_char_p
    l.host_paged_plan.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p, C.c_longlong, C.c_void_p, C.c_void_p]
    return l


class Plan:
    def __init__(self, lib, heads=8, kv=2, size=64, page=16, pages=100, dtype=1, seqs=8, tokens=200, table=400, lanes=((16, 64, 37, 1, 0), (128, 128, 5, 1, 0)), few=16, most=0):
        self.lib, self.kv, self.page, self.group, self.lanes, self.few, self.most = lib, kv, page, heads // max(1, kv), lanes, few, most
        why = C.create_string_buffer(300)
        cfg = (C.c_int * 9)(heads, kv, size, page, pages, dtype, seqs, tokens, table)
        flat = (C.c_int * 10)(*lanes[0], *lanes[1])
        self.h = lib.host_paged_create(cfg, flat, few, most, why, 300)
        self.why = why.value.decode()
        if self.h:
            lay = (C.c_int * 8)()
            lib.host_paged_layout(self.h, lay)
            self.total, *at, self.count, self.rows, self.dynamic = lay
            self.starts, self.joins = at[:2], at[2:]
            self.out = np.full(self.total, -7, np.int32)

    def __call__(self, pos0, n_new, tables):
        pos0, n_new, tables = (np.ascontiguousarray(x, np.int32) for x in (pos0, n_new, tables))
        step = (C.c_int * 6)()
        why = self.lib.host_paged_plan(self.h, len(pos0), pos0.ctypes.data, n_new.ctypes.data, tables.ctypes.data, tables.shape[1], self.out.ctypes.data, step)
        self.step = list(step)
        return why.decode()

    def __del__(self):
        if self.h:
            self.lib.host_paged_destroy(self.h)


@pytest.mark.parametrize("bad, word", [
    (dict(kv=3), "n_kv_heads"), (dict(kv=0), "n_kv_heads"), (dict(heads=0), "n_kv_heads"), (dict(size=0), "head_size"), (dict(size=257), "head_size"),
    (dict(page=0), "page_size"), (dict(pages=0), "n_pages"), (dict(pages=1 << 27, page=16), "n_pages"), (dict(dtype=2), "cache type"),
    (dict(seqs=0), "max_seqs"), (dict(tokens=0), "max_tokens"), (dict(table=0), "max_table")])
def test_configurations_that_are_refused(lib, bad, word):
    p = Plan(lib, **bad)
    assert not p.h and word in p.why


def table(rows, width=20):
    t = np.full((len(rows), width), -1, np.int32)
    for b, r in enumerate(rows):
        t[b, :len(r)] = r
    return t


def test_steps_that_are_refused(lib):
    p = Plan(lib)
    ok = ([20, 0], [1, 5], table([[3, 9], [4]]))
    assert p(*ok) == ""
    before = p.out.copy()
    for case, word in [
        (([-1, 0], [1, 5], ok[2]), "negative number of cached"),
        (([20, 0], [1, -5], ok[2]), "negative number of new"),
        (([20, 0], [1, 5], table([[3, 100], [4]])), "no such page"),       # behind the last
        (([20, 0], [1, 5], table([[-1, 9], [4]])), "no such page"),
        (([20, 0], [1, 5], table([[3, 9], [9]])), "used twice"),           # both sequences write page 9
        (([20, 0], [1, 5], table([[9, 9], [4]])), "used twice"),           # read and written by one
        (([20, 16], [1, 5], table([[3, 4], [4, 5]])), "used twice"),       # one reads what the other writes
        (([20, 0], [1, 5], table([[3], [4]], width=1)), "too narrow"),
        (([20, 0], [1, 200], table([[3, 9], list(range(10, 23))])), "max_tokens"),
        (([2**31 - 1024, 0], [1, 5], ok[2]), "too"),
        (([0] * 9, [1] * 9, table([[i] for i in range(9)])), "n_seq"),
    ]:
        assert word in p(*case), (case, word)
        assert (p.out == before).all()  # the step before stays
    narrow = Plan(lib, table=3)
    assert "max_table" in narrow([20, 16], [1, 1], table([[3, 9], [4, 5]]))
    assert narrow([20, 0], [1, 1], table([[3, 9], [4]])) == ""


def test_far_too_many_tokens_are_refused_at_once(lib):
    """Their tiles, billions, are not counted first."""
    p = Plan(lib, heads=64, kv=1, most=128)
    begin = time.perf_counter()
    assert "too narrow" in p([0] * 8, [2**31 - 2000] * 8, table([[0]] * 8))
    assert time.perf_counter() - begin < 1


def test_pages_that_are_only_read_may_be_shared(lib):
    p = Plan(lib)
    assert p([16, 16], [1, 3], table([[3, 9], [3, 4]])) == ""
    assert p([32, 32], [1, 3], table([[3, 3, 9], [3, 7, 4]])) == ""
    assert p([5, 5], [0, 0], table([[3], [3]])) == "" and p.step[0] == 0    # no new tokens: takes no part, whatever its table
    assert p([5, 5], [0, 1], table([[-4], [3]])) == "" and p.step[0] == 1
    assert p([], [], np.zeros((0, 1), np.int32)) == "" and p.step[:3] == [0, 0, 0]


def walk(p, k):
    """What the blocks of lane k take, as the kernels walk it: (tile, head, unit) in order, block by block; and the joins."""
    words = lambda at, n: p.out[at:at + n]  # noqa: E731
    got, parts = [], {}
    for c in range(p.lanes[k][2]):
        s = words(p.starts[k] + 16 * c, 16)
        tile, head, unit, left = (int(x) for x in s[:4])
        t, tiles, U, blocks, me = s[4:12], int(s[12]), int(s[13]), int(s[14]), int(s[15])
        assert left <= 0 or c < p.step[1 + k]
        if c < p.step[1 + k]:
            assert me == c and blocks == p.step[1 + k] and (t == words(tiles + 8 * tile, 8)).all()
        began = unit
        while left > 0:
            n = min(left, int(t[5]) - unit)
            assert n > 0
            got += [(tile, head, u) for u in range(unit, unit + n)]
            if n < t[5]:
                at = int(t[6]) + COST + head * (int(t[5]) + COST)
                block = lambda x: ((x + 1) * blocks - 1) // U  # noqa: E731
                parts.setdefault((tile, head), ([int(x) for x in t[[0, 2, 3]]] + [head, block(at), block(at + int(t[5]) - 1)], []))[1].append((c, int(unit == 0)))
                assert unit == 0 or unit == began
            left -= n + COST
            unit = began = 0
            if left > 0:
                head += 1
                if head == p.kv:
                    head, tile = 0, tile + 1
                    t = words(tiles + 8 * tile, 8)
    for (*_, first, last), blocks in parts.values():
        assert blocks == [(b, int(b == first)) for b in range(first, last + 1)]
    joins = [words(p.joins[k] + 8 * i, 6).tolist() for i in range(p.step[4 + k])]
    assert p.out[p.count + 1 + k] == p.step[4 + k] == len(parts) and joins == [j for j, _ in parts.values()]
    return got


@pytest.mark.parametrize("seed", range(12))
def test_every_unit_is_taken_once(lib, seed):
    rng = np.random.default_rng(seed)
    kv, group, page = int(rng.integers(1, 5)), int(rng.integers(1, 9)), int(rng.choice([1, 3, 16, 64]))
    n = int(rng.integers(1, 9))
    pos0 = rng.integers(0, 700, n)
    n_new = np.where(rng.random(n) < 0.3, rng.integers(1, 150, n), rng.integers(0, 3, n))
    used = [-(-int(a + b) // page) for a, b in zip(pos0, n_new)]
    lanes = ((16, 64, int(rng.integers(1, 300)), int(rng.integers(1, 4)), int(rng.choice([0, 3, 20]))), (128, 128, int(rng.integers(0, 20)), 1, int(rng.choice([0, 2]))))
    p = Plan(lib, heads=kv * group, kv=kv, page=page, pages=sum(used) + 1, tokens=max(1, int(n_new.sum())), table=max(1, sum(used)), lanes=lanes, few=int(rng.choice([16, 64])), most=int(rng.choice([0, 128])))
    ids = rng.permutation(sum(used) + 1)
    tab, at = np.zeros((n, max(used) + 2), np.int32), 0
    for b, u in enumerate(used):
        tab[b, :u] = ids[at:at + u]
        at += u
    assert p(pos0, n_new, tab) == ""
    assert p.step[0] == p.out[p.count] == n_new.sum()
    # rows: position and slot
    rows = p.out[p.rows:p.rows + 2 * p.step[0]].reshape(-1, 2)
    want = [(q, tab[b, q // page] * page + q % page) for b in range(n) for q in range(pos0[b], pos0[b] + n_new[b])]
    assert rows.tolist() == [list(w) for w in want]
    # tiles: every packed row once, with its sequence's table and enough units for its last row
    seen = []
    for k in range(2):
        height, unit = lanes[k][0], lanes[k][1]
        got = walk(p, k)
        assert len(set(got)) == len(got)
        tiles = {}
        for t, h, u in got:
            tiles.setdefault(t, {}).setdefault(h, []).append(u)
        if not got:
            continue
        base = int(p.out[p.starts[k] + 12])
        for t in range(len(tiles)):
            row0, p0, first, rows_in, tab_at, units = (int(x) for x in p.out[base + 8 * t:base + 8 * t + 6])
            b = int(np.searchsorted(np.cumsum(n_new), row0, side="right"))
            assert row0 == n_new[:b].sum() and p0 == pos0[b] and 1 <= rows_in <= height
            assert (p.out[tab_at:tab_at + used[b]] == tab[b, :used[b]]).all()
            assert units == (p0 + (first + rows_in - 1) // group) // unit + 1
            assert tiles[t] == {h: list(range(units)) for h in range(kv)}
            seen += [(b, r) for r in range(first, first + rows_in)]
            assert lanes[1][2] == 0 or (k == 0 and n_new[b] * group <= max(p.few, p.most)) or (k == 1 and n_new[b] * group > p.few)
    assert sorted(seen) == [(b, r) for b in range(n) for r in range(n_new[b] * group)]
    assert p.dynamic + p.step[3] <= p.total


def test_short_pairs_are_not_cut(lib):
    p = Plan(lib, heads=8, kv=2, pages=100, lanes=((8, 64, 40, 1, 9), (128, 128, 5, 1, 0)))
    ids = np.arange(99, dtype=np.int32).reshape(3, 33)
    assert p([500, 0, 300], [1, 1, 2], ids) == "" and p.step[1] == 6 and p.step[4] == 0
    assert len(walk(p, 0)) == sum(2 * u for u in (8, 1, 5))
    many = Plan(lib, heads=8, kv=2, pages=100, lanes=((8, 64, 5, 1, 9), (128, 128, 5, 1, 0)))  # fewer blocks than pairs: equal shares
    assert many([500, 0, 300], [1, 1, 2], ids) == "" and many.step[1] == 5
    walk(many, 0)


def test_which_lane_takes_what_either_could(lib):
    """A few rows more than the kernel for few surely takes: alone they go there, many such sequences to the other kernel, and beside a long chunk too."""
    p = Plan(lib, heads=8, kv=2, pages=2000, seqs=64, tokens=2000, table=4000, lanes=((8, 64, 40, 1, 0), (256, 128, 20, 1, 0)), most=128)
    ids = np.arange(1600, dtype=np.int32).reshape(40, 40)
    assert p([100], [16], ids[:1]) == "" and p.step[1] > 0 and p.step[2] == 0
    assert p([500] * 40, [16] * 40, ids) == "" and p.step[1] == 0 and p.step[2] > 0
    assert p([500] * 40, [4] * 40, ids) == "" and p.step[1] > 0 and p.step[2] == 0
    assert p([100, 0], [4, 600], ids[:2]) == "" and p.step[1] > 0 and p.step[2] > 0


def test_division(lib):
    rng = np.random.default_rng(0)
    for d in [1, 2, 3, 5, 7, 8, 12, 16, 20, 100, 127, 128, 129, 4095, 65536, (1 << 20) - 1, 1 << 20, (1 << 30) - 1, 1 << 30, *map(int, rng.integers(1, 1 << 20, 200))]:
        near = [k * d + e for k in map(int, rng.integers(0, (2**31 - 1) // d, 40)) for e in (-1, 0, 1)]
        for n in [0, 1, d - 1, d, 2**31 - 1, 2**31 - 2, *near]:
            if 0 <= n < 2**31:
                assert lib.host_paged_div(n, d) == n // d, (n, d)


def test_capacity_holds_any_step_of_it(lib):
    """One token of each of max_seqs sequences, and all of max_tokens in one: both fill what the layout has."""
    p = Plan(lib, heads=24, kv=8, seqs=40, tokens=40, table=120, pages=200, few=3)
    assert p([40] * 40, [1] * 40, np.arange(120, dtype=np.int32).reshape(40, 3)) == ""
    assert p.dynamic + p.step[3] <= p.total
    assert p([0], [40], np.arange(3, dtype=np.int32)[None]) == ""
    assert p.dynamic + p.step[3] <= p.total and p.step[2] > 0
