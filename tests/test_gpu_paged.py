"""Norms with rotation, append to pages and attention over them (csrc/paged*.cu) against their formulas in 64 bits (paged_reference.py)."""
import numpy as np
import pytest

import paged_reference as R
from slai_b200 import _lib
from slai_b200._lib import KV_F16, KV_F32, SlaiError
from slai_b200.ops import PagedKv, PagedLayer, QkNormRope

pytestmark = pytest.mark.gpu
F16, F32 = KV_F16, KV_F32


class Pages:
    """Sequences in pages, and the same on the host.  `order`: of a page's memory; `gap`: elements between rows that belong to nobody."""

    def __init__(self, be, hq, hk, hs, page, lens, dtype, order="head", gap=0, extra=2, max_tokens=None, seed=0, max_seqs=None, shift=0):
        self.be, self.hq, self.hk, self.hs, self.page, self.dtype = be, hq, hk, hs, page, dtype
        self.rng = np.random.default_rng(seed)
        n = len(lens)
        used = [max(1, -(-l // page)) for l in lens]
        self.n_pages = sum(used) + extra
        ids = self.rng.permutation(self.n_pages).astype(np.int32)
        self.tables = np.full((n, max(used)), -1, np.int32)
        at = 0
        for b, u in enumerate(used):
            self.tables[b, :u] = ids[at:at + u]
            at += u
        row = hs + gap
        self.strides = (hk * page * row, page * row, row) if order == "head" else (hk * page * row, row, hk * row)
        self.np_type = np.float16 if dtype == F16 else np.float32
        size = self.n_pages * hk * page * row + shift
        self.host = [self.rng.standard_normal(size).astype(self.np_type) for _ in range(2)]
        self.dev = [be.vector(a, self.np_type) for a in self.host]
        views = [d.view(shift, size - shift) for d in self.dev]
        self.shift = shift
        self.layer = PagedLayer(*views, *self.strides)
        self.kv = PagedKv(be, hq, hk, hs, page, self.n_pages, dtype, max_seqs=max_seqs or n, max_tokens=max_tokens or max(1, sum(lens)), max_table=max(1, sum(used)))

    def at(self, which, b, pos):
        """Positions `pos` of sequence b on the host: [len(pos)][hk][hs] (a copy)."""
        return self.host[which][self._index(b, pos)]

    def put(self, which, b, pos, rows):
        self.host[which][self._index(b, pos)] = rows

    def _index(self, b, pos):
        pos = np.asarray(pos)
        p, h, s = self.strides
        base = self.tables[b, pos // self.page].astype(np.int64) * p + (pos % self.page) * s + self.shift
        return base[:, None, None] + (np.arange(self.hk) * h)[None, :, None] + np.arange(self.hs)[None, None, :]

    def upload(self):
        for d, h in zip(self.dev, self.host):
            self.be.write_buffer(d.ptr, h)

    def download(self):
        self.host = [d.to_numpy() for d in self.dev]


def check(got, want, bound, what=""):
    assert got.shape == want.shape
    nan = np.isnan(want)
    assert (np.isnan(got) == nan).all(), f"{what}: NaN where none belongs, or none where one does"
    off = np.abs(np.where(nan, 0, got.astype(np.float64) - want))
    with np.errstate(invalid="ignore"):
        bad = ~(off <= np.where(nan, 0, bound))
    bad &= ~((got == want) | nan)  # equal infinities
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size}, first at {tuple(np.argwhere(bad)[0])}: off {off[tuple(np.argwhere(bad)[0])]}"


def attend(ctx, P, pos0, n_new, q=None, scale=0.0, q_ld=0, out_ld=0, only=None):
    """Runs the operator for the step and checks every row; `only`: rows that are checked."""
    be, rows, width = ctx.backend, int(np.sum(n_new)), P.hq * P.hs
    if q is None:
        q = P.rng.standard_normal((rows, P.hq, P.hs)).astype(np.float32) * 2
    P.kv.step(pos0, n_new, P.tables)
    qbuf = np.full((rows, q_ld or width), 7.5, np.float32)
    qbuf[:, :width] = q.reshape(rows, width)
    out = be.vector(np.full((rows + 2) * (out_ld or width), -3.25, np.float32))
    ctx.paged_attention(P.kv, P.layer, be.vector(qbuf), out, scale, q_ld, out_ld)
    got = out.to_numpy().reshape(rows + 2, out_ld or width)
    assert (got[rows:] == -3.25).all() and (got[:, width:] == -3.25).all()  # rows behind the last, floats between rows
    got, at = got[:rows, :width].reshape(rows, P.hq, P.hs), 0
    for b, (p, n) in enumerate(zip(pos0, n_new)):
        if n:
            pick = slice(None)
            held = np.arange(p + n)
            want, bound = R.attention(q[at:at + n], P.at(0, b, held), P.at(1, b, held), p, scale or P.hs**-0.5)
            check(got[at:at + n][pick], want[pick], bound[pick], f"sequence {b}")
        at += n
    return got


# ---- norms and rotation ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hs", [2, 48, 64, 80, 128, 200, 256])
@pytest.mark.parametrize("variant", [None, 0, 1])
@pytest.mark.parametrize("norms", [True, False])
def test_qk_norm_rope(ctx, backend, hs, variant, norms):
    rng = np.random.default_rng(hs)
    T, hq, hk = 13, 6, 2
    pos = np.array([0, 1, 2, 77, 511, 4095, 32767, 120000, 120001, 1 << 24, (1 << 31) - 2, 5, 9], np.int32)
    q, k = rng.standard_normal((T, hq, hs)).astype(np.float32) * 3, rng.standard_normal((T, hk, hs)).astype(np.float32)
    wq, wk = (rng.standard_normal((2, hs)) + 1).astype(np.float32)
    how = QkNormRope(hs, hq, hk, variant, 10000.0, 1e-5, backend.vector(wq) if norms else None, backend.vector(wk) if norms else None)
    qo, ko = backend.zeros(q.size), backend.zeros(k.size)
    ctx.qk_norm_rope(how, backend.vector(pos, np.int32), backend.vector(q), backend.vector(k), qo, ko)
    for got, x, w in ((qo, q, wq), (ko, k, wk)):
        check(got.to_numpy().reshape(x.shape), *R.norm_rope(x, w if norms else None, 1e-5, variant, 10000.0, pos))


@pytest.mark.parametrize("hs, T, hq, hk, pad, shift", [(128, 1, 64, 8, 0, 0), (128, 300, 32, 32, 0, 0), (64, 37, 25, 25, 4, 0), (128, 9, 4, 4, 3, 0), (128, 9, 4, 4, 0, 1),
                                                       (96, 5, 3, 1, 0, 0), (65, 4, 3, 1, 0, 0), (1, 4, 3, 1, 0, 0), (256, 17, 8, 1, 0, 0)])
@pytest.mark.parametrize("variant", [0, 1])
def test_rows_of_one_product_in_place_and_apart(ctx, backend, hs, T, hq, hk, pad, shift, variant):
    """q and k inside a fused product's rows; results in place, and rows whose position is negative stay as they are."""
    if hs % 2:
        variant = None
    rng = np.random.default_rng(T)
    ld = (hq + 2 * hk) * hs + pad
    x = rng.standard_normal(T * ld + shift).astype(np.float32)
    pos = rng.integers(0, 200000, T).astype(np.int32)
    if T > 2:
        pos[1] = -1
    w = (rng.standard_normal(hs) + 1).astype(np.float32)
    wd = backend.vector(w)
    buf = backend.vector(x)
    at = lambda h: buf.view(shift + h * hs, (T - 1) * ld + (hk if h else hq) * hs)  # noqa: E731
    how = QkNormRope(hs, hq, hk, variant, 500000.0, 1e-6, wd, wd, q_ld=ld, k_ld=ld, q_out_ld=ld, k_out_ld=ld)
    ctx.qk_norm_rope(how, backend.vector(pos, np.int32), at(0), at(hq), at(0), at(hq))
    rows = x[shift:].reshape(T, ld)
    got = buf.to_numpy()[shift:].reshape(T, ld)
    heads = lambda a: a[:, :(hq + hk) * hs].reshape(T, hq + hk, hs)  # noqa: E731
    want, bound = R.norm_rope(heads(rows), w, 1e-6, variant, 500000.0, np.maximum(pos, 0))
    want[pos < 0], bound[pos < 0] = heads(rows)[pos < 0], 0
    check(heads(got), want, bound)
    assert (got[:, (hq + hk) * hs:] == rows[:, (hq + hk) * hs:]).all() and (buf.to_numpy()[:shift] == x[:shift]).all()


def test_norms_of_zeros_and_large_values(ctx, backend):
    hs = 64
    x = np.zeros((6, 1, hs), np.float32)
    x[1], x[2, 0, 3], x[3], x[4] = 1e-20, 1e18, np.linspace(-1e15, 1e15, hs), 2.0**-60
    x[5, 0, 7] = np.nan
    how = QkNormRope(hs, 1, 0, 0, 10000.0, 1e-5, backend.vector(np.ones(hs)))
    out = backend.zeros(x.size)
    pos = np.arange(6)
    ctx.qk_norm_rope(how, backend.vector(pos, np.int32), backend.vector(x), None, out, None)
    want, bound = R.norm_rope(x, np.ones(hs), 1e-5, 0, 10000.0, pos)
    check(out.to_numpy().reshape(x.shape), want, bound + 1e-37)


# ---- append ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hq, hk, hs, page, dtype, order, gap, shift, variant, norms, pos0, n_new", [
    (6, 6, 48, 16, F32, "pos", 0, 0, 0, False, [100], [1]),
    (32, 32, 128, 16, F16, "head", 0, 0, 0, False, [515, 0, 15, 16, 31, 1023], [1, 1, 1, 1, 1, 1]),
    (8, 1, 128, 64, F16, "head", 0, 0, 1, True, [0, 63, 64, 120], [70, 1, 130, 8]),
    (6, 2, 64, 20, F32, "head", 0, 0, 1, True, [7, 19, 20, 0], [33, 1, 0, 20]),
    (4, 4, 80, 7, F16, "pos", 0, 0, 0, True, [3, 13], [9, 15]),
    (5, 5, 65, 1, F16, "pos", 0, 0, None, True, [3, 0], [2, 4]),
    (4, 2, 96, 16, F16, "head", 8, 0, 0, True, [3, 0], [20, 40]),
    (4, 2, 64, 16, F16, "head", 3, 1, 1, True, [3, 0], [20, 40]),
    (4, 2, 256, 16, F16, "pos", 0, 0, 1, False, [3, 200], [20, 3])])
def test_paged_append(ctx, backend, hq, hk, hs, page, dtype, order, gap, shift, variant, norms, pos0, n_new):
    P = Pages(backend, hq, hk, hs, page, [p + n for p, n in zip(pos0, n_new)], dtype, order, gap, shift=shift, seed=hs)
    rows, rng = sum(n_new), P.rng
    ld = (hq + 2 * hk) * hs
    x = rng.standard_normal((rows, ld)).astype(np.float32) * 2
    wq, wk = (rng.standard_normal((2, hs)) + 1).astype(np.float32)
    buf = backend.vector(x)
    part = lambda h, n: buf.view(h * hs, (rows - 1) * ld + n * hs)  # noqa: E731
    how = QkNormRope(hs, hq, hk, variant, 10000.0, 1e-5, backend.vector(wq) if norms else None, backend.vector(wk) if norms else None, q_ld=ld, k_ld=ld, v_ld=ld)
    qo = backend.zeros(rows * hq * hs)
    P.kv.step(pos0, n_new, P.tables)
    ctx.paged_append(P.kv, P.layer, how, part(0, hq), part(hq, hk), part(hq + hk, hk), qo)
    pos = np.concatenate([np.arange(p, p + n) for p, n in zip(pos0, n_new)])
    x = x.reshape(rows, hq + 2 * hk, hs)
    check(qo.to_numpy().reshape(rows, hq, hs), *R.norm_rope(x[:, :hq], wq if norms else None, 1e-5, variant, 10000.0, pos))
    wk_, bk = R.norm_rope(x[:, hq:hq + hk], wk if norms else None, 1e-5, variant, 10000.0, pos)
    before = [h.copy() for h in P.host]
    P.download()
    at = 0
    for b, (p, n) in enumerate(zip(pos0, n_new)):
        new = np.arange(p, p + n)
        if n:
            check(P.at(0, b, new).astype(np.float64), wk_[at:at + n], R.stored(wk_[at:at + n], bk[at:at + n], dtype == F16), "keys")
            assert (P.at(1, b, new) == x[at:at + n, hq + hk:].astype(P.np_type)).all()  # one rounding
            P.put(0, b, new, before[0][P._index(b, new)])
            P.put(1, b, new, before[1][P._index(b, new)])
        at += n
    assert all((a == b).all() for a, b in zip(P.host, before))  # nothing else was touched


def test_append_without_queries(ctx, backend):
    P = Pages(backend, 4, 2, 64, 16, [20], F32)
    P.kv.step([3], [17], P.tables)
    k, v = (P.rng.standard_normal((17, 2, 64)).astype(np.float32) for _ in range(2))
    ctx.paged_append(P.kv, P.layer, QkNormRope(64, 0, 2, None), None, backend.vector(k), backend.vector(v), None)
    P.download()
    assert (P.at(0, 0, np.arange(3, 20)) == k).all() and (P.at(1, 0, np.arange(3, 20)) == v).all()


# ---- attention ---------------------------------------------------------------------------------------------------------
CASES = [
    # hq, hk, hs, page, pos0, n_new
    (1, 1, 128, 16, [0], [1]),                                # nothing but itself
    (32, 32, 128, 16, [515], [1]),
    (8, 1, 128, 16, [1030, 0, 15, 16, 63, 64, 127, 3000], [1] * 8),
    (16, 2, 128, 64, [5000], [1]),                            # one long sequence over many blocks
    (3, 1, 64, 16, [200, 7], [1, 1]),
    (10, 2, 64, 32, [130, 700, 0], [1, 3, 5]),                # a group of five, a few tokens each
    (24, 2, 128, 16, [300, 11], [1, 2]),                      # a group of twelve
    (20, 1, 128, 16, [300, 11], [1, 1]),                      # a group of twenty
    (4, 4, 128, 16, [0], [64]),
    (4, 4, 128, 16, [0, 37, 300], [1, 129, 17]),
    (8, 2, 128, 64, [0, 190, 65], [200, 33, 257]),            # chunks of several conversations
    (8, 2, 64, 16, [100, 0, 511, 3], [90, 300, 1, 1]),        # a chunk beside tokens
    (6, 6, 48, 16, [100], [1]),
    (6, 6, 48, 20, [0, 45], [50, 7]),
    (4, 2, 80, 32, [77, 0], [1, 100]),
    (5, 1, 96, 128, [77, 0], [3, 140]),
    (2, 2, 256, 16, [77, 0, 300], [1, 40, 1]),
    (2, 1, 65, 7, [20, 0], [1, 19]),                          # odd sizes
    (2, 1, 1, 1, [20, 0], [1, 3]),
    (3, 1, 20, 3, [2, 100], [3, 1]),
    # chunks through tiles of 256 rows: heads narrower than the tile, pages that divide 128 positions, that are divided by them, neither
    (3, 3, 48, 20, [0, 45], [150, 131]),
    (4, 2, 56, 8, [130], [129]),
    (2, 1, 64, 128, [100, 256], [140, 200]),
    (3, 1, 128, 24, [111], [131]),
    (2, 2, 104, 256, [300], [300]),
    (2, 1, 128, 16, [9000], [150]),                           # few tiles over many blocks
    (1, 1, 128, 512, [1000, 0], [128, 129]),
    (40, 1, 128, 16, [77], [20]),                             # a group wider than a warp
]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("order", ["head", "pos"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:4])) + f"-{sum(c[5])}t")
def test_paged_attention(ctx, backend, case, order, dtype):
    hq, hk, hs, page, pos0, n_new = case
    attend(ctx, Pages(backend, hq, hk, hs, page, [p + n for p, n in zip(pos0, n_new)], dtype, order, seed=hs + page), pos0, n_new)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hs, gap, shift, pad", [(128, 1, 0, 0), (128, 8, 0, 4), (64, 0, 1, 1), (64, 8, 8, 3), (128, 0, 0, 1)])
def test_strides_and_alignment(ctx, backend, hs, gap, shift, pad, dtype):
    P = Pages(backend, 4, 2, hs, 16, [70, 300, 40], dtype, gap=gap, shift=shift, seed=5)
    attend(ctx, P, [69, 140, 0], [1, 160, 40], q_ld=4 * hs + pad if pad else 0, out_ld=4 * hs + 2 * pad if pad else 0)


@pytest.mark.parametrize("n_new", [[1, 1, 1], [130, 20, 1]])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_what_a_row_does_not_see_does_not_reach_it(ctx, backend, n_new, dtype):
    """Infinities and NaN in pages nobody uses, behind the last position, and in the values of tokens that follow a row's own."""
    pos0 = [100, 0, 33]
    P = Pages(backend, 8, 2, 128, 16, [p + n for p, n in zip(pos0, n_new)], dtype, seed=3)
    keep = [[P.at(w, b, np.arange(p + n)) for b, (p, n) in enumerate(zip(pos0, n_new))] for w in range(2)]
    for w in range(2):
        P.host[w][:] = np.nan
        P.host[w][::3] = np.inf
        for b in range(3):
            P.put(w, b, np.arange(len(keep[w][b])), keep[w][b])
    if n_new[0] > 1:  # tokens 60 and 128 of a chunk have a value that overflowed, token 90 a key
        for w, t, x in ((1, 60, np.inf), (1, 128, -np.inf), (0, 90, np.nan)):
            row = P.at(w, 0, [pos0[0] + t])
            row[0, 0, 5] = x
            P.put(w, 0, [pos0[0] + t], row)
    P.upload()
    attend(ctx, P, pos0, n_new)


def test_infinite_scores_and_values_follow_the_formula(ctx, backend):
    P = Pages(backend, 4, 2, 128, 16, [90, 200], F32, seed=4)
    for b, pos, w, h, x in ((0, 30, 1, 0, np.inf), (1, 100, 0, 1, np.inf)):
        row = P.at(w, b, [pos])
        row[0, h, :] = x if w == 1 else 0
        if w == 0:
            row[0, h, 3] = x
        P.put(w, b, [pos], row)
    P.upload()
    q = P.rng.standard_normal((2, 4, 128)).astype(np.float32)
    q[1, 2, 3], q[1, 3, 3] = -2.0, 2.0   # a score of -inf (weight zero), one of +inf (NaN)
    attend(ctx, P, [89, 199], [1, 1], q=q)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("size", [1e-30, 1e-3, 1.0, 30.0])
def test_sizes_of_queries(ctx, backend, size, dtype):
    P = Pages(backend, 8, 2, 128, 16, [190, 400], dtype, seed=6)
    q = (P.rng.standard_normal((1 + 140, 8, 128)) * size).astype(np.float32)
    attend(ctx, P, [189, 260], [1, 140], q=q)


@pytest.mark.parametrize("keys, values", [(1e-25, 1e30), (1e25, 1e-30), (1e-33, 1e-33), (1e30, 3e35)])
@pytest.mark.parametrize("hs, page", [(128, 16), (72, 40)])
def test_sizes_of_f32_keys_and_values(ctx, backend, keys, values, hs, page):
    """Far beyond halves; the queries make up for the keys, so that scores are the usual ones."""
    P = Pages(backend, 4, 2, hs, page, [150, 400, 61], F32, seed=12)
    P.host[0] *= np.float32(keys)
    P.host[1] *= np.float32(values)
    P.upload()
    q = (P.rng.standard_normal((37 + 140 + 3, 4, hs)) * 2 / keys).astype(np.float32)
    attend(ctx, P, [113, 260, 58], [37, 140, 3], q=q)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hq, hk", [(16, 16), (24, 8)])
def test_many_short_chunks(ctx, backend, hq, hk, dtype):
    """Several pairs to a block, most of them of one unit or two."""
    rng = np.random.default_rng(13)
    n_new = [int(x) for x in rng.integers(17, 61, 40)]
    pos0 = [int(x) for x in rng.integers(0, 90, 40) * (rng.random(40) < 0.5)]
    n_new[7], n_new[20], n_new[21] = 140, 1, 0
    attend(ctx, Pages(backend, hq, hk, 128, 16, [p + n for p, n in zip(pos0, n_new)], dtype, "pos", seed=13), pos0, n_new)


def test_keys_far_from_zero_and_scale(ctx, backend):
    P = Pages(backend, 4, 2, 128, 16, [300, 150], F16, seed=7)
    for b, n in ((0, 300), (1, 150)):
        P.put(0, b, np.arange(n), P.at(0, b, np.arange(n)) * np.float16(8) + np.float16(20))
    P.upload()
    attend(ctx, P, [299, 0], [1, 150], scale=0.03)
    attend(ctx, P, [299, 0], [1, 150], scale=-0.02)


def test_shared_pages_and_sequences_that_take_no_part(ctx, backend):
    P = Pages(backend, 4, 2, 128, 16, [64, 70, 70, 40], F16, seed=8)
    P.tables[1, :4] = P.tables[0, :4]   # a common prefix, read by both
    P.tables[3, 0] = -5                 # takes no part: its table is not looked at
    attend(ctx, P, [64, 64, 65, 39], [0, 6, 5, 0])


def test_a_step_without_tokens(ctx, backend):
    P = Pages(backend, 4, 2, 64, 16, [10], F16)
    P.kv.step([5], [0], P.tables)
    out = backend.vector(np.full(16, 2.5))
    ctx.paged_attention(P.kv, P.layer, backend.zeros(16), out)
    ctx.paged_append(P.kv, P.layer, QkNormRope(64, 4, 2), backend.zeros(1), backend.zeros(1), backend.zeros(1), out)
    assert (out.to_numpy() == 2.5).all()


def test_results_repeat(ctx, backend):
    """Bit for bit, run after run: sums over blocks are taken in the order of their positions."""
    P = Pages(backend, 16, 2, 128, 16, [3000, 1500, 40, 700], F16, seed=9)
    pos0, n_new = [2999, 1499, 39, 500], [1, 1, 1, 200]
    q = P.rng.standard_normal((203, 16, 128)).astype(np.float32)
    first = attend(ctx, P, pos0, n_new, q=q)
    qd, out = backend.vector(q), backend.zeros(q.size)
    for _ in range(5):
        ctx.paged_attention(P.kv, P.layer, qd, out)
        assert (out.to_numpy().reshape(first.shape) == first).all()


@pytest.mark.parametrize("n_new", [[1, 1], [140, 1]])
def test_a_cache_beyond_32_bits(ctx, backend, n_new):
    """Pages 2^28 elements apart: the last lie 5 GB behind the first."""
    hq, hk, hs, page, n_pages, stride = 4, 2, 128, 64, 11, 1 << 28
    rng = np.random.default_rng(2)
    free, _ = backend.mem_info()
    assert free > 3 * n_pages * stride * 2

    class Far:  # a buffer of n elements
        def __init__(self):
            self.n = (n_pages - 1) * stride + hk * page * hs
            self.ptr = backend.malloc(self.n * 2)

        def __len__(self):
            return self.n

    keys, values = Far(), Far()
    try:
        kv = PagedKv(backend, hq, hk, hs, page, n_pages, F16, max_seqs=2, max_tokens=200)
        layer = PagedLayer(keys, values, stride, page * hs, hs)
        tables = np.array([[10, 9, 0, 8], [7, 6, 5, -1]], np.int32)
        pos0 = [100, 130]
        held = [[rng.standard_normal((p + n, hk, hs)).astype(np.float16) for p, n in zip(pos0, n_new)] for _ in range(2)]
        for w, buf in enumerate((keys, values)):
            for b in range(2):
                x = held[w][b]
                for i in range(-(-len(x) // page)):
                    block = np.zeros((hk, page, hs), np.float16)
                    part = x[i * page:(i + 1) * page]
                    block[:, :len(part)] = part.transpose(1, 0, 2)
                    backend.write_buffer(buf.ptr + int(tables[b, i]) * stride * 2, block)
        kv.step(pos0, n_new, tables)
        rows = sum(n_new)
        # the step's own keys and values go in by the append (no norm, no rotation)
        k, v = (np.concatenate([held[w][b][p:] for b, p in enumerate(pos0)]).astype(np.float32) for w in range(2))
        ctx.paged_append(kv, layer, QkNormRope(hs, 0, hk, None), None, backend.vector(k), backend.vector(v), None)
        q, out = rng.standard_normal((rows, hq, hs)).astype(np.float32), backend.zeros(rows * hq * hs)
        ctx.paged_attention(kv, layer, backend.vector(q), out)
        got, at = out.to_numpy().reshape(rows, hq, hs), 0
        for b, (p, n) in enumerate(zip(pos0, n_new)):
            check(got[at:at + n], *R.attention(q[at:at + n], held[0][b], held[1][b], p, hs**-0.5))
            at += n
    finally:
        for buf in (keys, values):
            backend.free(buf.ptr)


# ---- together ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype, hs, hq, hk, page, variant", [(F16, 128, 8, 2, 16, 0), (F32, 48, 6, 6, 20, 1), (F16, 64, 4, 4, 64, 1)])
def test_conversations_in_pages(ctx, backend, dtype, hs, hq, hk, page, variant):
    """Prompts in chunks, then tokens beside another prompt, two layers: each layer's attention against 64-bit arithmetic over every token so far."""
    rng = np.random.default_rng(11)
    layers = [Pages(backend, hq, hk, hs, page, [170, 120, 90], dtype, max_tokens=150, seed=s) for s in (1, 1)]
    kv, tables = layers[0].kv, layers[0].tables
    w = (1 + 0.2 * rng.standard_normal((2, hs))).astype(np.float32)
    wd = [backend.vector(x) for x in w]
    ld = (hq + 2 * hk) * hs
    how = QkNormRope(hs, hq, hk, variant, 10000.0, 1e-5, *wd, q_ld=ld, k_ld=ld, v_ld=ld)
    held, pos = [[([], []) for _ in range(3)] for _ in layers], [0, 0, 0]
    for n_new in ([100, 0, 0], [50, 90, 0], [1, 1, 80], [1, 1, 1], [3, 0, 1]):
        kv.step(pos, n_new, tables)
        rows = sum(n_new)
        for P, hold in zip(layers, held):
            x = rng.standard_normal((rows, ld)).astype(np.float32)
            buf, qo, out = backend.vector(x), backend.zeros(rows * hq * hs), backend.zeros(rows * hq * hs)
            part = lambda h, n: buf.view(h * hs, (rows - 1) * ld + n * hs)  # noqa: E731
            ctx.paged_append(kv, P.layer, how, part(0, hq), part(hq, hk), part(hq + hk, hk), qo)
            ctx.paged_attention(kv, P.layer, qo, out)
            got, q = (a.to_numpy().reshape(rows, hq, hs) for a in (out, qo))
            P.download()
            at = 0
            for b, n in enumerate(n_new):
                if n:
                    heads = x[at:at + n].reshape(n, -1, hs)
                    here = np.arange(pos[b], pos[b] + n)
                    want_k, bound_k = R.norm_rope(heads[:, hq:hq + hk], w[1], 1e-5, variant, 10000.0, here)
                    cached = P.at(0, b, here)
                    check(cached.astype(np.float64), want_k, R.stored(want_k, bound_k, dtype == F16), "keys")
                    check(q[at:at + n], *R.norm_rope(heads[:, :hq], w[0], 1e-5, variant, 10000.0, here))
                    hold[b][0].append(cached)
                    hold[b][1].append(heads[:, hq + hk:].astype(P.np_type))
                    want, bound = R.attention(q[at:at + n], np.concatenate(hold[b][0]), np.concatenate(hold[b][1]), pos[b], hs**-0.5)
                    check(got[at:at + n], want, bound, f"sequence {b} at {pos[b]}")
                at += n
        pos = [p + n for p, n in zip(pos, n_new)]


@pytest.mark.parametrize("dtype", [F16, F32])
def test_a_recorded_pass_follows_the_steps(ctx, backend, dtype):
    """Append and attention recorded once, replayed for steps of other lengths: tokens only, a chunk beside tokens, fewer sequences."""
    hq, hk, hs = 8, 2, 128
    P = Pages(backend, hq, hk, hs, 16, [260, 200, 150], dtype, max_tokens=160, seed=12)
    how = QkNormRope(hs, hq, hk, 1)
    q, qo, out = (backend.zeros(160 * hq * hs) for _ in range(3))
    k, v = (backend.zeros(160 * hk * hs) for _ in range(2))

    def fill(rows):
        xs = [P.rng.standard_normal((160, h, hs)).astype(np.float32) for h in (hq, hk, hk)]
        for d, x in zip((q, k, v), xs):
            backend.write_buffer(d.ptr, x)
        return [x[:rows] for x in xs]

    def verify(pos0, n_new, xs):
        rows = sum(n_new)
        got = out.to_numpy().reshape(160, hq, hs)
        assert (got[rows:] == 4.5).all() and (qo.to_numpy().reshape(160, hq, hs)[rows:] == 4.5).all()
        rot = qo.to_numpy().reshape(160, hq, hs)[:rows]
        P.download()
        at = 0
        for b, (p, n) in enumerate(zip(pos0, n_new)):
            if n:
                here = np.arange(p, p + n)
                check(rot[at:at + n], *R.norm_rope(xs[0][at:at + n], None, 0, 1, 10000.0, here))
                assert (P.at(1, b, here) == xs[2][at:at + n].astype(P.np_type)).all()
                want, bound = R.attention(rot[at:at + n], P.at(0, b, np.arange(p + n)), P.at(1, b, np.arange(p + n)), p, hs**-0.5)
                check(got[at:at + n], want, bound, f"sequence {b}")
            at += n

    def clear():
        for d in (qo, out):
            backend.write_buffer(d.ptr, np.full(160 * hq * hs, 4.5, np.float32))

    calls = lambda: (ctx.paged_append(P.kv, P.layer, how, q, k, v, qo), ctx.paged_attention(P.kv, P.layer, qo, out))  # noqa: E731
    P.kv.step([259, 199, 0], [1, 1, 0], P.tables)
    calls()
    with backend.record() as rec:
        calls()
    for pos0, n_new in (([259, 199, 149], [1, 1, 1]), ([100, 199, 0], [150, 1, 0]), ([0, 0, 0], [0, 0, 0]), ([3, 199, 100], [2, 0, 50]), ([259, 0, 0], [1, 0, 0])):
        P.kv.step(pos0, n_new, P.tables)
        xs = fill(sum(n_new))
        clear()
        rec.launch(2)
        verify(pos0, n_new, xs)
    rec.close()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hq, hk, n_new", [(16, 8, [1] * 40), (16, 16, [131] * 9), (16, 8, [1] * 20 + [100] * 9)])
def test_a_recorded_pass_with_many_pairs_on_several_blocks(ctx, backend, hq, hk, n_new, dtype):
    """More joins than a recorded launch has blocks for at once.  (A recorded call may join in another order than the step's own: held to the formula's bound, not to
    that call's bits; its replays have the same bits.)"""
    rng = np.random.default_rng(21)
    pos0 = [int(x) for x in rng.integers(300, 1200, len(n_new))]
    P = Pages(backend, hq, hk, 128, 16, [p + n for p, n in zip(pos0, n_new)], dtype, seed=21)
    rows = sum(n_new)
    q = rng.standard_normal((rows, hq, 128)).astype(np.float32) * 2
    P.kv.step(pos0, n_new, P.tables)
    most = P.kv.max_tokens * hq * 128
    qd, out = backend.zeros(most), backend.vector(np.full(most, 4.5, np.float32))
    backend.write_buffer(qd.ptr, q.reshape(-1))
    with backend.record() as rec:
        ctx.paged_attention(P.kv, P.layer, qd, out)
    rec.launch()
    got, at = out.to_numpy(), 0
    rec.launch()
    assert np.array_equal(got, out.to_numpy()) and (got[q.size:] == 4.5).all()
    rec.close()
    for b, (p, n) in enumerate(zip(pos0, n_new)):
        held = np.arange(p + n)
        want, bound = R.attention(q[at:at + n], P.at(0, b, held), P.at(1, b, held), p, 128**-0.5)
        check(got[:q.size].reshape(q.shape)[at:at + n], want, bound, f"sequence {b}")
        at += n


def test_two_handles_and_two_contexts(ctx, backend):
    """Handles of one context alternate; another context on the same GPU works beside them."""
    from slai_b200.ops import Backend, LlmContext
    other = Backend(0)
    try:
        octx = LlmContext(other)
        a, b = (Pages(backend, 8, 2, 128, 16, [900, 500], F16, seed=s) for s in (1, 2))
        c = Pages(other, 8, 2, 128, 16, [900, 500], F16, seed=3)
        for P, cx in ((a, ctx), (c, octx), (b, ctx), (a, ctx), (c, octx)):
            attend(cx, P, [899, 400], [1, 100])
        del c, P
    finally:
        other.close()


# ---- refusals ----------------------------------------------------------------------------------------------------------
def refused(code, word, f, *args, **kw):
    with pytest.raises(SlaiError, match=word) as e:
        f(*args, **kw)
    assert e.value.code == code


def test_refusals(ctx, backend):
    S, I = _lib.ERR_SHAPE, _lib.ERR_INVALID_ARG
    refused(S, "n_kv_heads", PagedKv, backend, 6, 4, 64, 16, 10)
    refused(S, "head_size", PagedKv, backend, 4, 4, 257, 16, 10)
    P = Pages(backend, 4, 2, 64, 16, [40, 20], F16)
    buf = backend.zeros(4 * 64 * 60)
    refused(I, "slai_paged_step comes first", ctx.paged_attention, P.kv, P.layer, buf, buf)
    refused(S, "no such page", P.kv.step, [39, 19], [1, 1], np.full((2, 3), P.n_pages))
    refused(S, "used twice", P.kv.step, [39, 19], [1, 1], np.full((2, 3), 1))
    refused(S, "tables", P.kv.step, [39, 19], [1], P.tables)
    P.kv.step([39, 19], [1, 1], P.tables)
    refused(S, "max_tokens", P.kv.step, [0, 0], [40, 40], np.arange(6).reshape(2, 3))
    refused(S, "floats for", ctx.paged_attention, P.kv, P.layer, backend.zeros(4 * 64), buf)
    refused(S, "shorter", ctx.paged_attention, P.kv, P.layer, buf, buf, q_ld=255)
    refused(I, "scale", ctx.paged_attention, P.kv, P.layer, buf, buf, scale=float("nan"))
    refused(S, "elements", ctx.paged_attention, P.kv, PagedLayer(P.dev[0], backend.zeros(5, np.float16), *P.strides), buf, buf)
    refused(S, "strides", ctx.paged_attention, P.kv, PagedLayer(*P.dev, P.strides[0], 63, 64), buf, buf)
    refused(I, "unknown rotation", ctx.qk_norm_rope, QkNormRope(64, 4, 2, 3), backend.zeros(1, np.int32), buf, buf, buf, buf)
    refused(S, "even head_size", ctx.qk_norm_rope, QkNormRope(63, 4, 2, 1), backend.zeros(1, np.int32), buf, buf, buf, buf)
    refused(I, "base frequency", ctx.qk_norm_rope, QkNormRope(64, 4, 2, 1, 0.0), backend.zeros(1, np.int32), buf, buf, buf, buf)
    refused(S, "shorter", ctx.qk_norm_rope, QkNormRope(64, 4, 2, 1, q_ld=64), backend.zeros(1, np.int32), buf, buf, buf, buf)
    refused(S, "not the cache's", ctx.paged_append, P.kv, P.layer, QkNormRope(128, 4, 2), buf, buf, buf, buf)
    refused(S, "not the cache's", ctx.paged_append, P.kv, P.layer, QkNormRope(64, 4, 4), buf, buf, buf, buf)
    refused(I, "out cannot be q", ctx.paged_attention, P.kv, P.layer, buf, buf)
    refused(S, "elements of 4", ctx.paged_attention, Pages(backend, 4, 2, 64, 16, [40, 20], F32).kv, P.layer, buf, buf)  # f16 pages for an f32 cache
    two, out = backend.zeros(4 * 64 * 2), backend.zeros(4 * 64 * 60)
    with backend.record() as rec:
        refused(I, "recorded", P.kv.step, [39, 19], [1, 1], P.tables)
        refused(I, "recorded", ctx.qk_norm_rope, QkNormRope(64, 4, 2, 1, 12345.0), backend.pos if hasattr(backend, "pos") else buf.view(0, 1), buf, buf, buf, buf)
        refused(S, "floats for 60 rows", ctx.paged_attention, P.kv, P.layer, buf, two)  # (other steps come)
        refused(S, "floats for 60 rows", ctx.paged_append, P.kv, P.layer, QkNormRope(64, 4, 2, None), buf, two, two, buf)
        ctx.paged_attention(P.kv, P.layer, buf, out)
    rec.close()
    attend(ctx, P, [39, 19], [1, 1])  # and goes on
