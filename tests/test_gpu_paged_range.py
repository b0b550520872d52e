"""Paged operators over the range that their header allows: small and odd heads, wide groups, orders of memory, far positions, rows far apart."""
import numpy as np
import pytest

import paged_bounds as B
import paged_reference as R
from slai_b200._lib import KV_F16, KV_F32
from slai_b200.ops import PagedKv, PagedLayer, QkNormRope
from test_gpu_paged import Pages, check
from test_gpu_paged_accuracy import run

pytestmark = pytest.mark.gpu
F16, F32 = KV_F16, KV_F32


def near(P, got, q, pos0, n_new, scale=None):
    at = 0
    for b, (p, n) in enumerate(zip(pos0, n_new)):
        if n:
            held = np.arange(p + n)
            want, bound = B.attention(q[at:at + n], P.at(0, b, held), P.at(1, b, held), p, scale or P.hs**-0.5, P.dtype == F16)
            assert not B.far_rows(got[at:at + n], want, bound).any(), f"sequence {b}"
        at += n


def queries(P, rows):
    return (P.rng.standard_normal((rows, P.hq, P.hs)) * 2).astype(np.float32)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hs", [2, 4, 8, 12, 16, 24, 32, 40, 72, 88, 112, 120, 124, 136, 200])
def test_head_sizes(ctx, backend, hs, dtype):
    pos0, n_new = [300, 0, 77], [1, 140, 3]
    P = Pages(backend, 4, 2, hs, 16, [p + n for p, n in zip(pos0, n_new)], dtype, seed=hs)
    q = queries(P, sum(n_new))
    near(P, run(ctx, P, pos0, n_new, q), q, pos0, n_new)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hq, hk, n_new", [(7, 1, [1, 20]), (128, 1, [1, 2]), (66, 2, [1, 5]), (300, 1, [1, 1]), (9, 9, [2, 17])])
def test_groups(ctx, backend, hq, hk, n_new, dtype):
    pos0 = [200, 40]
    P = Pages(backend, hq, hk, 64, 16, [p + n for p, n in zip(pos0, n_new)], dtype, seed=hq)
    q = queries(P, sum(n_new))
    near(P, run(ctx, P, pos0, n_new, q), q, pos0, n_new)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("page", [1, 2, 4, 8, 100, 1000, 1024])
def test_page_sizes_under_chunks_and_tokens(ctx, backend, page, dtype):
    pos0, n_new = [300, 130, 9], [1, 150, 40]
    P = Pages(backend, 4, 2, 128, page, [p + n for p, n in zip(pos0, n_new)], dtype, seed=page)
    q = queries(P, sum(n_new))
    near(P, run(ctx, P, pos0, n_new, q), q, pos0, n_new)


class Laid(Pages):
    """Pages in any order of memory: `order` names the dimensions from the outermost on (p page, h head, s place); keys and values `both` in one buffer, side by side."""

    def __init__(self, be, order, both, *args, **kw):
        super().__init__(be, *args, **kw)
        n, step = {"p": self.n_pages, "h": self.hk, "s": self.page}, {}
        size = self.hs * (2 if both else 1)
        for d in reversed(order):
            step[d] = size
            size *= n[d]
        self.strides = (step["p"], step["h"], step["s"])
        if both:
            host = self.rng.standard_normal(size).astype(self.np_type)
            buf = be.vector(host, self.np_type)
            self.host = [host[:size - self.hs], host[self.hs:]]
            self.dev = [buf.view(0, size - self.hs), buf.view(self.hs, size - self.hs)]
            self.whole = buf
        else:
            self.host = [self.rng.standard_normal(size).astype(self.np_type) for _ in range(2)]
            self.dev = [be.vector(a, self.np_type) for a in self.host]
        self.layer = PagedLayer(*self.dev, *self.strides)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("order", ["phs", "psh", "hps", "hsp", "sph", "shp"])
def test_orders_of_memory(ctx, backend, order, both, dtype):
    """Append, then attention."""
    hq, hk, hs, pos0, n_new = 6, 2, 64, [300, 130, 9], [1, 150, 17]
    P = Laid(backend, order, both, hq, hk, hs, 16, [p + n for p, n in zip(pos0, n_new)], dtype, seed=len(order))
    rows = sum(n_new)
    q, k, v = queries(P, rows), *(P.rng.standard_normal((rows, hk, hs)).astype(np.float32) for _ in range(2))
    P.kv.step(pos0, n_new, P.tables)
    ctx.paged_append(P.kv, P.layer, QkNormRope(hs, 0, hk, None), None, backend.vector(k), backend.vector(v), None)
    at = 0
    for b, (p, n) in enumerate(zip(pos0, n_new)):
        P.put(0, b, np.arange(p, p + n), k[at:at + n].astype(P.np_type))
        P.put(1, b, np.arange(p, p + n), v[at:at + n].astype(P.np_type))
        at += n
    for d, h in zip(P.dev, P.host):
        assert np.array_equal(d.to_numpy(), h)
    near(P, run(ctx, P, pos0, n_new, q), q, pos0, n_new)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_a_read_page_several_times(ctx, backend, dtype):
    """One page over and over in one sequence, in several, and only read by all of them."""
    pos0, n_new = [7 * 16 + 3, 200, 70], [5, 1, 90]
    P = Pages(backend, 4, 2, 128, 16, [p + n for p, n in zip(pos0, n_new)], dtype, seed=2)
    P.tables[0, :7], P.tables[1, 2:9], P.tables[2, :4] = P.tables[1, 0], P.tables[1, 0], P.tables[1, 0]
    P.kv = PagedKv(backend, 4, 2, 128, 16, P.n_pages, dtype, max_seqs=3, max_tokens=96)
    q = queries(P, 96)
    near(P, run(ctx, P, pos0, n_new, q), q, pos0, n_new)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_many_sequences(ctx, backend, dtype):
    rng = np.random.default_rng(3)
    pos0 = [int(x) for x in rng.integers(0, 130, 700)]
    n_new = [int(x) for x in rng.choice([0, 1, 1, 1, 1, 2, 20], 700)]
    P = Pages(backend, 2, 1, 64, 16, [p + n for p, n in zip(pos0, n_new)], dtype, seed=3)
    q = queries(P, sum(n_new))
    near(P, run(ctx, P, pos0, n_new, q), q, pos0, n_new)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hq, tokens, far", [(1, 1, 2047), (1, 3, 1024), (8, 1, 512), (2, 40, 64)])
def test_positions_near_the_largest(ctx, backend, hq, tokens, far, dtype):
    """One page of 2^20 positions read `far` - 1 times over, then the one that the new tokens are in (its other places have keys that nobody looks at twice): up to position
    2^31 - 2^20 - 1.  The scores repeat, so the weights of a place add up: softmax over one page, each score with the page's share."""
    page, hs = 1 << 20, 8
    rng = np.random.default_rng(far)
    np_type = np.float16 if dtype == F16 else np.float32
    keys, values = (rng.standard_normal((2, page, hs)).astype(np_type) for _ in range(2))
    kv = PagedKv(backend, hq, 1, hs, page, 2, dtype, max_seqs=1, max_tokens=tokens, max_table=far)
    layer = PagedLayer(backend.vector(keys, np_type), backend.vector(values, np_type), page * hs, page * hs, hs)
    table = np.zeros((1, far), np.int32)
    table[0, -1] = 1
    pos0 = far * page - tokens
    kv.step([pos0], [tokens], table)
    q = rng.standard_normal((tokens, hq, hs)).astype(np.float32)
    out = backend.zeros(q.size)
    ctx.paged_attention(kv, layer, backend.vector(q), out)
    backend.synchronize()
    got = out.to_numpy().reshape(q.shape)
    k, v = keys.astype(np.float64), values.astype(np.float64)
    for t in range(0, tokens, 13):
        for h in range(hq):
            seen = [page, page - tokens + t + 1]
            s = [k[i, :seen[i]] @ q[t, h] * hs**-0.5 for i in range(2)]
            m = max(x.max() for x in s)
            w = [np.exp(s[0] - m) * (far - 1), np.exp(s[1] - m)]
            want = (w[0] @ v[0, :seen[0]] + w[1] @ v[1, :seen[1]]) / (w[0].sum() + w[1].sum())
            # weights: 2 (hs + 8) half steps of the scores' sizes, twice; sums of far * page positions: at least 296 / hq blocks have each an equal share of
            # them in turn, at least 8 at a time, each addition off by half a step of the sum so far at most, the smaller share of all roundings one way:
            # sqrt(additions) half steps of the largest, with room of four; all of the mean of the values' sizes
            sizes = max((np.abs(k[i, :seen[i]]) @ np.abs(q[t, h])).max() for i in range(2)) * hs**-0.5
            mean = (w[0] @ np.abs(v[0, :seen[0]]) + w[1] @ np.abs(v[1, :seen[1]])) / (w[0].sum() + w[1].sum())
            bound = mean * 2.0**-24 * (2 * (2 * (hs + 8) * sizes + 4 * sizes) + 4 * 2 * np.sqrt(far * page / 8))
            assert (np.abs(got[t, h] - want) <= bound).all(), (t, h, np.abs(got[t, h] - want).max(), bound.min())


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("n_new", [[1, 1], [1, 40]])
def test_rows_far_apart(ctx, backend, n_new, dtype):
    """Leading dimensions of q, k, v and of the results whose product with a row's number passes 32 bits (in floats)."""
    hq, hk, hs, pos0 = 4, 2, 64, [90, 20]
    rows = sum(n_new)
    ld = ((1 << 31) + 256) // (rows - 1) // 8 * 8 + 8
    P = Pages(backend, hq, hk, hs, 16, [p + n for p, n in zip(pos0, n_new)], dtype, seed=9)
    x = P.rng.standard_normal((rows, hq + 2 * hk, hs)).astype(np.float32)
    n = (rows - 1) * ld + (hq + 2 * hk) * hs
    assert backend.mem_info()[0] > 3 * 4 * n

    class Far:
        def __init__(self, ptr, n):
            self.ptr, self.n = ptr, n

        def __len__(self):
            return self.n

    base = [backend.malloc(4 * n) for _ in range(2)]
    try:
        for r in range(rows):
            backend.write_buffer(base[0] + 4 * r * ld, x[r])
        at = lambda i, h, heads: Far(base[i] + 4 * h * hs, (rows - 1) * ld + heads * hs)  # noqa: E731
        lds = dict(q_ld=ld, k_ld=ld, v_ld=ld, q_out_ld=ld, k_out_ld=ld)
        q, k, v, qo, ko = at(0, 0, hq), at(0, hq, hk), at(0, hq + hk, hk), at(1, 0, hq), at(1, hq, hk)
        P.kv.step(pos0, n_new, P.tables)
        pos = np.concatenate([np.arange(p, p + m) for p, m in zip(pos0, n_new)])
        read = lambda i, h, heads: np.stack([backend.read_buffer(base[i] + 4 * (r * ld + h * hs), np.empty((heads, hs), np.float32)) for r in range(rows)])  # noqa: E731
        ctx.qk_norm_rope(QkNormRope(hs, hq, hk, 0, **lds), backend.vector(pos, np.int32), q, k, qo, ko)
        want, bound = R.norm_rope(x[:, :hq + hk], None, 0, 0, 10000.0, pos)
        check(read(1, 0, hq + hk), want, bound)
        ctx.paged_append(P.kv, P.layer, QkNormRope(hs, hq, hk, 1, **lds), q, k, v, qo)
        want, bound = R.norm_rope(x[:, :hq + hk], None, 0, 1, 10000.0, pos)
        rotated = read(1, 0, hq)
        check(rotated, want[:, :hq], bound[:, :hq])
        P.download()
        first = 0
        for b, (p, m) in enumerate(zip(pos0, n_new)):
            new = np.arange(p, p + m)
            check(P.at(0, b, new).astype(np.float64), want[first:first + m, hq:], R.stored(want[first:first + m, hq:], bound[first:first + m, hq:], dtype == F16))
            assert np.array_equal(P.at(1, b, new), x[first:first + m, hq + hk:].astype(P.np_type))
            first += m
        ctx.paged_attention(P.kv, P.layer, qo, at(1, hq, hq), 0.0, ld, ld)  # results between the queries' rows
        near(P, read(1, hq, hq), rotated, pos0, n_new)
    finally:
        for p in base:
            backend.free(p)
