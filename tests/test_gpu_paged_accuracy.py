"""Paged attention, row by row as near to its formula as its operands allow (paged_bounds.py), and exact about infinities."""
import numpy as np
import pytest

import paged_bounds as B
from slai_b200._lib import KV_F16, KV_F32
from test_gpu_paged import Pages

pytestmark = pytest.mark.gpu
F16, F32 = KV_F16, KV_F32


def run(ctx, P, pos0, n_new, q, recorded=False):
    be, most = ctx.backend, P.kv.max_tokens * P.hq * P.hs
    P.kv.step(pos0, n_new, P.tables)
    qd, out = be.vector(np.resize(q.reshape(-1), most)), be.zeros(most)
    if recorded:
        with be.record() as rec:
            ctx.paged_attention(P.kv, P.layer, qd, out)
        rec.launch()
    else:
        ctx.paged_attention(P.kv, P.layer, qd, out)
    got = out.to_numpy()[:q.size].reshape(q.shape)
    if recorded:
        rec.close()
    return got


CASES = [
    # hq, hk, hs, page, pos0, n_new
    (32, 32, 128, 16, [515], [1]),                     # a head to a cache head: f32 tiles of one row
    (16, 4, 128, 16, [515, 1200, 60], [1, 1, 2]),      # four
    (16, 2, 128, 16, [515, 1200, 60], [1, 1, 1]),      # eight
    (16, 2, 64, 20, [700, 33], [1, 3]),                # pages that are no multiple of 16
    (16, 2, 128, 64, [9000], [1]),                     # over many blocks
    (24, 2, 128, 16, [600, 50], [1, 1]),               # twelve
    (5, 1, 96, 32, [700, 0], [1, 2]),
    (8, 8, 128, 16, [0], [64]),
    (8, 2, 128, 16, [300, 0], [37, 90]),               # chunks
    (8, 8, 128, 16, [0], [300]),
    (8, 1, 128, 64, [700], [100]),
    (6, 3, 64, 16, [100, 256], [150, 140]),
    (6, 6, 48, 20, [45], [140]),
    (4, 2, 104, 256, [300], [200]),
    (4, 1, 128, 16, [5000], [140]),                    # few tiles over many blocks
    (4, 2, 256, 16, [400, 0], [1, 40]),                # f32 arithmetic
    (3, 1, 65, 7, [300, 0], [1, 50]),
]


@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:4])) + f"-{sum(c[5])}t")
def test_rows(ctx, backend, case, dtype, recorded):
    hq, hk, hs, page, pos0, n_new = case
    P = Pages(backend, hq, hk, hs, page, [p + n for p, n in zip(pos0, n_new)], dtype, seed=hs + hq, max_tokens=sum(n_new) + 3)
    q = (P.rng.standard_normal((sum(n_new), hq, hs)) * 2).astype(np.float32)
    got, at = run(ctx, P, pos0, n_new, q, recorded), 0
    for b, (p, n) in enumerate(zip(pos0, n_new)):
        held = np.arange(p + n)
        want, bound = B.attention(q[at:at + n], P.at(0, b, held), P.at(1, b, held), p, hs**-0.5, dtype == F16)
        far = B.far_rows(got[at:at + n], want, bound)
        off = np.sqrt(((got[at:at + n].astype(np.float64) - want) ** 2).sum(-1)) / bound
        assert not far.any(), f"sequence {b}: {int(far.sum())} of {far.size} rows, by up to {off.max()} times the bound, first at {tuple(np.argwhere(far)[0])}"
        at += n


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hq, hk, hs", [(4, 4, 128), (8, 4, 128), (16, 2, 128), (8, 4, 72), (8, 4, 65)])
@pytest.mark.parametrize("pos0, n_new", [([90, 200], [1, 1]), ([6000], [1]), ([90, 61], [150, 40]), ([3000], [140]), ([100, 300], [260, 1])])
def test_infinities(ctx, backend, hq, hk, hs, pos0, n_new, dtype):
    """Where a row is computed by one block or joined from many, by tokens' kernels, by chunks' and by the one for odd sizes."""
    P = Pages(backend, hq, hk, hs, 16, [p + n for p, n in zip(pos0, n_new)], dtype, seed=hq)
    q = P.rng.standard_normal((sum(n_new), hq, hs)).astype(np.float32)

    def put(which, b, pos, head, d, x):
        row = P.at(which, b, [pos])
        row[0, head, d] = x
        P.put(which, b, [pos], row)

    group = hq // hk
    for b, (p, n) in enumerate(zip(pos0, n_new)):
        put(0, b, p // 3, 0, 3, np.inf)             # cache head 0: a key that is infinite: scores of either sign, by the query
        put(1, b, p // 3 + 1, 0, 9, np.inf)         # ... a value in one dimension
        put(1, b, p // 2, 1, 5, np.inf)             # cache head 1: values of either sign, in one dimension both
        put(1, b, p // 2 + 1, 1, 6, -np.inf)
        put(1, b, p - 1, 1, 7, np.inf)
        put(1, b, p - 7, 1, 7, -np.inf)
        put(1, b, p + n // 2, 1, 8, np.inf)         # ... that only the later tokens of a chunk see
        if n > 1:
            put(0, b, p + n - 2, hk - 1, 4, np.nan)  # a key that is no number, behind most of them
    q[:, :group, 3] = -1.5                          # -inf, no weight
    q[::3, :group, 3] = 1.5                         # +inf, no number (of every third token)
    q[-1, hq - 1, 11] = np.inf
    P.upload()
    got, at = run(ctx, P, pos0, n_new, q), 0
    for b, (p, n) in enumerate(zip(pos0, n_new)):
        held = np.arange(p + n)
        want, bound = B.attention_of_infinities(q[at:at + n], P.at(0, b, held), P.at(1, b, held), p, hs**-0.5)
        assert np.isinf(want).any() and np.isfinite(want).any()
        B.check_exactly(got[at:at + n], want, bound, f"sequence {b}")
        at += n


@pytest.mark.parametrize("dtype", [F16, F32])
def test_rows_without_a_finite_score(ctx, backend, dtype):
    """Nothing but -inf: 0 / 0, as the formula has it.  The first position alone, a token and the beginning of a chunk; and its next ones, which have finite scores too."""
    hq, hk, hs, pos0, n_new = 4, 2, 128, [0, 0], [1, 140]
    P = Pages(backend, hq, hk, hs, 16, n_new, dtype, seed=3)
    q = P.rng.standard_normal((141, hq, hs)).astype(np.float32)
    for b in range(2):
        row = P.at(0, b, [0])
        row[0, :, 3] = np.inf
        P.put(0, b, [0], row)
    q[:, :, 3] = -1.0
    P.upload()
    got, at = run(ctx, P, pos0, n_new, q), 0
    for b, n in enumerate(n_new):
        held = np.arange(n)
        want, bound = B.attention_of_infinities(q[at:at + n], P.at(0, b, held), P.at(1, b, held), 0, hs**-0.5)
        assert np.isnan(want[0]).all() and np.isfinite(want[1:]).all()
        B.check_exactly(got[at:at + n], want, bound, f"sequence {b}")
        at += n
