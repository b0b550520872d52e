"""Ways in which a program may use the paged operators beside one call after the other."""
import gc

import numpy as np
import pytest

import paged_reference as R
from slai_b200 import _lib
from slai_b200._lib import KV_F16, KV_F32, SlaiError
from slai_b200.ops import Backend, LlmContext, PagedKv, PagedLayer, QkNormRope
from test_gpu_paged import Pages, attend, check, refused

pytestmark = pytest.mark.gpu
F16, F32 = KV_F16, KV_F32


@pytest.mark.parametrize("dtype", [F16, F32])
def test_a_recorded_pass_outlives_its_handle(ctx, backend, dtype):
    """Its replays go on with the last step, whoever has asked for memory since; the handle's memory goes with the pass."""
    hq, hk, hs, most = 16, 8, 128, 150
    P = Pages(backend, hq, hk, hs, 16, [1500, 700, 300], dtype, max_tokens=most, seed=31)
    how = QkNormRope(hs, hq, hk, 1)
    x = [P.rng.standard_normal(most * h * hs).astype(np.float32) for h in (hq, hk, hk)]
    q, k, v = (backend.vector(a) for a in x)
    qo, out = backend.zeros(q.n), backend.zeros(q.n)
    P.kv.step([1499, 600, 299], [1, 100, 1], P.tables)
    calls = lambda: (ctx.paged_append(P.kv, P.layer, how, q, k, v, qo), ctx.paged_attention(P.kv, P.layer, qo, out))  # noqa: E731
    calls()
    with backend.record() as rec:
        calls()
    rec.launch()
    want = out.to_numpy()
    assert np.abs(want[:102 * hq * hs]).min() > 0

    def free_bytes():
        backend.synchronize()
        return backend.mem_info()[0]

    before = free_bytes()
    P.kv = None
    gc.collect()
    junk = [backend.vector(np.full(1 << 18, -1, np.int32), np.int32) for _ in range(64)]  # would lie where the plan and the partial results were
    backend.write_buffer(out.ptr, np.full(out.n, 4.5, np.float32))
    rec.launch(3)
    got = out.to_numpy()
    assert np.array_equal(got[:102 * hq * hs], want[:102 * hq * hs]) and (got[102 * hq * hs:] == 4.5).all()
    for j in junk:
        assert (j.to_numpy() == -1).all()
    del junk, j
    assert free_bytes() <= before
    rec.close()
    assert free_bytes() > before


def test_a_handle_is_not_destroyed_while_a_pass_is_recorded(ctx, backend):
    P = Pages(backend, 4, 2, 64, 16, [40, 20], F16)
    P.kv.step([39, 19], [1, 1], P.tables)
    q, out = backend.zeros(60 * 4 * 64), backend.zeros(60 * 4 * 64)
    ctx.paged_attention(P.kv, P.layer, q, out)
    with backend.record() as rec:
        ctx.paged_attention(P.kv, P.layer, q, out)
        refused(_lib.ERR_INVALID_ARG, "recorded", lambda: backend.check(backend.lib.slai_paged_destroy(P.kv.h)))
    rec.launch(2)
    backend.synchronize()
    rec.close()
    attend(ctx, P, [39, 19], [1, 1])


def test_a_shared_prefix_longer_than_the_pages_there_are(ctx, backend):
    """Eight sequences that share 12 pages of 28 use 112 table entries; a handle of the default size takes them."""
    hq, hk, hs, page, seqs = 8, 2, 128, 16, 8
    P = Pages(backend, hq, hk, hs, page, [14 * page - 3] * seqs, F16, seed=35)
    P.tables[:, :12], P.tables[:, 12:] = np.arange(12)[::-1], 12 + np.arange(2 * seqs).reshape(seqs, 2)
    P.kv = PagedKv(backend, hq, hk, hs, page, 28, F16, max_seqs=seqs, max_tokens=64)
    attend(ctx, P, [13 * page + 5] * seqs, [8] * seqs)


def test_results_that_share_floats_with_what_is_still_read(ctx, backend):
    """In place with the same leading dimension; refused otherwise, however the rows come to overlap."""
    I, hq, hk, hs, T = _lib.ERR_INVALID_ARG, 4, 2, 64, 20
    ld = (hq + 2 * hk) * hs
    rng = np.random.default_rng(36)
    x = rng.standard_normal((T + 4, ld)).astype(np.float32)
    pos = backend.vector(np.arange(T), np.int32)
    buf, apart = backend.vector(x), [backend.zeros(T * hq * hs) for _ in range(2)]
    part = lambda at, n: buf.view(at, (T - 1) * ld + n * hs)  # noqa: E731
    q, k, v = part(0, hq), part(hq * hs, hk), part((hq + hk) * hs, hk)
    how = lambda **kw: QkNormRope(hs, hq, hk, 1, q_ld=ld, k_ld=ld, v_ld=ld, **kw)  # noqa: E731
    whole = buf.view(0, buf.n)
    refused(I, "q_out .* shares floats with q ", ctx.qk_norm_rope, how(k_out_ld=ld), pos, q, k, whole, k)             # in place, but packed
    refused(I, "k_out .* shares floats with k ", ctx.qk_norm_rope, how(q_out_ld=ld), pos, q, k, q, buf.view(hq * hs, buf.n - hq * hs))
    refused(I, "q_out .* shares floats with k ", ctx.qk_norm_rope, how(q_out_ld=ld), pos, q, k, part(hq * hs, hq), apart[1])
    refused(I, "q_out .* shares floats with k_out", ctx.qk_norm_rope, how(), pos, q, k, apart[0], apart[0])
    refused(I, "k_out .* shares floats with q ", ctx.qk_norm_rope, how(k_out_ld=ld), pos, q, k, apart[0], part(hs, hk))
    refused(I, "q_out .* shares floats with q ", ctx.qk_norm_rope, how(q_out_ld=ld), pos, q, k, part(ld, hq), apart[1])  # a row further on
    P = Pages(backend, hq, hk, hs, 16, [T], F32, max_tokens=T)
    P.kv.step([0], [T], P.tables)
    refused(I, "q_out .* shares floats with q ", ctx.paged_append, P.kv, P.layer, how(), q, k, v, whole)
    refused(I, "q_out .* shares floats with k ", ctx.paged_append, P.kv, P.layer, how(q_out_ld=ld), q, k, v, part(hq * hs, hq))
    refused(I, "q_out .* shares floats with v", ctx.paged_append, P.kv, P.layer, QkNormRope(hs, hq, hk, 1, v_ld=ld, q_out_ld=ld), apart[0], apart[1], v, part((hq + hk - 1) * hs, hq))
    refused(I, "out .* shares floats with q", ctx.paged_attention, P.kv, P.layer, q, part(hs, hq), 0.0, ld, ld)
    refused(I, "out .* shares floats with q", ctx.paged_attention, P.kv, P.layer, q, part(ld, hq), 0.0, ld, ld)
    refused(I, "out .* shares floats with q", ctx.paged_attention, P.kv, P.layer, q, buf.view(hs, buf.n - hs), 0.0, ld, 0)
    assert np.array_equal(buf.to_numpy().reshape(x.shape), x)
    # what shares nothing is taken: results between the queries' rows
    P.host[0][:], P.host[1][:] = rng.standard_normal(P.host[0].size), rng.standard_normal(P.host[0].size)
    P.upload()
    ctx.paged_attention(P.kv, P.layer, q, part(hq * hs, hq), 0.0, ld, ld)
    got = buf.to_numpy().reshape(x.shape)
    want, bound = R.attention(x[:T, :hq * hs].reshape(T, hq, hs), P.at(0, 0, np.arange(T)), P.at(1, 0, np.arange(T)), 0, hs**-0.5)
    check(got[:T, hq * hs:].reshape(T, hq, hs), want, bound)
    assert np.array_equal(got[:, :hq * hs], x[:, :hq * hs]) and np.array_equal(got[T:], x[T:])
    # one token's row has no next: in place and packed are the same
    one = backend.vector(x[0])
    at = lambda h, n: one.view(h * hs, n * hs)  # noqa: E731
    ctx.qk_norm_rope(how(), backend.vector([5], np.int32), at(0, hq), at(hq, hk), at(0, hq), at(hq, hk))
    want, bound = R.norm_rope(x[:1, :(hq + hk) * hs].reshape(1, hq + hk, hs), None, 0, 1, 10000.0, [5])
    check(one.to_numpy()[:(hq + hk) * hs].reshape(want.shape), want, bound)


def test_an_append_through_strides_that_overlap(ctx, backend):
    P = Pages(backend, 4, 2, 64, 16, [40, 20], F16)
    P.kv.step([39, 19], [1, 1], P.tables)
    x = [backend.zeros(2 * 4 * 64) for _ in range(4)]
    large = [backend.zeros(4 * P.dev[0].n, np.float16) for _ in range(2)]  # (room for whatever the strides reach)
    for strides in ((64, 64, 64), (2 * 16 * 64, 16 * 64, 16 * 64), (16 * 64, 16 * 64, 64), (2 * 16 * 64 - 1, 16 * 64, 64)):
        refused(_lib.ERR_SHAPE, "lie on one another", ctx.paged_append, P.kv, PagedLayer(*large, *strides), QkNormRope(64, 4, 2), *x)
    ctx.paged_append(P.kv, P.layer, QkNormRope(64, 4, 2), *x)
    before = [h.copy() for h in P.host]
    P.download()
    for w in range(2):
        assert not P.at(w, 0, [39]).any() and not P.at(w, 1, [19]).any()
        P.put(w, 0, [39], before[w][P._index(0, [39])])
        P.put(w, 1, [19], before[w][P._index(1, [19])])
        assert np.array_equal(P.host[w], before[w])


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hs, page, pos0, n_new", [(128, 16, [7000], [300]), (128, 20, [300, 0], [100, 200]), (64, 64, [2000, 5], [150, 1])])
def test_chunks_with_the_shortest_wait_limit(dtype, hs, page, pos0, n_new):
    """16 rounds are enough for the waits inside a chunk's kernel (the prompt's products need more); one that took longer would be reported at the next synchronisation, once,
    and go on until what it waits for is there.  Either way the bits are the same."""
    be = Backend(0)
    ctx = LlmContext(be)
    P = Pages(be, 16, 4, hs, page, [p + n for p, n in zip(pos0, n_new)], dtype, seed=41)
    q = be.vector(P.rng.standard_normal(sum(n_new) * 16 * hs))
    out = be.zeros(q.n)
    P.kv.step(pos0, n_new, P.tables)

    def call():
        be.write_buffer(out.ptr, np.full(out.n, 4.5, np.float32))
        ctx.paged_attention(P.kv, P.layer, q, out)
        be.synchronize()

    call()
    want = out.to_numpy()
    be.set_wait_limit(16)
    for _ in range(12):
        try:
            call()
        except SlaiError as e:
            assert e.code == _lib.ERR_TIMEOUT and "paged attention" in str(e)
            be.synchronize()  # (reported once)
        assert np.array_equal(out.to_numpy(), want)
    be.set_wait_limit(1 << 20)
    call()
    assert np.array_equal(out.to_numpy(), want)
    del P, q, out
    be.close()
