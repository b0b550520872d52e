"""The paged operators' Python side (slai_b200/ops.py) with a library that only notes what it is asked: no GPU."""
import numpy as np
import pytest

from slai_b200 import _lib
from slai_b200._lib import KV_F16, SlaiError
from slai_b200.ops import Backend, GpuVector, LlmContext, PagedKv, PagedLayer, QkNormRope, RecordedPass


class Library:
    """Answers 0 to every call and keeps (name, arguments)."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            if name == "slai_paged_create":
                args[2]._obj.value = 1000 + len(self.calls)
            return 0
        return call

    def named(self, name):
        return [args for n, args in self.calls if n == name]


class NoGpu(Backend):
    def __init__(self):
        self.lib, self.h, self.device, self.at = Library(), 1, 0, 4096

    def malloc(self, nbytes):
        self.at += nbytes + 256
        return self.at

    def close(self):
        pass


@pytest.fixture
def be():
    return NoGpu()


def test_a_handle_that_is_dropped_while_a_pass_is_recorded_is_destroyed_behind_it(be):
    with RecordedPass(be):
        kv = PagedKv(be, 4, 2, 64, 16, 10)
        h = kv.h.value
        del kv
        assert not be.lib.named("slai_paged_destroy")  # (it would end the recording)
    assert [a[0].value for a in be.lib.named("slai_paged_destroy")] == [h]
    names = [n for n, _ in be.lib.calls]
    assert names.index("slai_pass_end") < names.index("slai_paged_destroy")
    kv = PagedKv(be, 4, 2, 64, 16, 10)
    h = kv.h.value
    del kv
    assert [a[0].value for a in be.lib.named("slai_paged_destroy")][1:] == [h]


def refused(code, word, f, *args, **kw):
    with pytest.raises(SlaiError, match=word) as e:
        f(*args, **kw)
    assert e.value.code == code


def cache(be, hq=4, hk=2, hs=64, page=16, n_pages=10, dtype=KV_F16, **kw):
    """A handle and a layer of the right size."""
    pages = [GpuVector(be, n_pages * hk * page * hs, np.float16 if dtype == KV_F16 else np.float32) for _ in range(2)]
    return PagedKv(be, hq, hk, hs, page, n_pages, dtype, **kw), PagedLayer(*pages, hk * page * hs, page * hs, hs)


def test_a_handle_is_used_in_its_own_context(be):
    """Its calls run on its context's stream, which another context's buffers are not ordered with."""
    other = NoGpu()
    kv, layer = cache(other)
    kv.step([3], [1], np.zeros((1, 1), np.int32))
    x = [GpuVector(be, 4 * 64) for _ in range(5)]
    refused(_lib.ERR_INVALID_ARG, "another context", LlmContext(be).paged_attention, kv, layer, x[0], x[1])
    refused(_lib.ERR_INVALID_ARG, "another context", LlmContext(be).paged_append, kv, layer, QkNormRope(64, 4, 2), *x[:4])
    for b in (be, other):
        assert not b.lib.named("slai_paged_attention") and not b.lib.named("slai_paged_append")
    ctx = LlmContext(other)
    ctx.paged_attention(kv, layer, x[0], x[1])
    ctx.paged_append(kv, layer, QkNormRope(64, 4, 2), *x[:4])
    assert len(other.lib.named("slai_paged_attention")) == len(other.lib.named("slai_paged_append")) == 1


@pytest.mark.parametrize("wrong", [np.float16, np.uint8, np.float64, np.int32])
def test_rows_of_another_type_are_refused(be, wrong):
    """Enough elements, but not of four bytes: the kernels would read and write behind them.  (Those of four or more bytes would be read as what they are not.)"""
    ctx, S = LlmContext(be), _lib.ERR_SHAPE
    kv, layer = cache(be)
    kv.step([3, 2], [1, 1], np.array([[0], [1]], np.int32))
    f = lambda heads: GpuVector(be, 2 * heads * 64)  # noqa: E731
    bad = lambda heads: GpuVector(be, 2 * heads * 64, wrong)  # noqa: E731
    how, pos = QkNormRope(64, 4, 2), GpuVector(be, 2, np.int32)
    for i in range(4):
        x = [f(4), f(2), f(4), f(2)]
        x[i] = bad(4 if i % 2 == 0 else 2)
        refused(S, "rows are floats, not " + np.dtype(wrong).name, ctx.qk_norm_rope, how, pos, *x)
        x = [f(4), f(2), f(2), f(4)]
        x[i] = bad(4 if i in (0, 3) else 2)
        refused(S, "rows are floats, not " + np.dtype(wrong).name, ctx.paged_append, kv, layer, how, *x)
    refused(S, "rows are floats", ctx.paged_attention, kv, layer, bad(4), f(4))
    refused(S, "rows are floats", ctx.paged_attention, kv, layer, f(4), bad(4).view(0, 512))
    refused(S, "norm weights", QkNormRope, 64, 4, 2, q_norm=GpuVector(be, 64, wrong))
    if np.dtype(wrong).itemsize != 4:
        refused(S, "positions are int32", ctx.qk_norm_rope, how, GpuVector(be, 2, wrong), f(4), f(2), f(4), f(2))
    assert not [n for n, _ in be.lib.calls if n in ("slai_qk_norm_rope", "slai_paged_append", "slai_paged_attention")]


def test_rows_of_a_type_of_ones_own(be):
    """Anything with a device pointer and a length; where it names its elements' type, that is f32 in any of its spellings."""
    class Mine:
        def __init__(self, n, **kw):
            self.ptr, self.n = 4096, n
            self.__dict__.update(kw)

        def __len__(self):
            return self.n

    ctx = LlmContext(be)
    kv, layer = cache(be)
    kv.step([3], [1], np.zeros((1, 1), np.int32))
    for kw in ({}, dict(dtype=np.float32), dict(dtype="float32"), dict(dtype=np.dtype("<f4"))):
        ctx.paged_attention(kv, layer, Mine(256, **kw), Mine(256, **kw))
        ctx.qk_norm_rope(QkNormRope(64, 4, 2), Mine(1), Mine(256, **kw), Mine(128, **kw), Mine(256, **kw), Mine(128, **kw))
    assert len(be.lib.named("slai_paged_attention")) == len(be.lib.named("slai_qk_norm_rope")) == 4


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("wrong", [1 << 31, (1 << 32) + 1, -(1 << 31) - 1, 1 << 64, 1.5, float("nan"), float("inf"), None, "a"])
def test_lengths_and_tables_that_are_no_int32_numbers(be, which, wrong):
    """... are refused, not cut to 32 bits: 2^32 + 1 would name page 1."""
    kv, _ = cache(be)
    args = [[3, 2], [1, 1], [[0], [1]]]
    for t in (np.int64, np.int32, np.uint16, np.float64):
        kv.step(*(np.array(a, t) for a in args))
    kv.step(*args)
    kv.step([], [], np.zeros((0, 3)))  # nobody takes part
    kv.step(np.array([1]), np.array([1]), np.zeros((1, 0), np.int64))  # (the library refuses a table that is too narrow)
    done = len(be.lib.named("slai_paged_step"))
    assert done == 7 and be.lib.named("slai_paged_step")[0][1] == 2
    if which == 2:
        args[2][1][0] = wrong
    else:
        args[which][1] = wrong
    refused(_lib.ERR_SHAPE, "int32", kv.step, *args)
    assert len(be.lib.named("slai_paged_step")) == done and kv.rows == 1
    if isinstance(wrong, int) and wrong < 1 << 62:
        args[which] = np.array(args[which], np.int64)
        refused(_lib.ERR_SHAPE, "int32", kv.step, *args)


@pytest.mark.parametrize("n_pages, max_seqs, want", [(100, 8, 800), (1, 1, 1), (1 << 16, 64, 1 << 20), (1 << 21, 4, 1 << 21), (0, 8, 0), (-3, 8, -3), (1 << 28, 1 << 20, 1 << 28)])
def test_tables_have_room_for_pages_that_sequences_share(be, n_pages, max_seqs, want):
    """(What is no number of pages goes on to the library, which refuses it.)"""
    PagedKv(be, 4, 2, 64, 1, n_pages, max_seqs=max_seqs)
    assert be.lib.named("slai_paged_create")[-1][1]._obj.max_table == want
    PagedKv(be, 4, 2, 64, 1, n_pages, max_seqs=max_seqs, max_table=7)
    assert be.lib.named("slai_paged_create")[-1][1]._obj.max_table == 7
