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
