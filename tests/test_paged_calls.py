"""The paged operators' Python side (slai_b200/ops.py) with a library that only notes what it is asked: no GPU."""
import numpy as np
import pytest

from slai_b200.ops import Backend, GpuVector, PagedKv, RecordedPass


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
