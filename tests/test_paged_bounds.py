"""That the bounds of paged_bounds.py let through what f32 arithmetic and the kernels' operands leave, and nothing coarser."""
import numpy as np
import pytest

import paged_bounds as B

SHAPES = [(515, 1, 128), (0, 64, 128), (300, 17, 64), (3000, 1, 128), (190, 33, 128), (100, 9, 48), (7000, 2, 128)]


def inputs(pos0, n, hs, f16, seed=1, hq=4, hk=2):
    rng = np.random.default_rng(seed)
    q = (rng.standard_normal((n, hq, hs)) * 2).astype(np.float32)
    k, v = (rng.standard_normal((pos0 + n, hk, hs)).astype(np.float16 if f16 else np.float32) for _ in range(2))
    return q, k, v


def cut(x, bits):
    """x cut to `bits` significant bits, as tf32's 11 of a low part are."""
    m, e = np.frexp(np.asarray(x, np.float64))
    return np.ldexp(np.trunc(np.ldexp(m, bits)), e - bits)


def tf32(x):
    m, e = np.frexp(np.asarray(x, np.float64))
    return np.ldexp(np.rint(np.ldexp(m, 11)), e - 11)


def emulate(q, k, v, pos0, scale, queries, keys, weights, values, low=True):
    """The formula in 64 bits with operands carried by the functions given; (high, low) pairs lose low x low."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    n, hq, hs = q.shape
    group, out = hq // k.shape[1], np.empty(q.shape)

    def product(a, b):  # (high, low) each
        return a[0] @ b[0] + (a[0] @ b[1] + a[1] @ b[0] if low else 0)

    for t in range(n):
        for h in range(hq):
            kk, vv = k[:pos0 + t + 1, h // group], v[:pos0 + t + 1, h // group]
            s = product(keys(kk), queries((q[t, h] * np.float32(scale)).astype(np.float32).astype(np.float64)))
            w = np.exp(s - s.max())
            out[t, h] = product(weights(w), values(vv)) / w.sum()
    return out


half = lambda x: (np.asarray(x, np.float16).astype(np.float64), np.zeros_like(x))  # noqa: E731
halves = lambda x: (half(x)[0], half(x - half(x)[0])[0])  # noqa: E731
whole = lambda x: (x, np.zeros_like(x))  # noqa: E731
pair = lambda x: (tf32(x), cut(x - tf32(x), 11))  # noqa: E731
high = lambda x: (tf32(x), np.zeros_like(x))  # noqa: E731


@pytest.mark.parametrize("shape", SHAPES)
def test_the_kernels_operands_are_within(shape):
    pos0, n, hs = shape
    for f16 in (True, False):
        q, k, v = inputs(pos0, n, hs, f16)
        want, bound = B.attention(q, k, v, pos0, hs**-0.5, f16)
        form = (halves, whole, halves, whole) if f16 else (pair,) * 4
        got = emulate(q, k, v, pos0, hs**-0.5, *form)
        assert not B.far_rows(got, want, bound).any()
        # ... and so is f32 arithmetic
        e = np.einsum("thd,lhd->thl", q, np.repeat(k.astype(np.float32), 2, 1)) * np.float32(hs**-0.5)
        seen = np.arange(pos0 + n)[None, :] <= pos0 + np.arange(n)[:, None]
        e = np.where(seen[:, None], e, -np.inf).astype(np.float32)
        e = np.exp(e - e.max(-1, keepdims=True))
        got = np.einsum("thl,lhd->thd", e, np.repeat(v.astype(np.float32), 2, 1)) / e.sum(-1, keepdims=True)
        assert not B.far_rows(got, want, bound).any()


@pytest.mark.parametrize("shape", SHAPES)
def test_what_is_coarser_is_found(shape):
    """A low-order product that is lost or read from the wrong place."""
    pos0, n, hs = shape

    def found(f16, *form, **kw):
        q, k, v = inputs(pos0, n, hs, f16)
        want, bound = B.attention(q, k, v, pos0, hs**-0.5, f16)
        far = B.far_rows(emulate(q, k, v, pos0, hs**-0.5, *form, **kw), want, bound)
        return far.mean() > 0.5

    assert found(True, half, whole, halves, whole)     # queries of 11 bits
    assert found(True, halves, whole, half, whole)     # weights of 11 bits
    for lost in range(4):
        assert found(False, *(high if i == lost else pair for i in range(4)))
    assert found(False, pair, pair, pair, pair, low=False)


def test_infinities():
    """-inf scores have no weight, +inf and NaN scores none that is a number, infinite values reach their dimension alone; what is not so is found."""
    q, k, v = inputs(40, 3, 16, False, seed=4)
    k[10, 0, 3], k[11, 1, 2], v[12, 0, 5], v[13, 1, 6], v[14, 1, 6], v[41, 0, 7] = np.inf, np.nan, np.inf, np.inf, -np.inf, -np.inf
    q[:, 0, 3], q[:, 1, 3] = -2, 2
    want, bound = B.attention_of_infinities(q, k, v, 40, 0.25)
    assert np.isnan(want[:, 1]).all() and np.isnan(want[:, 2:]).all()
    assert (want[:, 0, 5] == np.inf).all() and np.isfinite(want[0, 0, 7]) and (want[1:, 0, 7] == -np.inf).all()
    rest = [d for d in range(16) if d not in (5, 7)]
    keep = np.delete(np.arange(43), 10)
    assert np.isfinite(want[:, 0, rest]).all()
    e = np.exp(np.asarray(k, np.float64)[keep, 0] @ q[2, 0] * 0.25)
    assert np.allclose(want[2, 0, rest], (e @ np.asarray(v, np.float64)[keep, 0] / e.sum())[rest], rtol=1e-12)
    B.check_exactly(want, want, bound)
    for at, x in (((0, 0, 0), 12345.0), ((0, 0, 5), 0.0), ((0, 0, 5), -np.inf), ((0, 0, 4), np.inf), ((0, 1, 4), 1.0), ((0, 0, 4), np.nan), ((2, 0, 4), want[2, 0, 4] + 1e-3)):
        wrong = want.copy()
        wrong[at] = x
        with pytest.raises(AssertionError):
            B.check_exactly(wrong, want, bound)
