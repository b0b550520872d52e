"""How near the paged attention has to come to its formula: a bound on a row's whole error that a lost low-order product breaks, and one that stays finite, and exact about
infinities, where some keys or values are infinite.  (paged_reference.attention's bound is each element's worst case: a thousand times what ordinary rows are off by.)"""
import numpy as np


def attention(q, k, v, pos0, scale, f16):
    """q [n][Hq][hs] (tokens at pos0 ..), k, v [L][Hk][hs] as cached -> (result [n][Hq][hs], bound on the length of a row's error [n][Hq]).

    With w the weights, s the scores, o the result; the error of o is the sum of w_t ds_t (v_t - o), of the weights' and values' own roundings, and of the sums'.
    Operands: queries and weights over f16 caches are pairs of halves, each rounded: 2^-22 of the value.  Over f32 caches queries, keys, weights and values are pairs of
      tf32 numbers, the high one rounded (2^-11), the low one cut (2^-10 of that): 2^-21 each, and 2^-22 for the product of low parts that is left out.  The roundings of
      different elements have nothing to do with one another: four times the root of the sum of their squares.
    Sums on the matrix units are cut, not rounded, towards zero: by 2^-23 of what has been summed so far at each of hs / 16 (f32 caches: hs / 8) steps and two more; the low
      parts of tf32 pairs are cut too, 2^-20 of the products.  That makes scores smaller, all by about the same share of their size: the result moves along the sum
      of w_t s_t (v_t - o), and by what differs between positions, which is taken like the roundings.
    The exponential: its argument has two roundings, the function two more: four half steps of the score's size, at least of 1.
    Sums of values: 16 positions a step, at most 128 in a row (8 steps, and two, for each product), cut, by a share of a sum so far, whose size is that of
      the root of the sum of its terms' squares (three times that); these sums then follow one another in f32 (a rounding each, of no fewer than 8 positions)."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    n, hq, hs = q.shape
    group, two = hq // k.shape[1], 2.0
    operand = two**-22 if f16 else 2.5 * two**-21
    carried = two**-22 if f16 else 2 * two**-21
    steps = (hs / (16 if f16 else 8) + 2) * two**-23 + (0 if f16 else two**-20)
    out, bound = np.empty_like(q), np.empty((n, hq))
    for t in range(n):
        L = pos0 + t + 1
        for h in range(hq):
            kk, vv = k[:L, h // group], v[:L, h // group]
            products = kk * q[t, h] * scale
            s = products.sum(1)
            w = np.exp(s - s.max())
            w /= w.sum()
            o = w @ vv
            away = np.sqrt(((vv - o) ** 2).sum(1))
            loose = 4 * operand * np.sqrt((products**2).sum(1))
            size = np.maximum(1, np.abs(s)) * (steps + 4 * two**-24)
            terms = np.sqrt((w**2 * (vv**2).sum(1)).sum())
            bound[t, h] = (np.sqrt(((w * (loose + 4 * size) * away) ** 2).sum()) + steps * np.sqrt((((w * s) @ (vv - o)) ** 2).sum())
                           + terms * (4 * carried + 3 * 10 * two**-23 + 4 * np.sqrt(L / 8) * two**-24))
            out[t, h] = o
    return out, bound


def far_rows(got, want, bound):
    """Rows [n][Hq] whose error is longer than the bound."""
    return ~(np.sqrt(((np.asarray(got, np.float64) - want) ** 2).sum(-1)) <= bound)


def attention_of_infinities(q, k, v, pos0, scale):
    """The formula where keys and values may be infinite or NaN -> (result, bound), each [n][Hq][hs]; the bound (paged_reference.attention's, each dimension for itself and
    of what is finite) is finite wherever the result is."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    n, hq, hs = q.shape
    group, u = hq // k.shape[1], 2.0**-24
    out, bound = np.empty_like(q), np.empty_like(q)
    with np.errstate(invalid="ignore", over="ignore"):
        for t in range(n):
            L = pos0 + t + 1
            for h in range(hq):
                kk, vv = k[:L, h // group], v[:L, h // group]
                s = kk @ q[t, h] * scale
                sizes = np.abs(kk) @ np.abs(q[t, h]) * abs(scale)
                e = np.exp(s - s.max())
                out[t, h] = (e[:, None] * vv).sum(0) / e.sum()
                fine = np.isfinite(s)
                largest = np.where(np.isfinite(vv), np.abs(vv), 0).max(0)
                ds = (2 * (hs + 8) * sizes[fine].max() + 4 * np.abs(s[fine]).max()) * u if fine.any() else 0
                bound[t, h] = (2 * ds + 2 * (L + 16) * u) * largest
    return out, bound


def check_exactly(got, want, bound, what=""):
    """NaN and each infinity just where they belong; all else within a bound that is finite."""
    got, fine = np.asarray(got, np.float64), np.isfinite(want)
    assert got.shape == want.shape and np.isfinite(bound[fine]).all()
    assert (np.isnan(got) == np.isnan(want)).all(), f"{what}: NaN where none belongs, or none where one does"
    inf = np.isinf(want)
    assert (got[inf] == want[inf]).all(), f"{what}: {int((got[inf] != want[inf]).sum())} of {int(inf.sum())} infinities are not there"
    assert np.isfinite(got[fine]).all(), f"{what}: infinities where none belong"
    off = np.abs(got[fine] - want[fine])
    assert (off <= bound[fine]).all(), f"{what}: {int((off > bound[fine]).sum())} of {off.size} off, by up to {off.max()}"
