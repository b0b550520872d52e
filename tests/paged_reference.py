"""The paged operators from their formulas in 64 bits (numpy), and how far f32 arithmetic may be from them."""
import numpy as np

U = 2.0**-24  # half a step of f32, relative


def norm_rope(x, w, eps, variant, base, pos):
    """x [T][H][hs] -> (result, bound).  Bound: the sum of squares has hs roundings, halved by the root; products and the weight 4; an angle is off by
    pi * 2^-24 and its cosine and sine by 2 units in the last place of 1 (16 together, times the pair's size)."""
    x = np.asarray(x, np.float64)
    hs = x.shape[-1]
    y = x
    if w is not None:
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * np.asarray(w, np.float64)
    if variant is None:
        return y, np.abs(y) * (hs / 2 + 8) * U
    ang = np.asarray(pos, np.float64)[:, None, None] * np.float64(np.float32(base)) ** (-2.0 * np.arange(hs // 2) / hs)
    lo, hi = (slice(0, None, 2), slice(1, None, 2)) if variant == 0 else (slice(0, hs // 2), slice(hs // 2, None))
    out, bound = np.empty_like(y), np.empty_like(y)
    a, b = y[..., lo], y[..., hi]
    out[..., lo], out[..., hi] = a * np.cos(ang) - b * np.sin(ang), a * np.sin(ang) + b * np.cos(ang)
    bound[..., lo] = bound[..., hi] = (np.abs(a) + np.abs(b)) * (hs / 2 + 24) * U
    return out, bound


def stored(y, bound, f16):
    """... and what the cache holds of it: half a step of f16 more (2^-11 of the value, 2^-25 where it is subnormal)."""
    return bound + (np.abs(y) + bound) * 2.0**-11 + 2.0**-25 if f16 else bound


def attention(q, k, v, pos0, scale):
    """q [n][Hq][hs] (tokens at pos0 ..), k, v [L][Hk][hs] as cached -> (result, bound), each [n][Hq][hs].

    Bound.  A score is a sum of hs products: each rounded, q perhaps carried as 22 bits, sums truncated rather than rounded: 2 (hs + 8) half steps of the sum
    of the products' sizes, 4 of the score itself for its way through the exponential.  A weight is off by that, relative; the weighted mean of the values by
    twice it (numerator and denominator), plus 2 (L + 16) half steps for the two sums, of the largest value."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    n, hq, hs = q.shape
    group = hq // k.shape[1]
    out, bound = np.empty_like(q), np.empty_like(q)
    for t in range(n):
        L = pos0 + t + 1
        for h in range(hq):
            kk, vv = k[:L, h // group], v[:L, h // group]
            with np.errstate(invalid="ignore", over="ignore"):
                s = kk @ q[t, h] * scale
                sizes = np.abs(kk) @ np.abs(q[t, h]) * abs(scale)
                e = np.exp(s - s.max())
                out[t, h] = (e @ vv) / e.sum()
                ds = (2 * (hs + 8) * sizes.max() + 4 * np.abs(s).max()) * U
                bound[t, h] = (2 * ds + 2 * (L + 16) * U) * np.abs(vv).max()
    return out, bound
