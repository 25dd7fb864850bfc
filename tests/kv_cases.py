"""Caches on which lost weights, lost keys and too few bits show in the outputs,
for tests/kv_bound.py: lists of (K, V) rows to append, fp16."""
import numpy as np


def _rows(rng, kh, n, d, vx=1.0):
    k = rng.standard_normal((kh, n, d))
    return k.astype(np.float16), (rng.standard_normal((kh, n, d)) * vx).astype(np.float16)


def far_apart(rng, kh, d, power, large_first, units=8, tail=0):
    """Half of the keys with values of 2^(power - 13), half of 2^-13, of equal weight
    on the average. tail: as many rows more, of the half that comes last."""
    sizes = [2.0 ** (power - 13), 2.0 ** -13]
    if not large_first:
        sizes.reverse()
    return [_rows(rng, kh, 32 * units, d, x) for x in sizes] + ([_rows(rng, kh, tail, d, sizes[1])] if tail else [])


def zeros(rng, kh, d, size, zeros_first, units=8, tail=0):
    """Half of the keys with values of `size`, half with none; the tail likewise
    `tail` rows of none."""
    a, b = _rows(rng, kh, 32 * units, d, 0.0), _rows(rng, kh, 32 * units, d, size)
    return ([a, b] if zeros_first else [b, a]) + ([_rows(rng, kh, tail, d, 0.0)] if tail else [])


def strong_key(rng, kh, d, q, scale, gap, keys=2048, block=16.0):
    """One key `gap` above the others' scores for the query q [d], its V zero, in 32
    keys whose other values are `block` times the rest's."""
    k, v = _rows(rng, kh, keys, d)
    k = (0.05 * k).astype(np.float16)
    v[:, :32] *= np.float16(block)
    q = q.astype(np.float64)
    k[:, 5] = (q * (gap / (scale * (q @ q)))).astype(np.float16)
    v[:, 5] = 0
    return [(k, v)]


def marks(rng, kh, d, keys):
    """V names its unit of 32 keys: 1 in dim `unit` % d, 0 elsewhere, so an output is
    the weight of its units."""
    k, v = _rows(rng, kh, keys, d, 0.0)
    at = np.arange(keys)
    v[:, at, at // 32 % d] = 1
    return [(k, v)]
