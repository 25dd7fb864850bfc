"""The paged KV cache and its attention as include/rk_npu_attention_paged.h defines
them, in 64 bits, and how far the kernels may be off."""
import numpy as np


def frequencies(rotary, theta):
    return np.array([theta ** (-2.0 * j / rotary) for j in range(rotary // 2)])


def rotate(x, positions, freq, interleaved):
    """x [heads][rows][d], rotated by the rows' positions, in 64 bits."""
    y = np.array(x, np.float64)
    n = len(freq)
    for j in range(n):
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + n)
        angle = np.asarray(positions, np.float64) * freq[j]
        c, s = np.cos(angle), np.sin(angle)
        u, v = y[..., a].copy(), y[..., b].copy()
        y[..., a], y[..., b] = u * c - v * s, v * c + u * s
    return y


def rotate_bound(x, y, half):
    """|kernel - y| at most, for rows x rotated to y. Of f32 values: the turn, held
    in f32 after 64-bit reduction, is off by 2^-26 turns, 2 pi 2^-26 < 2^-23 in the
    angle; sine and cosine by 2 units in the last place, 2^-23 of 1; two products and
    a sum by 3 half units. With m the larger of |x| of the pair, which is at most
    the row's largest magnitude: 2 m (2^-23 + 2^-23 + 3 2^-24) < 2^-20 m. Then fp16's
    rounding, half a unit (2^-11 of the value, 2^-25 where it is subnormal)."""
    m = np.abs(np.asarray(x, np.float64)).max(axis=-1, keepdims=True)
    e = 2.0 ** -20 * m
    return e + (np.maximum(2.0 ** -11 * (np.abs(y) + e), 2.0 ** -25) if half else 0.0)


def attention(q, k, v, scale, first, causal):
    """q [qh][rows][d], row i at token first + i; k, v [kh][tokens][d] -> [qh][rows][d], 64 bits."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    qh, rows, d = q.shape
    kh, tokens, _ = k.shape
    out = np.zeros((qh, rows, d))
    for h in range(qh):
        for r in range(rows):
            n = min(tokens, max(0, first + r + 1)) if causal else tokens
            if n == 0:
                continue
            with np.errstate(invalid="ignore", over="ignore"):
                s = scale * (k[h // (qh // kh), :n] @ q[h, r])
                p = np.exp(s - s.max())
                out[h, r] = (p / p.sum()) @ v[h // (qh // kh), :n]
    return out


def attention_bound(q, k, scale, half_out, one_weight, tokens):
    """The kernels' largest distance from `attention`, relative to the largest |v|.
    Scores: d products of fp16, exact in f32, added in f32 in any order: off by at
    most d 2^-24 of the sum of the magnitudes, which Cauchy bounds by |q| |k|; the
    product with scale log2(e) (itself rounded) and its difference from the maximum
    round 3 times: with S = scale |q| |k| max, a score is off by (d + 3) 2^-24 S 1.4427
    binary powers and a weight by that times ln 2 = (d + 3) 2^-24 S, plus exp2's 2
    units, 2^-22. Weights as two fp16 are off by 2^-22 (one: 2^-11), their sum and the
    products' sums by one f32 rounding a step, at most tokens / 32 + 16 steps in a row
    of 32-key matrix steps and joins (2^-24 each; a matrix step's own 32 products round
    within 2^-22). All of it counts twice: in the weights' products and in their
    sum. Below 2^-14 fp16 has steps of 2^-24, half of which is lost of each token's
    weight, where the row's largest weight is above 2^5: 2^-30 of it. fp16 output: half a
    unit, 2^-11."""
    q, k = np.asarray(q, np.float64), np.asarray(k, np.float64)
    s = scale * np.sqrt((q ** 2).sum(-1).max() * (k ** 2).sum(-1).max())
    d = q.shape[-1]
    weight = (d + 3) * 2.0 ** -24 * s + 2.0 ** -22 + (2.0 ** -11 if one_weight else 2.0 ** -22)
    sums = (tokens / 32 + 16) * 2.0 ** -24 + 2.0 ** -22 + tokens * 2.0 ** -30
    return 2.0 * (weight + sums) + (2.0 ** -11 if half_out else 0.0)
