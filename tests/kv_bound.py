"""Attention over the 8-bit KV cache in 64 bits, with a bound for each output of
its own: what f32 sums of fp16 weights may be off by, relative to the row's own
weights and values, and not to the largest value of the cache."""
import numpy as np

from tests import kv_model


def steps(model):
    """[kh][length]: the scale each key's values of V are multiples of; a block of zeros
    has that of fp16's least value. The tail's units of 32 tokens take 2^e, their largest
    magnitude within 64..128 of it, or 2^-30."""
    least = 2.0 ** -24 / kv_model.TOP[model.fmt]
    parts = [np.repeat(np.where(np.any(codes, axis=(1, 2)), scales, least)[:, None], model.B, 1)
             for codes, scales in model.blocks]
    tail = np.abs(model.tail.astype(np.float64))
    for u in range(0, tail.shape[1], 32):
        top = tail[:, u:u + 32].max(axis=(1, 2))
        e = np.where(top > 0, np.exp2(np.floor(np.log2(np.where(top > 0, top, 1.0))) - 6), 2.0 ** -30)
        parts.append(np.repeat(e[:, None], tail[:, u:u + 32].shape[1], 1))
    return np.concatenate(parts, axis=1)[:, :model.length]


def attention(q, k, v, step, scale, position, causal, f16):
    """softmax(scale q k) v in float64 and how far each output may be off. q
    [qh][rows][d] fp16, k and v [kh][keys][d] f32, finite; step: steps().

    With W a row's weights (sum 1), out = sum W v:
    - a score in powers of 2 is off by (d + 5) 2^-24 of the sum A of its products'
      magnitudes (d additions; scale, block scale, V's exponent, the reference and the
      multiply-add round once each), and by 2^-15 where the multiply-add's result is
      below 2^8, beyond which a weight is 0. ln 2 of it is the weight's relative
      error; exp2, the logarithm of a scale's fraction and its reciprocal: 2^-21;
    - a weight goes into the products rounded to fp16, by 2^-11 of itself, or as two
      of them, 2^-22; the sum of the weights takes it as it is;
    - both sums add a number a key: 2^-24 each, of the sum of magnitudes;
    - what goes into the products is a weight times its V scale, in units that keep
      the row's largest above 2^9 (f32 output: 2^5); below 2^-14 it is off by up to
      2^-25 instead;
    - the output: 2^-11 of itself, or 2^-22 for the quotient. Products of two of
      these: 1 % of it all."""
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    qh, rows, d = q.shape
    kh, keys, _ = k.shape
    out, most = np.empty(q.shape), np.empty(q.shape)
    seen = np.arange(keys)[None, :] <= (position + np.arange(rows))[:, None] if causal else np.ones((rows, keys), bool)
    to_bits = scale * np.log2(np.e)
    for h in range(qh):
        g = h // (qh // kh)
        s = np.where(seen, q[h] @ k[g].T * scale, -np.inf)
        w = np.exp(s - s.max(axis=1, keepdims=True))
        w /= w.sum(axis=1, keepdims=True)
        size = np.where(seen, np.abs(q[h]) @ np.abs(k[g]).T, 0.0).max(axis=1) * to_bits
        out[h] = w @ v[g]
        size_v = w @ np.abs(v[g])
        weight = (np.log(2.0) * ((d + 5) * 2.0 ** -24 * size + 2.0 ** -15) + 2.0 ** -21)[:, None]
        n = seen.sum(axis=1)[:, None] * 2.0 ** -24
        counts = np.abs(v[g]) / step[g][:, None]
        most[h] = (2 * weight + (2.0 ** -11 if f16 else 2.0 ** -22) + 2 * n) * size_v
        most[h] += 2.0 ** (-34 if f16 else -30) * (w * step[g]).max(axis=1, keepdims=True) * (seen @ counts)
        most[h] += (2.0 ** -11 if f16 else 2.0 ** -22) * np.abs(out[h])
    return out, 1.01 * most + (2.0 ** -25 if f16 else 2.0 ** -149)


def wave(q, k, v, step, scale, f16, unit=32, plant=None):
    """The arithmetic that the bound counts, on one row over all keys, a unit at a
    time: weights times V's scale in fp16 units of a reference that follows the
    largest, f32 sums. plant: a mistake to find. "units": fp16 output's largest is at
    1 first, not at 2^9; "sum": the same, and the sum is that of the rounded weights;
    "zeros": a block of zeros takes part in the reference with scale 1; "drop": one
    unit is left out; "offset": codes plus 128 are multiplied, and 128 times the sum of
    the weights taken off at the end."""
    f32 = np.float32
    s = (k.astype(np.float64) @ q.astype(np.float64)) * scale * np.log2(np.e)
    shift, lazy = (0.0 if plant in ("units", "sum") else 9.0, 6.0) if f16 else (6.0, 8.0)
    m, den, num, taken = -1e30, 0.0, np.zeros(k.shape[1]), 0.0
    for i, u in enumerate(range(0, len(s), unit)):
        if plant == "drop" and i == 1:
            continue
        vs = 1.0 if plant == "zeros" and not v[u:u + unit].any() else float(step[u])
        top = s[u:u + unit].max() + np.log2(vs)
        if top > m + lazy + shift:
            new = np.ceil(top) - shift
            alpha = np.exp2(max(m - new, -2000.0))
            num, den, taken, m = num * alpha, den * alpha, taken * alpha, new
        p = np.exp2(s[u:u + unit] + np.log2(vs) - m).astype(f32)
        high = p.astype(np.float16)
        used = high.astype(np.float64) if f16 else high + (p - high.astype(f32)).astype(np.float16).astype(np.float64)
        den += float((used if plant == "sum" else p.astype(np.float64)).sum()) / vs
        codes = v[u:u + unit].astype(np.float64) / vs
        if plant == "offset":
            num, taken = (num + used @ (codes + 128.0)).astype(f32).astype(np.float64), taken + used.sum()
        else:
            num += used @ codes
    return (num - 128.0 * taken) / den
