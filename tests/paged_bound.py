"""Attention over the paged KV cache in 64 bits, with a bound for each output of its
own: what f32 sums of fp16 weights may be off by, relative to the row's own weights
and values, and not to the largest query, key and value of the call."""
import numpy as np


def attention(q, k, v, scale, first, causal, f16, one):
    """softmax(scale q k) v in float64 and how far each output may be off. q
    [qh][rows][d] fp16, row i at token first + i; k and v [kh][tokens][d] fp16,
    finite; every row sees a token. f16: the output's type; one: a weight goes into
    the products as one fp16, not two.

    With W a row's weights (sum 1), out = sum W v:
    - a score in powers of 2 is off by (n + 3) 2^-24 of the sum A of its products'
      magnitudes, n of them not 0 (n additions; scale and its product with log2(e)
      round, the score's product with that once), and by 2^-17 where its difference
      from the maximum is rounded, below 2^7, beyond which a weight is 0. ln 2 of it
      is the weight's relative error; exp2: 2^-22;
    - a weight is rounded to fp16, by 2^-11 of itself, or to two of them, 2^-22, and
      2^-24 more where those are scaled and split again; the sum of the weights takes
      f32 ones or the rounded ones;
    - both sums add a number a key: 2^-24 each, of the sum of magnitudes;
    - below 2^-14 a weight is off by up to 2^-25 instead, where the row's largest is
      above 2^5. A move of the maximum scales weights that wait, by 2^-6 at most, and
      rounds them again: what they were off by counts no more. One fp16: above 2^8, the
      scale in two factors, the second below 2^-1, with a rounding each: 1.5 2^-25;
    - the output: 2^-11 of itself, or 2^-22 for the quotient. Products of two of
      these: 3 % of it all."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    qh, rows, d = q.shape
    kh, tokens, _ = k.shape
    out, most = np.empty(q.shape), np.empty(q.shape)
    seen = np.arange(tokens)[None, :] <= (first + np.arange(rows))[:, None] if causal else np.ones((rows, tokens), bool)
    for h in range(qh):
        g = h // (qh // kh)
        s = np.where(seen, q[h] @ k[g].T * scale, -np.inf)
        w = np.exp(s - s.max(axis=1, keepdims=True))
        w /= w.sum(axis=1, keepdims=True)
        size = np.where(seen, np.abs(q[h]) @ np.abs(k[g]).T, 0.0).max(axis=1) * scale * np.log2(np.e)
        n = ((q[h] != 0).astype(float) @ (k[g] != 0).T).max(axis=1)
        out[h] = w @ v[g]
        size_v = w @ np.abs(v[g])
        score = (np.log(2.0) * ((n + 3) * 2.0 ** -24 * size + 2.0 ** -17) + 2.0 ** -22)[:, None]
        weight = 2.0 ** -11 if one else 2.0 ** -22 + 2.0 ** -24
        sums = 2 * seen.sum(axis=1)[:, None] * 2.0 ** -24
        most[h] = (2 * score + (2 if one else 1) * weight + sums) * size_v
        most[h] += (1.5 * 2.0 ** -33 if one else 2.0 ** -30) * w.max(axis=1, keepdims=True) * (seen @ np.abs(v[g]))
        most[h] += (2.0 ** -11 if f16 else 2.0 ** -22) * np.abs(out[h])
    return out, 1.03 * most + (2.0 ** -25 if f16 else 2.0 ** -149)


def jumps(rng, d, units, at, high, jump):
    """q [rows][d] and k, v [tokens][d] of one head, `units` of 32 keys, whose scores are
    products of one dim (exact): near 0, then in unit at - 1 `high` powers of 2, then in
    unit `at` one key at `jump`. Row 0 sees those, the others parts of them. Unit u names
    itself in dim u of V; the dims from 32 on are of every key."""
    q, k = np.zeros((20, d), np.float16), np.zeros((32 * units, d), np.float16)
    q[:, 0] = 1.0 - np.arange(20) / 32.0
    k[:, 0] = -rng.integers(0, 16, 32 * units) / 8.0
    k[:32, 0] = 0.0
    k[32 * (at - 1):32 * at, 0] = high
    k[32 * at + rng.integers(0, 32), 0] = jump
    v = np.zeros((32 * units, d), np.float16)
    v[np.arange(32 * units), np.arange(32 * units) // 32] = 1.0
    v[:, 32:] = rng.standard_normal((32 * units, d - 32))
    return q, k, v


SCALE = float(np.float32(np.log(2.0)))  # (a score of 1 is a power of 2)


def wave(q, k, v, scale, one, plant=None):
    """The arithmetic that the bound counts, on one row over all keys, 32 at a time: a
    unit's weights wait for the next one's step, which may move the maximum, before
    they are multiplied. plant: a mistake to find. "alpha": weights that wait are scaled
    by a factor in fp16; "drop": one unit is left out."""
    f32, f16 = np.float32, np.float16
    s = (k.astype(np.float64) @ q.astype(np.float64)) * scale * np.log2(np.e)
    lazy, shift = (6.0, 9.0) if one else (8.0, 6.0)
    m, den, num = -1e30, f32(0.0), np.zeros(k.shape[1])
    high = low = np.zeros(32, f16)
    before = slice(0, 32)
    for i, u in enumerate(range(0, len(s), 32)):
        if plant == "drop" and i == 1:
            continue
        top = s[u:u + 32].max()
        if top > m + lazy + shift:
            new = np.ceil(top) - shift
            alpha = np.exp2(f32(max(m - new, -2000.0)))
            m, den, num = new, den * alpha, num * float(alpha)
            if plant == "alpha":
                high, low = high * f16(alpha), low * f16(alpha)
            else:
                w = (high.astype(f32) + low.astype(f32)) * alpha
                high = w.astype(f16)
                low = np.zeros_like(high) if one else (w - high.astype(f32)).astype(f16)
        num = num + (high.astype(float) + low.astype(float)) @ v[before].astype(float)
        p = np.exp2(s[u:u + 32] - m).astype(f32)
        high = p.astype(f16)
        low = np.zeros_like(high) if one else (p - high.astype(f32)).astype(f16)
        before = slice(u, u + 32)
        den = den + p.sum(dtype=f32)
    return (num + (high.astype(float) + low.astype(float)) @ v[before].astype(float)) / float(den)
