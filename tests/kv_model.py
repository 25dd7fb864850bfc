"""The 8-bit KV cache's contents as include/rk_npu_attention_q8.h defines them,
in numpy: the oracle of its tests. Values are exact: codes are whole numbers or
e4m3 values found in 64 bits, scales and code x scale are single f32
operations."""
import numpy as np

TOP = {"i8": 127.0, "e4m3": 448.0}


def e4m3_round(x):
    """float64 values within +-448 to the nearest e4m3 value, ties to even: 4
    significant bits, steps of 2^-9 below 2^-6."""
    step = np.exp2(np.maximum(np.frexp(x)[1], -5) - 4.0)
    return np.round(x / step) * step


def quantise(rows, fmt):
    """rows [kh][block][d] fp16 -> (codes float64, scales f32 [kh]); a block with
    an infinity or NaN has a NaN scale."""
    x = rows.astype(np.float64)
    top = np.abs(x).max(axis=(1, 2))
    codes = np.zeros_like(x)
    scales = np.ones(len(x), np.float32)
    for g in range(len(x)):
        if not np.isfinite(top[g]):
            scales[g] = np.nan
        elif top[g] > 0:
            q = x[g] * TOP[fmt] / top[g]
            codes[g] = np.round(q) if fmt == "i8" else e4m3_round(q)
            scales[g] = np.float32(top[g]) / np.float32(TOP[fmt])
    return codes, scales


def values(block):
    codes, scales = block
    return codes.astype(np.float32) * scales[:, None, None]


class KvModel:
    """K or V of one cache."""

    def __init__(self, kh, d, fmt, block):
        self.fmt, self.B, self.kh, self.d = fmt, block, kh, d
        self.length, self.blocks = 0, []
        self.tail = np.zeros((kh, 0, d), np.float16)  # (empty while the last block is read as codes)
        self.kept = {}  # token block -> its first fp16 rows

    @property
    def deep(self):
        """Truncated into a block that is read as codes."""
        return len(self.blocks) * self.B > self.length

    def append(self, rows):
        with np.errstate(over="ignore"):
            rows = rows.astype(np.float16)
        B, b0, t = self.B, self.length // self.B, self.length % self.B
        kept = {}
        if self.deep:
            with np.errstate(over="ignore"):
                old = values(self.blocks.pop())[:, :t].astype(np.float16)
        else:
            old = self.tail
            if t:
                kept[b0] = old
        x = np.concatenate([old, rows], axis=1)
        n = x.shape[1]
        for i in range(n // B):
            self.blocks.append(quantise(x[:, i * B:(i + 1) * B], self.fmt))
        if n // B:
            kept[b0 + n // B - 1] = x[:, (n // B - 1) * B:n // B * B]
        self.tail = x[:, n // B * B:]
        if n % B:
            kept[b0 + n // B] = self.tail
        self.kept = kept
        self.length += rows.shape[1]

    def truncate(self, length):
        if length == self.length:
            return
        B, b, t = self.B, length // self.B, length % self.B
        self.kept = {i: x[:, :t] if i == b else x for i, x in self.kept.items() if i <= b}
        exact = t and b in self.kept and self.kept[b].shape[1] == t
        self.tail = self.kept[b] if exact else np.zeros((self.kh, 0, self.d), np.float16)
        self.blocks = self.blocks[:b if exact or not t else b + 1]
        self.length = length

    def values(self):
        """[kh][length][d] f32."""
        parts = [values(x) for x in self.blocks] + [self.tail.astype(np.float32)]
        return np.concatenate(parts, axis=1)[:, :self.length]


def attention(q, k, v, scale, position, causal):
    """softmax(scale q k) v in float64; q [qh][rows][d] fp16, k and v [kh][keys][d].
    A value that is not finite counts where its key is seen: infinite, or NaN,
    whatever the key's weight."""
    q, k, v = q.astype(np.float64), k.astype(np.float64), v.astype(np.float64)
    qh, rows, _ = q.shape
    kh, keys, _ = k.shape
    out = np.empty(q.shape)
    seen = np.arange(keys)[None, :] <= (position + np.arange(rows))[:, None] if causal else np.ones((rows, keys), bool)
    wild = ~np.isfinite(v)
    plain = np.where(wild, 0.0, v)
    with np.errstate(invalid="ignore"):
        for h in range(qh):
            g = h // (qh // kh)
            s = np.where(seen, q[h] @ k[g].T * scale, -np.inf)
            p = np.exp(s - s.max(axis=1, keepdims=True))
            out[h] = (p @ plain[g]) / p.sum(axis=1, keepdims=True)
            for j in np.nonzero(wild[g].any(axis=1))[0]:
                out[h] += np.where(seen[:, j:j + 1] & wild[g, j][None, :], v[g, j][None, :], 0.0)
    return out


def bound(q, k, v, scale, f16, i8=False):
    """How far f32 arithmetic may be from attention(), per element, relative to
    the largest |value|.

    A score in powers of 2 is off by at most (d + 3) 2^-24 of the sum of its
    products' magnitudes (d additions; the products are exact; scale, block scale
    and the multiply-add round once each) and 2^-23 of its distance from the
    maximum, below 2^8 where a weight is not 0; ln 2 of that is the weight's
    relative error, plus 2^-22 for exp2 and 2^-22 for the two fp16 that stand for
    it (fp16 output: 2^-11 for the one). Numerator and denominator each take it
    once, and add `keys` numbers (2^-24 each, at most). An fp16 output rounds by
    2^-11 of itself; an f32 one by the quotient's 2 roundings.

    fp16 output over i8 codes may take the products of u = code + 128 instead and
    128 times the sum of the other operand off them. u ks is below 2.01 of the
    block's largest |k|, so a score's d additions add at most 3.02 of it times the
    sum of |q| (u's and the sum's own); the numerator's of u and of the weights
    come to 3.02 keys in place of 1."""
    d, keys = q.shape[2], k.shape[1]
    q, k = np.abs(q.astype(np.float64)), np.abs(k.astype(np.float64))
    group = len(q) // len(k)
    s = max(float((q[h] @ k[h // group].T).max()) for h in range(len(q))) * scale * 1.4427
    more = 3.02 * float(k.max() * q.sum(axis=2).max()) * scale * 1.4427 if f16 and i8 else 0.0
    s, sums = s + more, 2 if not more else 4.02
    weight = np.log(2.0) * ((d + 3) * 2.0 ** -24 * s + 2.0 ** -15) + 2.0 ** -22 + (2.0 ** -11 if f16 else 2.0 ** -22)
    return 2 * weight + sums * keys * 2.0 ** -24 + (2.0 ** -11 if f16 else 2.0 ** -22)
