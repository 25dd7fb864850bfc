"""The paged attention where a row's weights lie far apart: each output within a bound
of its own (tests/paged_bound.py), in every kernel, for both output types."""
import numpy as np
import pytest
import torch

from open_rknpu2_lm_infer_amd import device as D
from tests import paged_bound as B

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


@pytest.fixture(scope="module")
def ctx():
    return D.DeviceContext(0)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


class Held:
    """Sequences of one length, k and v [sequences][kh][tokens][d], in pages all over a pool."""

    def __init__(self, ctx, qh, k, v, scale, page=64, causal=True, seed=0):
        self.sequences, self.kh, self.tokens, self.d = k.shape
        self.ctx, self.qh, self.k, self.v, self.scale, self.causal = ctx, qh, k, v, scale, causal
        each = -(-self.tokens // page)
        order = np.random.default_rng(seed).permutation(self.sequences * each)
        self.pages = D.KvPages(ctx, qh, self.kh, self.d, scale, self.sequences * each, page=page, capacity=8192,
                               causal=causal)
        # (room for max_tokens behind the pages, not read)
        self.table = np.full((self.sequences, max(each, 8192 // page)), -1, np.int32)
        self.table[:, :each] = order.reshape(self.sequences, each)
        self.put(k, v)

    def batch(self, rows, **kw):
        return D.PagedBatch(dev(self.table), ints([self.tokens] * self.sequences),
                            ints([rows * s for s in range(self.sequences + 1)]), max_rows=rows, **kw)

    def put(self, k, v):
        wide = [dev(x.transpose(1, 0, 2, 3).reshape(self.kh, -1, self.d)) for x in (k, v)]
        self.pages.append(self.batch(self.tokens), *wide)

    def check(self, q, dtype, **kw):
        """q [sequences][qh][rows][d] at the sequences' ends."""
        rows = q.shape[2]
        print(f"d={self.d} qh={self.qh} kh={self.kh} rows={rows} causal={self.causal} {dtype} {kw}", flush=True)
        one = dtype == F16 and rows * self.qh // self.kh > (16 if self.d == 256 else 32)
        out = torch.full((self.qh, self.sequences * rows, self.d), 77.0, dtype=dtype, device="cuda")
        flat = q.transpose(1, 0, 2, 3).reshape(self.qh, -1, self.d)
        D.attention_paged(self.ctx, self.pages, self.batch(rows, **kw), dev(flat), out)
        self.pages.check()
        got = out.double().cpu().numpy().reshape(self.qh, self.sequences, rows, self.d)
        for s in range(self.sequences):
            want, most = B.attention(q[s], self.k[s], self.v[s], self.scale, self.tokens - rows, self.causal,
                                     dtype == F16, one)
            worst = np.abs(got[:, s] - want) / most
            top = float(worst.max())
            assert top <= 1.0, f"sequence {s}: {top} of the bound at {np.unravel_index(worst.argmax(), worst.shape)}"


# --- a maximum that jumps -----------------------------------------------------------

JUMPS = [9, 16, 23, 24, 25, 26, 31, 40]


def jumping(ctx, d, causal, units, seed):
    """Sequences of `units` units, each with a jump of its own, at a unit of its own."""
    rng = np.random.default_rng(seed)
    cases = [(1 + (5 * i + seed) % (units - 1), (0.0, 5.875, 7.875)[i % 3], float(JUMPS[i % 8])) for i in range(24)]
    made = [[B.jumps(rng, d, units, at, high, jump) for _ in range(2)] for at, high, jump in cases]
    q, k, v = (np.stack([np.stack([head[i] for head in heads]) for heads in made]) for i in range(3))
    return np.repeat(q, 4, axis=1), Held(ctx, 8, k, v, B.SCALE, causal=causal, seed=seed)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_maximum_that_jumps(ctx, d, causal, dtype):
    """Keys of the unit before a jump count in the output as in the sum: kernels of few
    rows and of many, in stages of one unit and of two (many tokens allowed), in one
    piece and split."""
    q, held = jumping(ctx, d, causal, 12, d)
    for rows in (1, 4, 8, 20):
        for most in (384, 8192):
            held.check(q[:, :, :rows], dtype, max_tokens=most)
    q, held = jumping(ctx, d, causal, 31, d + 1)   # (an odd number of units, split)
    for rows in (8, 20):
        held.check(q[:, :, :rows], dtype, max_tokens=992)


# --- values at the end of fp16's range -----------------------------------------------

@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_the_largest_values(ctx, d, causal):
    """Keys of like weight, which rounds up by nearly half a step, and values of 65504 and
    -65504: a mean of finite values is finite."""
    tokens = 400
    k = np.zeros((2, 2, tokens, d), np.float16)
    k[..., 0] = np.log2(1.0 + 1.03 * 2.0 ** -11)
    v = np.full((2, 2, tokens, d), 65504.0, np.float16)
    v[..., ::2] *= -1
    v[..., 5] = 1.0
    q = np.zeros((2, 8, 20, d), np.float16)
    q[..., 0] = 1.0
    held = Held(ctx, 8, k, v, B.SCALE, causal=causal)
    for dtype in (F32, F16):
        for rows in (1, 4, 8, 20):
            for most in (400, 8192):
                held.check(q[:, :, :rows], dtype, max_tokens=most)
