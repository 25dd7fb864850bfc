"""The 8-bit KV cache and its attention on the GPU against tests/kv_model.py:
what the cache holds bit for bit, attention within kv_model.bound (derived from
the arithmetic alone)."""
import ctypes

import numpy as np
import pytest
import torch

from open_rknpu2_lm_infer_amd import _ffi as F
from open_rknpu2_lm_infer_amd import device as D
from open_rknpu2_lm_infer_amd import npu
from tests import kv_model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return D.DeviceContext(0)


class Pair:
    """A cache and its model, driven together."""

    def __init__(self, ctx, qh, kh, d, fmt="i8", block=32, capacity=512, causal=True, rows=256, scale=None, seed=0):
        self.ctx, self.qh, self.kh, self.d, self.causal, self.i8 = ctx, qh, kh, d, causal, fmt == "i8"
        self.scale = float(np.float32(d ** -0.5 if scale is None else scale))
        print(f"qh={qh} kh={kh} d={d} {fmt} block={block} causal={causal} seed={seed}", flush=True)
        self.cache = D.KvCacheQ8(ctx, qh, kh, d, self.scale, capacity, fmt=fmt, block=block, causal=causal,
                                 max_query_rows=rows)
        self.k, self.v = (kv_model.KvModel(kh, d, fmt, block) for _ in range(2))
        self.rng = np.random.default_rng(seed)

    def rows(self, n, dtype=np.float16):
        k = self.rng.standard_normal((self.kh, n, self.d))
        k[:, :, ::17] *= 6.0
        return k.astype(dtype), self.rng.standard_normal((self.kh, n, self.d)).astype(dtype)

    def append(self, k, v):
        self.k.append(k)
        self.v.append(v)
        self.cache.append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())

    def fill(self, n, dtype=np.float16):
        self.append(*self.rows(n, dtype))

    def truncate(self, n):
        self.k.truncate(n)
        self.v.truncate(n)
        self.cache.truncate(n)

    def check_contents(self, first=0, n=None, dtype=torch.float32):
        n = self.k.length - first if n is None else n
        got = [torch.full((self.kh, n, self.d), 77.0, dtype=dtype, device="cuda") for _ in range(2)]
        self.cache.read(first, *got)
        for name, g, m in zip("kv", got, (self.k, self.v)):
            want = m.values()[:, first:first + n]
            if dtype == torch.float16:
                want = want.astype(np.float16)
            assert np.array_equal(g.cpu().numpy(), want, equal_nan=True), f"{name} differs"
        assert self.cache.length == self.k.length

    def check_run(self, rows, position, dtype=torch.float32, q=None):
        print(f"  run rows={rows} position={position} length={self.k.length} {dtype}", flush=True)
        q = self.rng.standard_normal((self.qh, rows, self.d)).astype(np.float16) if q is None else q
        out = torch.full((self.qh, rows, self.d), 77.0, dtype=dtype, device="cuda")
        D.attention_q8(self.ctx, self.cache, torch.from_numpy(q).cuda(), out, position)
        return self.compare(q, out, position)

    def compare(self, q, out, position):
        k, v = self.k.values(), self.v.values()
        want = kv_model.attention(q, k, v, self.scale, position, self.causal)
        got = out.double().cpu().numpy()
        fine = np.isfinite(want)
        assert np.array_equal(np.isfinite(got), fine)
        assert np.array_equal(got[~fine], want[~fine], equal_nan=True)
        top = np.abs(v[np.isfinite(v)]).max()
        most = kv_model.bound(q, np.nan_to_num(k), v, self.scale, out.dtype == torch.float16, self.i8) * top
        assert np.abs(got[fine] - want[fine]).max(initial=0.0) <= most
        return got


# --- contents -------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("block", [32, 64, 128])
def test_contents_match_the_definition(ctx, d, fmt, block):
    """Appends of odd sizes, over block ends and over several blocks, read back
    whole and in pieces, as f32 and as fp16."""
    p = Pair(ctx, 4, 2, d, fmt, block, capacity=1024, seed=d + block)
    for n in (1, 30, 1, 2, block - 1, 3 * block + 5, 1, 129):
        p.fill(n)
        p.check_contents()
    p.check_contents(dtype=torch.float16)
    p.check_contents(block - 1, 2)
    p.check_contents(5, block + 60)
    p.check_contents(p.k.length - 1, 1)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_f32_rows_strides_and_odd_addresses(ctx, fmt):
    """f32 rows (rounded to fp16), token-major views, padded strides and element
    alignment, in and out; what lies between rows stays."""
    p = Pair(ctx, 2, 2, 64, fmt, 32, seed=9)
    k, v = p.rows(75, np.float32)
    p.k.append(k)
    p.v.append(v)
    both = torch.from_numpy(np.concatenate([k, v]).transpose(1, 0, 2).copy()).cuda()  # [rows][heads][d]
    p.cache.append(both[:, :2].transpose(0, 1), both[:, 2:].transpose(0, 1))
    p.check_contents()
    for dtype in (torch.float16, torch.float32):
        k, v = p.rows(40, np.float16)
        flat = torch.zeros(2, 2 * 40 * 69 + 3, dtype=dtype, device="cuda")
        views = [flat[i, 3:].as_strided((2, 40, 64), (40 * 69, 69, 1), flat[i, 3:].storage_offset()) for i in range(2)]
        for view, x in zip(views, (k, v)):
            view.copy_(torch.from_numpy(x))
        p.k.append(k)
        p.v.append(v)
        p.cache.append(*views)
        p.check_contents()
        flat.fill_(5.0)
        p.cache.read(60, *views)
        for i, m in enumerate((p.k, p.v)):
            assert np.array_equal(views[i].float().cpu().numpy(),
                                  m.values()[:, 60:100].astype(np.float16 if dtype == torch.float16 else np.float32))
            views[i].fill_(5.0)
        assert bool((flat == 5.0).all())


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_borders_zeros_and_extremes(ctx, fmt):
    """Quotients on a border of two codes, blocks of zeros, of the smallest
    subnormal and of the largest fp16, rows that overflow fp16, infinities, NaN."""
    p = Pair(ctx, 1, 1, 64, fmt, 32, seed=11)
    top = int(kv_model.TOP[fmt])
    grid = np.arange(-top, top + 1) / (2.0 * top) * 2.0  # x / a in steps of half a code
    for a in (127.0, 448.0, 1.75, 65504.0, 2.0 ** -24, 3 * 2.0 ** -24, 0.0):
        x = (p.rng.choice(grid, (1, 32, 64)) * a).astype(np.float16)
        x[0, 7, 9] = -a
        p.append(x, x[:, ::-1].copy())
    x = p.rng.standard_normal((1, 32, 64)).astype(np.float32)
    for bad in (70000.0, np.inf, -np.inf, np.nan):
        x[0, 31, 63] = bad
        p.append(x, x)
    p.fill(9)
    p.check_contents()


def test_truncation_and_drafts(ctx):
    """Taking back any part of the last append, the tail or the last complete
    block is exact, however often; a deeper one continues from the codes; what was
    read stays readable."""
    for block in (32, 64):
        p = Pair(ctx, 2, 2, 64, "i8", block, seed=block)
        p.fill(250)
        for draft in (1, 5, block, 2 * block + 3, 3 * block):
            at = p.k.length
            p.fill(draft)
            p.check_contents()
            p.truncate(at + draft // 2)
            p.truncate(at)
            p.check_contents()
            p.fill(3)
            p.check_contents()
        n = p.k.length
        p.truncate(n - n % block - 7)  # into the last complete block
        p.check_contents()
        p.fill(2)
        p.check_contents()
        p.truncate(block + 11)  # deep
        assert p.k.deep
        p.check_contents()
        p.check_run(3, block + 8)
        p.truncate(block + 5)
        p.check_contents()
        p.fill(4)
        p.check_contents()
        p.check_run(5, p.k.length - 5)
        p.truncate(block + 3)  # (a part of what the codes gave is kept again)
        p.fill(2 * block)
        p.check_contents()
        p.truncate(7)
        p.fill(block - 7)  # completes the block it was cut into
        p.check_contents()
        p.truncate(block)
        p.check_contents()
        p.truncate(0)
        assert p.cache.length == 0
        p.fill(1)
        p.check_contents()


def test_growth_keeps_everything(ctx):
    p = Pair(ctx, 2, 2, 128, "e4m3", 32, capacity=1000, seed=4)
    small = D.KvCacheQ8(ctx, 2, 2, 128, p.scale, 1000, fmt="e4m3", block=32, initial_capacity=64)
    p.cache = small
    assert small.info().capacity == 64 and small.info().max_capacity == 1024
    p.fill(50)
    with pytest.raises(npu.NpuError):
        p.cache.append(torch.zeros(2, 15, 128, device="cuda"), torch.zeros(2, 15, 128, device="cuda"))
    assert small.length == 50
    g = small.info().generation
    small.reserve(700)
    assert small.info().capacity == 704 and small.info().generation == g + 1
    p.check_contents()
    p.fill(640)
    p.truncate(333)
    small.reserve(1024)
    p.check_contents()
    p.fill(500)
    p.check_contents()
    p.check_run(7, p.k.length - 7)
    with pytest.raises(npu.NpuError):
        small.reserve(1025)


# --- attention ------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_attention_row_counts(ctx, d, fmt, dtype):
    """1 to 65 query rows per query head: every row tile, with rows past the last
    one, over blocks and tail; causal rows inside and at the end of the context."""
    p = Pair(ctx, 6, 2, d, fmt, 32, seed=d)
    p.fill(300)
    for rows in (1, 5, 6, 11, 23, 65):
        p.check_run(rows, p.k.length - rows, dtype)
    p.check_run(9, 17, dtype)
    p.check_run(33, 0, dtype)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("length", [33, 64, 100, 129, 300, 1111, 1400])
def test_attention_much_work_kernel(ctx, d, fmt, length):
    """The kernel for much work, forced onto short contexts: one stage, odd and even
    counts of them, a tail, several splits, rows past the last block's."""
    with D.plan_switch("HM_Q8_TILE", 1):
        for causal, block, dtype in ((True, 32, torch.float32), (False, 64, torch.float16), (True, 128, torch.float16)):
            p = Pair(ctx, 6, 2, d, fmt, block, causal=causal, capacity=1500, seed=d + length)
            p.fill(length)
            for rows in (1, 33, min(90, length)):
                p.check_run(rows, length - rows if length >= rows else 0, dtype)
    p.check_run(1, 0, torch.float32)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("length", [40, 100, 129, 600, 1400])
def test_attention_wide_heads_of_two_row_groups(ctx, fmt, length):
    """Heads of 256, two row groups a wave, forced onto short contexts."""
    with D.plan_switch("HM_Q8_TILE", 2):
        for causal, block, dtype in ((True, 32, torch.float32), (False, 128, torch.float16)):
            p = Pair(ctx, 6, 2, 256, fmt, block, causal=causal, capacity=1500, seed=length)
            p.fill(length)
            for rows in (1, 11, 33):
                p.check_run(rows, length - rows, dtype)


def test_kernels_by_work(ctx):
    """Calls that take two row groups of 256 by themselves: the same bits as forced."""
    p = Pair(ctx, 8, 1, 256, "e4m3", 32, capacity=9000, seed=4)
    p.fill(9000)
    q = torch.randn(8, 160, 256, device="cuda", dtype=torch.float16)
    outs = []
    for value in (-1, 2, 0):
        with D.plan_switch("HM_Q8_TILE", value):
            outs.append(torch.empty(8, 160, 256, device="cuda"))
            D.attention_q8(ctx, p.cache, q, outs[-1], 9000 - 160)
    assert torch.equal(outs[0], outs[1]) and not torch.equal(outs[0], outs[2])
    p.compare(q[:, :4].cpu().numpy(), outs[0][:, :4], 9000 - 160)


def test_much_work_takes_its_kernel(ctx):
    """A call large enough for it by itself, 256 rows of 8 heads over 17000 keys of
    256: the same bits as forced, others than without."""
    p = Pair(ctx, 8, 1, 256, "i8", 64, capacity=17000, seed=3)
    p.fill(17000)
    q = torch.randn(8, 256, 256, device="cuda", dtype=torch.float16)
    outs = []
    for value in (-1, 1, 0):
        with D.plan_switch("HM_Q8_TILE", value):
            outs.append(torch.empty(8, 256, 256, device="cuda"))
            D.attention_q8(ctx, p.cache, q, outs[-1], 17000 - 256)
    assert torch.equal(outs[0], outs[1]) and not torch.equal(outs[0], outs[2])
    assert torch.allclose(outs[0], outs[2], rtol=0, atol=1e-4)
    p.compare(q[:, :4].cpu().numpy(), outs[0][:, :4], 17000 - 256)


@pytest.mark.parametrize("tile", [0, 1, 2])
def test_special_values_in_both_kernels(ctx, tile):
    """Poisoned blocks, infinities of the tail, scales far apart and late maxima, each
    kernel forced."""
    with D.plan_switch("HM_Q8_TILE", tile):
        test_scales_of_all_sizes_share_a_row(ctx)
        test_not_finite_values(ctx)
        test_peaked_scores(ctx)
        test_wide_heads_not_finite_over_splits(ctx)


@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 160, 255, 257])
def test_attention_lengths(ctx, length):
    """Contexts of one token, of the tail alone, of whole blocks and of both, with
    and without the mask, 32- and 128-token blocks."""
    for block, causal, fmt in ((32, True, "i8"), (128, False, "e4m3"), (64, False, "i8")):
        p = Pair(ctx, 4, 2, 64, fmt, block, causal=causal, seed=length)
        p.fill(length)
        rows = min(length, 19)
        p.check_run(rows, length - rows)
        p.check_run(1, 0, torch.float16)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("qh,kh,d,rows,length", [(32, 8, 128, 1, 4001), (32, 8, 128, 4, 3970), (16, 2, 256, 1, 5000),
                                                 (16, 8, 64, 40, 3000), (32, 8, 128, 128, 2050), (16, 2, 256, 70, 1100),
                                                 (8, 1, 128, 256, 1500), (3, 3, 64, 256, 900), (1, 1, 128, 1, 9000)])
def test_attention_split_over_blocks(ctx, qh, kh, d, rows, length, causal):
    """Keys spread over blocks whose partial results meet, few rows and many."""
    for i, dtype in enumerate((torch.float32, torch.float16)):
        p = Pair(ctx, qh, kh, d, ("i8", "e4m3")[i], (64, 32)[i], capacity=length, causal=causal, seed=rows + length)
        p.fill(length)
        p.check_run(rows, length - rows, dtype)


def test_attention_strides_and_f32_queries(ctx):
    """Token-major queries and outputs, padded strides, element alignment; f32
    queries are rounded to fp16."""
    p = Pair(ctx, 4, 2, 64, "i8", 32, seed=21)
    p.fill(200)
    q = p.rng.standard_normal((4, 37, 64)).astype(np.float32)
    q16 = q.astype(np.float16)
    for qt, ot in ((torch.float32, torch.float32), (torch.float16, torch.float16), (torch.float32, torch.float16)):
        src = torch.from_numpy(q).cuda().to(qt).transpose(0, 1).contiguous().transpose(0, 1)
        flat = torch.full((37 * 4 * 71 + 1,), 9.0, dtype=ot, device="cuda")
        out = flat[1:].as_strided((4, 37, 64), (71, 4 * 71, 1), 1)
        D.attention_q8(p.ctx, p.cache, src, out, 150)
        p.compare(q16, out, 150)
        out.fill_(9.0)
        assert bool((flat == 9.0).all())


def test_scales_of_all_sizes_share_a_row(ctx):
    """Blocks whose K and V differ by up to 2^30 in scale, and scores that put the
    weight on any of them: neither the sums nor the products lose the small ones."""
    for fmt in ("i8", "e4m3"):
        p = Pair(ctx, 2, 1, 64, fmt, 32, seed=31)
        for kx, vx in ((1.0, 1.0), (1.0, 2.0 ** -20), (30.0, 2.0 ** -10), (0.0, 1.0), (1.0, 0.0), (1e-6, 1e4),
                       (4.0, 2.0 ** -23), (1.0, 100.0)):
            k, v = p.rows(32)
            p.append((k * np.float16(kx)).astype(np.float16), (v.astype(np.float64) * vx).astype(np.float16))
        p.append(*[x * np.float16(s) for x, s in zip(p.rows(20), (1.0, 2.0 ** -8))])
        for rows in (1, 9, 40):
            p.check_run(rows, p.k.length - rows)
        # one tiny-valued block alone in sight, and the tail after it: relative
        # to that block's values
        q = Pair(ctx, 1, 1, 64, fmt, 32, causal=False, seed=32)
        k, v = q.rows(32)
        q.append(k, (v * np.float16(2.0 ** -14)).astype(np.float16))
        k, v = q.rows(17)
        q.append(k, (v * np.float16(2.0 ** -14)).astype(np.float16))
        for rows in (1, 3):
            q.check_run(rows, 0)


def test_what_lies_behind_the_last_row_does_not_count(ctx):
    """A truncated tail leaves large, infinite and NaN rows behind its end: a run
    gives the bits that it gives on a cache that never held them."""
    outs = []
    q = torch.randn(2, 5, 64, device="cuda", dtype=torch.float16)
    for after in (None, 60000.0, float("inf"), float("nan")):
        p = Pair(ctx, 2, 1, 64, "i8", 32, seed=33)
        k, v = p.rows(45)
        p.append(k, (v * np.float16(2.0 ** -14)).astype(np.float16))
        if after is not None:
            x = np.full((1, 19, 64), after, np.float16)
            p.append(x, x)
            p.truncate(45)
        outs.append(torch.empty(2, 5, 64, device="cuda"))
        D.attention_q8(ctx, p.cache, q, outs[-1], 40)
        p.compare(q.cpu().numpy(), outs[-1], 40)
    assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_peaked_scores(ctx):
    """Scores hundreds apart: the maximum moves late and by much, almost all of the
    weight lies on one key."""
    for causal in (True, False):
        p = Pair(ctx, 4, 2, 128, "i8", 32, causal=causal, capacity=1024, scale=1.0, seed=41)
        p.fill(700)
        for rows, dtype in ((1, torch.float32), (16, torch.float16), (30, torch.float32)):
            p.check_run(rows, 700 - rows, dtype)


def test_not_finite_values(ctx):
    """An infinity or NaN in the tail shows for the rows that see its token only;
    in a complete block the block reads as NaN; a masked block shows nothing."""
    p = Pair(ctx, 4, 2, 64, "i8", 32, seed=51)
    p.fill(64)
    k, v = p.rows(20)
    v[0, 3, 5], v[1, 10, 7], v[1, 12, 7], v[0, 15, 60] = np.inf, -np.inf, np.inf, np.nan
    p.append(k, v)
    got = p.check_run(20, 64)
    assert np.isinf(got).any() and np.isnan(got).any() and np.isfinite(got[:, :3]).all()
    p.check_run(1, 66)
    p.check_run(20, 64, torch.float16)
    # K of the tail: a NaN score makes the row NaN, from its token on
    p.truncate(64)
    k, v = p.rows(20)
    k[0, 8, 2] = np.nan
    p.append(k, v)
    out = torch.empty(4, 20, 64, device="cuda")
    q = p.rng.standard_normal((4, 20, 64)).astype(np.float16)
    D.attention_q8(ctx, p.cache, torch.from_numpy(q).cuda(), out, 64)
    out = out.cpu().numpy()
    assert np.isnan(out[:2, 8:]).all() and np.isfinite(out[:2, :8]).all() and np.isfinite(out[2:]).all()
    # a complete block with an infinity: rows that see none of it are as ever
    p.fill(12)
    assert np.isnan(p.k.values()[0, 64:96]).all()
    p.check_contents()
    p.check_run(64, 0)
    out = torch.empty(4, 40, 64, device="cuda")
    q = p.rng.standard_normal((4, 40, 64)).astype(np.float16)
    D.attention_q8(ctx, p.cache, torch.from_numpy(q).cuda(), out, 50)
    out = out.cpu().numpy()
    assert np.isnan(out[:2, 14:]).all() and np.isfinite(out[:2, :14]).all() and np.isfinite(out[2:]).all()


def test_wide_heads_not_finite_over_splits(ctx):
    """The same with the keys spread over blocks, head_dim 256 and a long tail."""
    p = Pair(ctx, 2, 1, 256, "e4m3", 128, capacity=4096, causal=False, seed=52)
    p.fill(2048)
    k, v = p.rows(100)
    v[0, 99, 3], v[0, 40, 255] = np.inf, -np.inf
    p.append(k, v)
    p.check_run(1, 0)
    p.check_run(17, 0, torch.float16)


# --- streams, graphs, refusals ----------------------------------------------------

def test_other_streams(ctx):
    """The calls go to the stream they are given: the result is there when that
    stream is done, behind work that it waits for."""
    p = Pair(ctx, 8, 2, 128, "i8", 32, capacity=2048, seed=61)
    k, v = p.rows(1000)
    q = p.rng.standard_normal((8, 3, 128)).astype(np.float16)
    src = [torch.from_numpy(x).cuda() for x in (k, v, q)]
    late = [torch.zeros_like(x) for x in src]
    out = torch.empty(8, 3, 128, device="cuda")
    ws = ctx.attention_workspace(p.cache)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            big = big @ big * 1e-3
        for a, b in zip(late, src):
            a.copy_(b)
        p.cache.append(late[0], late[1])
        D.attention_q8(ctx, p.cache, late[2], out, 997, ws=ws)
        for a in late:
            a.zero_()
    s.synchronize()
    p.k.append(k)
    p.v.append(v)
    p.compare(q, out, 997)
    p.check_contents()


def test_captured_step_replays(ctx):
    """A captured append, read and run: each replay gives what the eager calls
    give, with eager work between, also where the append completes blocks."""
    for rows, held in ((1, 95), (1, 500), (40, 77), (100, 40)):
        p = Pair(ctx, 8, 2, 64, "e4m3", 32, capacity=1024, seed=rows)
        p.fill(held)
        k, v = p.rows(rows)
        q = p.rng.standard_normal((8, rows, 64)).astype(np.float16)
        kt, vt, qt = (torch.from_numpy(x).cuda() for x in (k, v, q))
        out = torch.zeros(8, rows, 64, device="cuda")
        back = [torch.zeros(2, held + rows, 64, device="cuda") for _ in range(2)]
        ws = ctx.attention_workspace(p.cache)

        def step():
            p.cache.append(kt, vt)
            D.attention_q8(ctx, p.cache, qt, out, held, ws=ws)
            p.cache.read(0, *back)

        p.k.append(k)
        p.v.append(v)
        step()
        torch.cuda.synchronize()
        eager = [out.clone()] + [b.clone() for b in back]
        p.compare(q, out, held)
        p.cache.truncate(held)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for i in range(4):
            for t in [out] + back:
                t.fill_(3.0)
            torch.randn(1000, device="cuda").sum()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(eager, [out] + back):
                assert torch.equal(a, b), f"replay {i}"
        assert p.cache.length == held + rows
        p.fill(9)
        p.check_contents()


@pytest.mark.parametrize("kh,n", [(1, 270001), (8, 33100)])
def test_narrow_heads_over_many_keys(ctx, kh, n):
    """Heads of 64 over keys enough for two blocks a CU: 256 splits of one head (the
    most there are) and 64 of eight; against 64 bits of the values read."""
    print(f"kh={kh} keys={n}", flush=True)
    cache = D.KvCacheQ8(ctx, 2 * kh, kh, 64, 0.125, n, fmt="e4m3", max_query_rows=4)
    x = torch.randn(kh, n, 64, device="cuda", dtype=torch.float16)
    cache.append(x, torch.randn_like(x))
    k, v = (torch.empty(kh, n, 64, device="cuda") for _ in range(2))
    cache.read(0, k, v)
    q = torch.randn(2 * kh, 4, 64, device="cuda", dtype=torch.float16)
    out = torch.empty(2 * kh, 4, 64, device="cuda")
    D.attention_q8(ctx, cache, q, out, n - 4)
    for h in (0, 2 * kh - 1):
        for r in (0, 3):
            seen = n - 3 + r
            score = (k[h // 2, :seen].double() * q[h, r].double()).sum(1) * 0.125
            want = (torch.softmax(score, 0)[:, None] * v[h // 2, :seen].double()).sum(0)
            most = kv_model.bound(q[h:h + 1, r:r + 1].cpu().numpy(), k[h // 2:h // 2 + 1].cpu().numpy(), None, 0.125, False)
            assert float((out[h, r].double() - want).abs().max()) <= most * float(v.abs().max())


@pytest.mark.parametrize("d,kh", [(64, 16), (128, 8), (256, 4)])
def test_long_averages_of_f16_output(ctx, d, kh):
    """Equal weights over many keys in one split, where sums of offset codes would
    outgrow those of codes: no further from 64 bits than the kernel that multiplies
    codes. Both errors are roundings of weights and outputs, 1024 independent values
    each, so either's root mean square has a relative standard deviation of 1024^-.5 /
    2^.5 = 2.2 %, their ratio 3.1 %: 1.2 is six of them."""
    n, m, qh = 100000, 256, 32
    print(f"d={d} kh={kh} keys={n}", flush=True)
    cache = D.KvCacheQ8(ctx, qh, kh, d, d ** -0.5, n, causal=False, max_query_rows=m)
    x = torch.randn(kh, n, d, device="cuda", dtype=torch.float16)
    cache.append(x, torch.randn_like(x))
    values = [torch.empty(kh, n, d, device="cuda") for _ in range(2)]
    cache.read(0, *values)
    want = values[1].double().mean(1)
    q, errors = torch.zeros(qh, m, d, device="cuda", dtype=torch.float16), []
    for kernel in (2, 1):
        out = torch.empty(qh, m, d, device="cuda", dtype=torch.float16)
        with D.plan_switch("HM_Q8_TILE", kernel):
            D.attention_q8(ctx, cache, q, out, 0)
        errors.append(float((out[::qh // kh, m - 1].double() - want).square().mean().sqrt()))
    assert errors[0] <= 1.2 * errors[1], errors


def test_repeated_calls_give_the_same_bits(ctx):
    p = Pair(ctx, 32, 8, 128, "i8", 32, capacity=4096, seed=71)
    p.fill(3000)
    for rows, dtype in ((1, torch.float32), (64, torch.float16)):
        q = torch.randn(32, rows, 128, device="cuda", dtype=torch.float16)
        outs = [torch.empty(32, rows, 128, dtype=dtype, device="cuda") for _ in range(3)]
        for o in outs:
            D.attention_q8(ctx, p.cache, q, o, 3000 - rows)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_refusals(ctx):
    """Wrong shapes, types, places, positions and geometries change nothing."""
    L = F.lib()
    p = Pair(ctx, 4, 2, 64, "i8", 32, capacity=96, rows=8, seed=81)
    p.fill(50)
    ws = ctx.attention_workspace(p.cache)
    raw, good = p.cache.handle.raw, torch.zeros(4, 8, 64, device="cuda")

    def heads(t, **kw):
        h = D._heads(t, *t.shape[::2])
        for name, value in kw.items():
            setattr(h, name, value)
        return ctypes.byref(h)

    q, kv = heads(good), heads(good[:2])
    bad = F.RK_NPU_ERR_PARAM
    for rows, position in ((0, 0), (-1, 0), (9, 0), (1, -1), (1, 50), (8, 43), (1, 2 ** 31 - 1)):
        assert L.rk_npu_hip_attention_q8_device_run(ws.raw, raw, q, rows, position, q, None) == bad
    host = np.zeros(4 * 8 * 64, np.float32)
    for kw in (dict(data=None), dict(type=2), dict(type=-1), dict(head_stride=-64), dict(row_stride=-64),
               dict(data=good.data_ptr() + 2), dict(data=host.ctypes.data)):
        assert L.rk_npu_hip_attention_q8_device_run(ws.raw, raw, heads(good, **kw), 1, 0, q, None) == bad
        assert L.rk_npu_hip_attention_q8_device_run(ws.raw, raw, q, 1, 0, heads(good, **kw), None) == bad
        assert L.rk_npu_hip_attention_q8_device_append(raw, heads(good[:2], **kw), kv, 1, None) == bad
        assert L.rk_npu_hip_attention_q8_device_append(raw, kv, heads(good[:2], **kw), 1, None) == bad
        assert L.rk_npu_hip_attention_q8_device_read(raw, 0, 1, heads(good[:2], **kw), None, None) == bad
    # outputs whose rows overlap
    for kw in (dict(row_stride=63), dict(head_stride=8 * 64 - 1), dict(row_stride=0), dict(head_stride=0)):
        assert L.rk_npu_hip_attention_q8_device_run(ws.raw, raw, q, 8, 0, heads(good, **kw), None) == bad
        assert L.rk_npu_hip_attention_q8_device_read(raw, 0, 8, heads(good[:2], **kw), None, None) == bad
    for first, rows in ((0, 0), (-1, 1), (0, 51), (50, 1), (2 ** 31 - 1, 2 ** 31 - 1), (49, 2)):
        assert L.rk_npu_hip_attention_q8_device_read(raw, first, rows, kv, kv, None) == bad
    assert L.rk_npu_hip_attention_q8_device_read(raw, 0, 1, None, None, None) == bad
    for rows in (0, -1, 47, 2 ** 31 - 1):
        assert L.rk_npu_hip_attention_q8_device_append(raw, kv, kv, rows, None) == bad
    for n in (-1, 51):
        assert L.rk_npu_hip_attention_q8_cache_truncate(raw, n) == bad
    assert L.rk_npu_hip_attention_q8_cache_reserve(ctx.shared.ctx.raw, raw, 97) == bad
    # a workspace of another geometry, a cache of another kind, an empty cache
    other = Pair(ctx, 4, 2, 64, "i8", 32, rows=8, scale=0.5)
    assert L.rk_npu_hip_attention_q8_device_run(ctx.attention_workspace(other.cache).raw, raw, q, 1, 0, q, None) == bad
    assert L.rk_npu_hip_attention_q8_device_run(ctx.attention_workspace(other.cache).raw, other.cache.handle.raw, q, 1,
                                                0, q, None) == bad
    assert L.rk_npu_hip_attention_run(ws.raw, raw, good.data_ptr(), 1, 0, good.data_ptr(), 0, None) == bad
    assert L.rk_npu_hip_attention_q8_device_append(ws.raw, kv, kv, 1, None) == bad
    for t in (good.double(), good.transpose(1, 2), good[:3], good.cpu(), good[0]):
        with pytest.raises(npu.NpuError):
            D.attention_q8(ctx, p.cache, t, t, 0)
    cfg = F.rk_npu_hip_attention_q8_config()
    L.rk_npu_hip_attention_q8_config_init(ctypes.byref(cfg))
    cfg.attention.head_dim = 96
    out = ctypes.c_void_p(1)
    assert L.rk_npu_hip_attention_q8_cache_create(ctx.domain, ctypes.byref(cfg),
                                                  ctypes.byref(out)) == F.RK_NPU_ERR_UNSUPPORTED
    assert not out.value
    p.check_contents()
    p.check_run(8, 42)


def test_failed_allocations_leave_the_cache_whole(ctx):
    L = F.lib()
    cfg = F.rk_npu_hip_attention_q8_config()
    L.rk_npu_hip_attention_q8_config_init(ctypes.byref(cfg))
    stats = F.rk_npu_domain_memory_stats()
    assert L.rk_npu_iommu_domain_memory_stats(ctx.domain, ctypes.byref(stats)) == 0
    live = stats.live_bytes
    out = ctypes.c_void_p(1)
    L.rk_npu_hip_inject_alloc_failures(2)  # (an allocation is tried twice)
    assert L.rk_npu_hip_attention_q8_cache_create(ctx.domain, ctypes.byref(cfg),
                                                  ctypes.byref(out)) == F.RK_NPU_ERR_NOMEM
    L.rk_npu_hip_inject_alloc_failures(0)
    assert not out.value
    assert L.rk_npu_iommu_domain_memory_stats(ctx.domain, ctypes.byref(stats)) == 0 and stats.live_bytes == live
    p = Pair(ctx, 2, 2, 64, seed=5)
    p.cache = D.KvCacheQ8(ctx, 2, 2, 64, p.scale, 512, initial_capacity=64)
    p.fill(60)
    L.rk_npu_hip_inject_alloc_failures(2)
    with pytest.raises(npu.NpuError):
        p.cache.reserve(512)
    L.rk_npu_hip_inject_alloc_failures(0)
    assert p.cache.info().capacity == 64
    p.check_contents()
    p.cache.reserve(512)
    p.fill(100)
    p.check_contents()
