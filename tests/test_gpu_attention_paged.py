"""The paged KV cache on the GPU against tests/paged_model.py: what its pages hold,
attention within paged_model's bounds (derived from the arithmetic alone)."""
import ctypes

import numpy as np
import pytest
import torch

from open_rknpu2_lm_infer_amd import _ffi as F
from open_rknpu2_lm_infer_amd import device as D
from open_rknpu2_lm_infer_amd import npu
from tests import paged_model as M

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return D.DeviceContext(0)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


class Pool:
    """Pages and what they hold: per sequence the tokens' K and V, as fp16 values."""

    def __init__(self, ctx, qh, kh, d, sequences, page=64, most=512, causal=True, seed=0, spare=3, scale=None, **rope):
        print(f"qh={qh} kh={kh} d={d} sequences={sequences} page={page} causal={causal} seed={seed} {rope}", flush=True)
        self.ctx, self.qh, self.kh, self.d, self.page, self.causal = ctx, qh, kh, d, page, causal
        self.rng = np.random.default_rng(seed)
        each = -(-most // page)
        self.scale = float(np.float32(d ** -0.5 if scale is None else scale))
        self.pages = D.KvPages(ctx, qh, kh, d, self.scale, sequences * each + spare, page=page,
                               capacity=each * page, causal=causal, **rope)
        self.table = self.rng.permutation(sequences * each + spare)[:sequences * each].reshape(sequences, each).astype(np.int32)
        self.k = [np.zeros((kh, 0, d), np.float16) for _ in range(sequences)]
        self.v = [np.zeros((kh, 0, d), np.float16) for _ in range(sequences)]

    def lengths(self):
        return [x.shape[1] for x in self.k]

    def batch(self, rows, lengths=None, pad=0, **kw):
        """rows: of each sequence. pad: rows of the arrays before the first."""
        offsets = np.concatenate([[0], np.cumsum(rows)]) + pad
        lengths = self.lengths() if lengths is None else lengths
        kw.setdefault("max_rows", max(1, max(rows)))
        return D.PagedBatch(dev(self.table), ints(lengths), ints(offsets.tolist()), **kw)

    def rows(self, n, heads, dtype=np.float16, outliers=False):
        x = self.rng.standard_normal((heads, n, self.d))
        if outliers:
            x[:, :, ::17] *= 6.0
        return x.astype(dtype)

    def fill(self, counts, dtype=np.float16):
        """Appends counts[s] rows to each sequence (no rotation)."""
        total = sum(counts)
        k, v = self.rows(total, self.kh, dtype, True), self.rows(total, self.kh, dtype)
        self.put(counts, k, v)

    def put(self, counts, k, v):
        at = 0
        for s, n in enumerate(counts):
            self.k[s] = np.concatenate([self.k[s], k[:, at:at + n].astype(np.float16)], axis=1)
            self.v[s] = np.concatenate([self.v[s], v[:, at:at + n].astype(np.float16)], axis=1)
            at += n
        if at:
            self.pages.append(self.batch(counts), dev(k), dev(v))

    def check_held(self, dtype=torch.float16):
        lengths = self.lengths()
        got = [torch.full((self.kh, sum(lengths), self.d), 77.0, dtype=dtype, device="cuda") for _ in range(2)]
        self.pages.read(self.batch(lengths), *got)
        self.pages.check()
        for g, m in zip(got, (self.k, self.v)):
            want = np.concatenate(m, axis=1)
            assert np.array_equal(g.cpu().numpy().astype(np.float16), want, equal_nan=True)

    def attend(self, rows, lengths=None, dtype=torch.float32, q=None, ws=None, pad=0, behind=0, **kw):
        """Runs and checks rows[s] newest rows of each sequence; the output."""
        lengths = self.lengths() if lengths is None else lengths
        print(f"  attend rows={rows[:8]} lengths={lengths[:8]} {dtype}", flush=True)
        total = pad + sum(rows) + behind
        q = self.rows(total, self.qh) if q is None else q
        out = torch.full((self.qh, total, self.d), 77.0, dtype=dtype, device="cuda")
        D.attention_paged(self.ctx, self.pages, self.batch(rows, lengths, pad, **kw), dev(q), out, ws=ws)
        self.pages.check()
        self.compare(rows, lengths, q, out, pad)
        return out

    def compare(self, rows, lengths, q, out, pad=0):
        got = out.double().cpu().numpy()
        half, q = out.dtype == torch.float16, q.astype(np.float16)
        one = half and max(rows) * self.qh // self.kh > (16 if self.d == 256 else 32)
        at = pad
        assert np.all(got[:, :pad] == 77.0) and np.all(got[:, pad + sum(rows):] == 77.0), "rows of no sequence changed"
        for s, (n, length) in enumerate(zip(rows, lengths)):
            k, v, mine = self.k[s][:, :length], self.v[s][:, :length], slice(at, at + n)
            at += n
            if n == 0:
                continue
            want = M.attention(q[:, mine], k, v, self.scale, length - n, self.causal)
            fine = np.isfinite(want)
            g = got[:, mine]
            assert np.array_equal(np.isfinite(g), fine), f"sequence {s}"
            assert np.array_equal(g[~fine], want[~fine], equal_nan=True)
            if length == 0:
                assert np.all(g == 0.0)
                continue
            top = np.abs(v[np.isfinite(v)].astype(np.float64)).max(initial=0.0)
            most = M.attention_bound(np.nan_to_num(q[:, mine]), np.nan_to_num(k, posinf=0, neginf=0), self.scale, half, one, length) * top
            err = np.abs(g[fine] - want[fine]).max(initial=0.0)
            assert err <= most, f"sequence {s}: {err} > {most}"


# --- append and read -------------------------------------------------------------

@pytest.mark.parametrize("d,page,rotary,interleaved,dtype", [
    (64, 16, 64, False, np.float16), (64, 32, 16, True, np.float32), (128, 64, 128, False, np.float32),
    (128, 16, 32, False, np.float16), (256, 256, 64, True, np.float16), (256, 128, 256, False, np.float32),
    (128, 64, 0, False, np.float32), (64, 64, 64, True, np.float32)])
def test_append_rotates_and_stores(ctx, d, page, rotary, interleaved, dtype):
    """Ragged rows at every place of a page, in three calls, q rotated in place."""
    p = Pool(ctx, 6, 2, d, 5, page=page, most=400, rotary_dim=rotary, rope_theta=1e5, interleaved=interleaved)
    freq = M.frequencies(rotary, 1e5) if rotary else np.zeros(0)
    lengths = np.zeros(5, int)
    want = [[], []]
    for rows in ([1, 17, 0, 64, 300], [1, 1, 1, 1, 1], [50, 3, 90, 7, 0]):
        total = sum(rows)
        k, v, q = p.rows(total, 2, dtype), p.rows(total, 2, dtype), p.rows(total, 6, dtype)
        before = lengths.copy()
        lengths += rows
        where = np.concatenate([np.arange(a, b) for a, b in zip(before, lengths)])
        b = p.batch(rows, lengths.tolist())
        qt = dev(q)
        p.pages.append(b, dev(k), dev(v), q=qt, q_out=qt)
        out = [torch.full((2, total, d), 77.0, dtype=torch.float16, device="cuda") for _ in range(2)]
        p.pages.read(b, *out)
        p.pages.check()
        rk, rq = M.rotate(k, where, freq, interleaved), M.rotate(q, where, freq, interleaved)
        assert np.all(np.abs(out[0].double().cpu().numpy() - rk) <= M.rotate_bound(k, rk, True))
        assert np.array_equal(out[1].cpu().numpy(), v.astype(np.float16))
        assert np.all(np.abs(qt.double().cpu().numpy() - rq) <= M.rotate_bound(q, rq, dtype == np.float16) +
                      (2.0 ** -24 * np.abs(rq) if dtype == np.float32 else 0))
        want[0].append((before, rows, out[0].cpu().numpy()))
        want[1].append((before, rows, out[1].cpu().numpy()))
    # everything again, after the later appends
    out = [torch.empty((2, int(lengths.sum()), d), dtype=torch.float32, device="cuda") for _ in range(2)]
    p.pages.read(p.batch(lengths.tolist(), lengths.tolist()), *out)
    begins = np.concatenate([[0], np.cumsum(lengths)])
    for got, calls in zip(out, want):
        got = got.cpu().numpy()
        for before, rows, piece in calls:
            at = 0
            for s, n in enumerate(rows):
                a = begins[s] + before[s]
                assert np.array_equal(got[:, a:a + n], piece[:, at:at + n].astype(np.float32))
                at += n


def test_positions_far_and_given(ctx):
    """Positions of their own, up to the ends of 32 bits, and frequencies of their own."""
    freq = [1.0, 0.7, 1e-3, 3.0, 2.5e-5, 0.0, -1.0, 0.1]
    p = Pool(ctx, 2, 2, 64, 1, most=64, rotary_dim=16, frequencies=freq)
    where = [0, 1, -1, 131071, 1 << 20, (1 << 31) - 1, -(1 << 31), 12345]
    k, q = p.rows(8, 2, np.float32), p.rows(8, 2, np.float32)
    out = torch.full((2, 8, 64), 77.0, dtype=torch.float32, device="cuda")
    b = p.batch([8], [8])
    p.pages.append(b, dev(k), dev(k), q=dev(q), q_out=out, positions=ints(where))
    got = torch.empty((2, 8, 64), dtype=torch.float16, device="cuda")
    p.pages.read(b, got, torch.empty_like(got))
    rk, rq = M.rotate(k, where, freq, False), M.rotate(q, where, freq, False)
    # (a 64-bit angle of up to 2^31 x 3 radians is off by 2^-20 in the model itself: 2^-53 of it)
    slack = np.abs(np.array(where, float))[None, :, None] * 3 * 2.0 ** -52 * np.abs(k).max()
    assert np.all(np.abs(got.double().cpu().numpy() - rk) <= M.rotate_bound(k, rk, True) + slack)
    assert np.all(np.abs(out.double().cpu().numpy() - rq) <= M.rotate_bound(q, rq, False) + 2.0 ** -24 * np.abs(rq) + slack)


def test_strided_token_major_rows(ctx):
    """A projection's [rows][q heads, k heads, v heads] output, q_out with gaps between its rows."""
    p = Pool(ctx, 4, 2, 128, 2, most=128, rotary_dim=128)
    every = p.rng.standard_normal((100, 8, 128)).astype(np.float32)
    t = dev(every).transpose(0, 1)
    room = torch.full((100, 5, 136), 77.0, dtype=torch.float16, device="cuda")
    q_out = room[:, :4, 3:131].transpose(0, 1)
    b = p.batch([63, 37], [63, 37])
    p.pages.append(b, t[4:6], t[6:], q=t[:4], q_out=q_out)
    got = [torch.empty((2, 100, 128), dtype=torch.float16, device="cuda") for _ in range(2)]
    p.pages.read(b, *got)
    where = np.concatenate([np.arange(63), np.arange(37)])
    x = every.transpose(1, 0, 2)
    freq = M.frequencies(128, 1e4)
    rk, rq = M.rotate(x[4:6], where, freq, False), M.rotate(x[:4], where, freq, False)
    assert np.all(np.abs(got[0].double().cpu().numpy() - rk) <= M.rotate_bound(x[4:6], rk, True))
    assert np.array_equal(got[1].cpu().numpy(), x[6:].astype(np.float16))
    assert np.all(np.abs(q_out.double().cpu().numpy() - rq) <= M.rotate_bound(x[:4], rq, True))
    room[:, :4, 3:131] = 77.0
    assert bool((room == 77.0).all()), "values beside q_out's rows changed"


def test_one_row_each_without_offsets(ctx):
    p = Pool(ctx, 2, 1, 64, 70, most=40, page=16)
    n = [int(x) for x in p.rng.integers(0, 40, 70)]
    p.fill(n)
    k, v = p.rows(72, 1), p.rows(72, 1)
    lengths = [x + 1 for x in n]
    lengths[3] = lengths[69] = 0     # idle places
    b = D.PagedBatch(dev(p.table), ints(lengths), max_tokens=40)
    p.pages.append(b, dev(k), dev(v))
    out = torch.full((1, 72, 64), 77.0, dtype=torch.float16, device="cuda")
    ov = out.clone()
    p.pages.read(b, out, ov)
    p.pages.check()
    got = out.cpu().numpy()
    for s in range(72):
        assert np.array_equal(got[:, s], np.full((1, 64), 77.0, np.float16) if s in (3, 69, 70, 71) else k[:, s])
    for s in range(70):
        if lengths[s]:
            p.k[s] = np.concatenate([p.k[s], k[:, s:s + 1]], axis=1)
            p.v[s] = np.concatenate([p.v[s], v[:, s:s + 1]], axis=1)
    p.check_held()
    q = p.rows(72, 2)
    y = torch.full((2, 72, 64), 77.0, dtype=torch.float16, device="cuda")
    D.attention_paged(ctx, p.pages, b, dev(q), y)
    p.pages.check()
    p.compare([1] * 70, lengths, q, y)


# --- attention -------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("qh,kh", [(4, 4), (8, 2), (8, 1), (16, 1)])
def test_one_token(ctx, d, qh, kh):
    """One row a sequence, lengths around every border, every page size."""
    for page, lengths in ((16, [1, 2, 15, 16, 17, 31, 32, 33]), (32, [0, 64, 100, 1]), (64, [63, 65, 400]),
                          (256, [255, 257, 500])):
        p = Pool(ctx, qh, kh, d, len(lengths), page=page, seed=page + d)
        p.fill(lengths)
        for dtype in (torch.float32, torch.float16):
            p.attend([1] * len(lengths), dtype=dtype)


@pytest.mark.parametrize("d,qh,kh", [(64, 8, 8), (128, 8, 2), (256, 4, 1), (128, 6, 2), (64, 48, 2)])
@pytest.mark.parametrize("causal", [True, False])
def test_rows(ctx, d, qh, kh, causal):
    """Ragged rows over ragged lengths: whole prompts, drafts, no rows, rows before the first token."""
    p = Pool(ctx, qh, kh, d, 6, page=32, most=300, causal=causal, seed=d + qh)
    p.fill([40, 1, 129, 300, 77, 0])
    for rows in ([40, 1, 129, 7, 0, 0], [1, 0, 5, 2, 33, 0], [45, 3, 1, 100, 64, 2]):
        for dtype in (torch.float32, torch.float16):
            p.attend(rows, dtype=dtype, pad=2, behind=3)


@pytest.mark.parametrize("d,qh,kh,lengths,rows", [
    (128, 8, 2, [3000, 17, 900], [1, 1, 1]), (64, 4, 1, [5000], [1]), (256, 8, 1, [2000, 1999], [1, 1]),
    (128, 32, 2, [2500, 31], [1, 1]), (64, 8, 2, [4000, 700, 0, 1], [4, 3, 1, 1]), (128, 8, 1, [3000, 40], [20, 40]),
    (256, 4, 2, [1500, 700], [9, 60])])
def test_long_lengths_are_split_and_joined(ctx, d, qh, kh, lengths, rows):
    p = Pool(ctx, qh, kh, d, len(lengths), page=64, most=max(lengths), seed=d)
    p.fill(lengths)
    for dtype in (torch.float32, torch.float16):
        p.attend(rows, dtype=dtype)
        p.attend(rows, dtype=dtype, max_tokens=max(lengths))


@pytest.mark.parametrize("rows", [[1, 0], [3, 4], [100, 57]])
def test_more_rows_allowed_than_there_are(ctx, rows):
    """A batch whose max_rows passes the call's rows: append, read and attention."""
    p = Pool(ctx, 4, 2, 64, 2, page=16, most=200)
    p.fill([30, 20])
    k, v = p.rows(sum(rows), 2), p.rows(sum(rows), 2)
    lengths = [a + n for a, n in zip(p.lengths(), rows)]
    b = p.batch(rows, lengths, max_rows=512)
    p.pages.append(b, dev(k), dev(v))
    got = [torch.empty(2, sum(rows), 64, dtype=torch.float16, device="cuda") for _ in range(2)]
    p.pages.read(b, *got)
    assert np.array_equal(got[0].cpu().numpy(), k) and np.array_equal(got[1].cpu().numpy(), v)
    for s, at in enumerate((0, rows[0])):
        p.k[s] = np.concatenate([p.k[s], k[:, at:at + rows[s]]], axis=1)
        p.v[s] = np.concatenate([p.v[s], v[:, at:at + rows[s]]], axis=1)
    for dtype in (torch.float32, torch.float16):
        p.attend(rows, dtype=dtype, max_rows=512)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_drafts(ctx, d, causal):
    """2 to 8 rows of 4 heads a KV head: every row tile of few rows, whole and split."""
    p = Pool(ctx, 8, 2, d, 5, page=16, most=1500, causal=causal, seed=d)
    p.fill([1500, 5, 33, 700, 64])
    for rows in ([2, 2, 2, 2, 2], [4, 1, 3, 4, 0], [5, 5, 5, 5, 5], [8, 7, 1, 0, 8]):
        for dtype in (torch.float32, torch.float16):
            p.attend(rows, dtype=dtype, behind=1)
    p.attend([8, 7, 1, 0, 8], [1400, 5, 3, 0, 40])


@pytest.mark.parametrize("qh,kh,d", [(64, 1, 64), (256, 1, 64), (32, 32, 128), (40, 1, 256), (96, 3, 64)])
def test_many_heads(ctx, qh, kh, d):
    """One row whose heads fill several row tiles, many KV heads, a number that 8 does not divide."""
    p = Pool(ctx, qh, kh, d, 3, page=32, most=900, seed=qh)
    p.fill([900, 1, 40])
    for dtype in (torch.float32, torch.float16):
        p.attend([1, 1, 1], dtype=dtype)
    n = p.lengths()
    q = p.rows(3, qh)
    out = torch.full((qh, 3, d), 77.0, device="cuda")
    D.attention_paged(ctx, p.pages, D.PagedBatch(dev(p.table), ints(n)), dev(q), out)
    p.compare([1, 1, 1], n, q, out)


@pytest.mark.parametrize("rows", [[700, 40, 500], [900, 700, 500]])
def test_prompts_of_many_blocks(ctx, rows):
    """More row tiles than CUs: long ones first, over all sequences."""
    p = Pool(ctx, 32, 8, 64, 3, page=64, most=1000, seed=1)
    p.fill([rows[0], rows[1] + 33, rows[2]])
    p.attend(rows, dtype=torch.float16, pad=1)


def test_many_sequences_split(ctx):
    """More sequences than a wave has lanes, one long: splits, and a schedule of several a lane."""
    p = Pool(ctx, 4, 2, 64, 150, page=32, most=2100, seed=5)
    n = [int(x) for x in p.rng.integers(0, 60, 150)]
    n[140], n[3] = 2100, 1000
    p.fill(n)
    p.attend([1] * 150)
    p.attend([int(x) for x in p.rng.integers(0, 9, 150)], dtype=torch.float16)
    p.attend([int(x) for x in p.rng.integers(0, 30, 150)])


class Shared:
    """Many sequences over the pages of one, each as long as it says."""

    def __init__(self, ctx, qh, kh, d, sequences, tokens, most=5000, causal=True):
        self.p = Pool(ctx, qh, kh, d, 1, page=64, most=most, causal=causal, seed=d + sequences)
        self.p.fill([tokens])
        self.table = dev(self.p.table).expand(sequences, -1).contiguous()
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device="cuda")

    def attend(self, rows, lengths, dtype, out=None, run=True, max_tokens=5000):
        """rows: of each sequence (None: a row each, no offsets). Only checks where not run."""
        p, each = self.p, [1] * len(lengths) if rows is None else rows
        begins = np.concatenate([[0], np.cumsum(each)])
        if run:
            self.lengths.copy_(ints(lengths))
            offsets = None if rows is None else ints(begins.tolist())
            self.b = D.PagedBatch(self.table, self.lengths, offsets, max_rows=max(each), max_tokens=max_tokens)
            self.q = p.rows(int(begins[-1]), p.qh)
            out = torch.full((p.qh, int(begins[-1]), p.d), 77.0, dtype=dtype, device="cuda")
            D.attention_paged(p.ctx, p.pages, self.b, dev(self.q), out)
            p.pages.check()
        # paged_model's attention and bound, in 64 bits on the GPU
        half, group = out.dtype == torch.float16, p.qh // p.kh
        one = half and max(each) * group > (16 if p.d == 256 else 32)
        most = M.attention_bound(self.q, p.k[0], p.scale, half, one, max(lengths)) * np.abs(p.v[0]).max()
        k, v = (dev(a[0]).double() for a in (p.k, p.v))
        q, got = dev(self.q).double(), out.double()
        for s, (n, length) in enumerate(zip(each, lengths)):
            mine = slice(int(begins[s]), int(begins[s]) + n)
            if n == 0 or length == 0:
                assert bool((got[:, mine] == 0.0).all())
                continue
            scores = p.scale * torch.matmul(q[:, mine].reshape(p.kh, group * n, p.d), k[:, :length].transpose(1, 2).contiguous())
            scores = scores.view(p.kh, group, n, length)
            if p.causal:
                seen = torch.arange(length - n, length, device="cuda")
                scores.masked_fill_(torch.arange(length, device="cuda")[None, :] > seen[:, None], -np.inf)
            weights = torch.softmax(scores, dim=-1).nan_to_num_(0.0)     # (rows that see no token)
            want = torch.matmul(weights.view(p.kh, group * n, length), v[:, :length]).view(p.qh, n, p.d)
            err = float((got[:, mine] - want).abs().max())
            assert err <= most, f"sequence {s}: {err} > {most}"
        return out


@pytest.mark.parametrize("d,qh,kh,sequences,rows", [
    (64, 32, 32, 33, 1), (128, 32, 32, 40, 1), (64, 64, 32, 70, 3), (256, 32, 32, 36, 1), (128, 16, 16, 66, 2), (64, 16, 8, 130, 1),
    (128, 64, 32, 34, 5), (256, 32, 16, 65, 5)])
@pytest.mark.parametrize("causal", [True, False])
def test_long_sequences_among_many(ctx, causal, d, qh, kh, sequences, rows):
    """More sequences than the blocks that splits aim at: one long, some, at the border of
    being split, all of them, none; idle ones and ones of no rows among them."""
    x = Shared(ctx, qh, kh, d, sequences, 2100, causal=causal)
    rng = np.random.default_rng(sequences)
    few = [int(n) for n in rng.integers(0, 70, sequences)]
    for where in ([sequences - 1], [0, 1, 20], [sequences // 2, 5, 31, 32], range(0, sequences, 5), []):
        lengths = list(few)
        for i, s in enumerate(where):
            lengths[s] = (2100, 1025, 1024, 2049, 1057, 2048)[i % 6]
        for dtype in (torch.float32, torch.float16):
            x.attend(None if rows == 1 else [int(n) for n in rng.integers(0, rows + 1, sequences - 1)] + [rows], lengths, dtype)
    lengths = [1200 - 7 * i for i in range(sequences)]
    x.attend(None if rows == 1 else [rows] * sequences, lengths, torch.float16)


def test_a_long_sequence_among_a_thousand(ctx):
    x = Shared(ctx, 8, 8, 64, 1024, 9000, most=9000)
    rng = np.random.default_rng(0)
    for where in ([1023], [0, 1, 500], []):
        lengths = [int(n) for n in rng.integers(0, 50, 1024)]
        for s in where:
            lengths[s] = 9000 - s
        x.attend(None, lengths, torch.float32, max_tokens=9000)
        x.attend([int(n) for n in rng.integers(0, 3, 1023)] + [2], lengths, torch.float16, max_tokens=9000)


def test_a_captured_step_of_many_follows_the_long_ones(ctx):
    """One captured step whose long sequences come and go, and one of a wrong length."""
    x = Shared(ctx, 32, 32, 64, 40, 5000)
    p, ws = x.p, ctx.attention_workspace(x.p.pages, own=True)
    x.attend(None, [30] * 40, torch.float32)
    q, out = dev(x.q), torch.zeros(32, 40, 64, device="cuda")
    D.attention_paged(ctx, p.pages, x.b, q, out, ws=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        D.attention_paged(ctx, p.pages, x.b, q, out, ws=ws)
    for i in range(6):
        lengths = [(7 * s + i) % 60 for s in range(40)]
        for s in range(i):
            lengths[(11 * s + i) % 40] = 5000 - 600 * s
        x.lengths.copy_(ints(lengths))
        out.fill_(77.0)
        graph.replay()
        torch.cuda.synchronize()
        p.pages.check()
        x.attend(None, lengths, torch.float32, out=out, run=False)
    for wrong in (-1, 5001, 2 ** 31 - 1):
        told = [20] * 40
        told[3], told[4] = wrong, 5000
        x.lengths.copy_(ints(told))
        graph.replay()
        with pytest.raises(npu.NpuError):
            p.pages.check()
        told[3] = 0
        x.attend(None, told, torch.float32, out=out, run=False)


@pytest.mark.parametrize("sequences", [100, 300])
def test_a_long_sequence_is_split_among_any_number(ctx, sequences):
    """Keys of one weight, 2^10 in a row's units, whose first 128 values are 2^14: what a wave
    adds of 32 others of 2^-11, 2^4, is less than half a step of its f32 sum, 2^29. One block
    over the whole sequence loses all of them, 2^-16 of the output; of 32 splits and more
    only the first does."""
    tokens = 65536
    p = Pool(ctx, 8, 8, 64, 1, page=256, most=tokens, seed=1)
    v = np.full((8, tokens, 64), 2.0 ** -11, np.float16)
    v[:, :128] = 2.0 ** 14
    p.put([tokens], np.zeros((8, tokens, 64), np.float16), v)
    lengths = [20] * sequences
    lengths[50] = tokens
    b = D.PagedBatch(dev(p.table).expand(sequences, -1).contiguous(), ints(lengths))
    out = torch.empty(8, sequences, 64, device="cuda")
    D.attention_paged(ctx, p.pages, b, dev(p.rows(sequences, 8)), out)
    p.pages.check()
    want = (128 * 2.0 ** 14 + (tokens - 128) * 2.0 ** -11) / tokens
    assert float((out[:, 50].double() / want - 1.0).abs().max()) < 2.0 ** -20
    assert float((out[:, 49].double() / 2.0 ** 14 - 1.0).abs().max()) < 2.0 ** -20


@pytest.mark.parametrize("d,qh,kh,sequences,rows,tokens", [
    (64, 32, 32, 40, 1, 9000), (128, 64, 32, 40, 3, 9000), (64, 32, 8, 33, 16, 9000), (256, 16, 8, 17, 20, 5000)])
def test_long_lengths_in_one_block(ctx, d, qh, kh, sequences, rows, tokens):
    """Blocks that walk thousands of tokens: many sequences over the same pages, a table with room between its rows."""
    p = Pool(ctx, qh, kh, d, 1, page=64, most=tokens, seed=d)
    p.fill([tokens])
    wide = torch.full((sequences, p.table.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    wide[:, :p.table.shape[1]] = dev(p.table)
    q = p.rows(sequences * rows, qh)
    lengths = [tokens - 3 * i for i in range(sequences)]
    b = D.PagedBatch(wide[:, :p.table.shape[1]], ints(lengths), ints([rows * i for i in range(sequences + 1)]), max_rows=rows)
    for dtype in (torch.float32, torch.float16):
        out = torch.full((qh, sequences * rows, d), 77.0, dtype=dtype, device="cuda")
        D.attention_paged(ctx, p.pages, b, dev(q), out)
        p.pages.check()
        assert bool(torch.isfinite(out).all()) and float(out.abs().max()) < 70.0
        for s in (0, sequences // 2, sequences - 1):
            mine = slice(s * rows, (s + 1) * rows)
            p.compare([rows], [lengths[s]], q[:, mine], out[:, mine])


def test_pages_beyond_32_bits(ctx):
    """A pool whose K and V pass 2^32 bytes each, rows in its last pages."""
    pages = D.KvPages(ctx, 8, 8, 256, 0.0625, 4200, page=256, rotary_dim=0)
    assert pages.bytes() == 2 * 4200 * 256 * 8 * 256 * 2 > 2 ** 33
    rng = np.random.default_rng(0)
    k, v = (rng.standard_normal((8, 300, 256)).astype(np.float16) for _ in range(2))
    table = ints([[4199, 4198], [4100, 0]])
    b = D.PagedBatch(table, ints([290, 10]), ints([0, 290, 300]), max_rows=290)
    pages.append(b, dev(k), dev(v))
    got = [torch.empty(8, 300, 256, dtype=torch.float16, device="cuda") for _ in range(2)]
    pages.read(b, *got)
    assert np.array_equal(got[0].cpu().numpy(), k) and np.array_equal(got[1].cpu().numpy(), v)
    for rows in ([1, 1], [20, 10]):
        total = sum(rows)
        q = rng.standard_normal((8, total, 256)).astype(np.float16)
        out = torch.empty(8, total, 256, device="cuda")
        D.attention_paged(ctx, pages, D.PagedBatch(table, ints([290, 10]), ints([0, rows[0], total]), max_rows=rows[0]), dev(q), out)
        pages.check()
        for mine, keys in ((slice(0, rows[0]), slice(0, 290)), (slice(rows[0], total), slice(290, 300))):
            n = mine.stop - mine.start
            want = M.attention(q[:, mine], k[:, keys], v[:, keys], 0.0625, keys.stop - keys.start - n, True)
            most = M.attention_bound(q[:, mine], k[:, keys], 0.0625, False, False, 290) * np.abs(v).max()
            assert np.abs(out.double().cpu().numpy()[:, mine] - want).max() <= most


def test_f32_queries_and_strides(ctx):
    """f32 queries are rounded to fp16; token-major q and output views; no alignment beyond the type's."""
    p = Pool(ctx, 4, 2, 128, 3, most=200)
    p.fill([200, 64, 5])
    rows = [20, 1, 5]
    q = p.rows(26, 4, np.float32)
    p.attend(rows, q=q)
    room = torch.zeros(26 * 4 * 129 + 1, device="cuda")
    qt = room[1:].view(26, 4, 129)[..., :128].transpose(0, 1)
    qt.copy_(dev(q))
    for dtype in (torch.float16, torch.float32):
        back = torch.full((26 * 4 * 131 + 1,), 77.0, dtype=dtype, device="cuda")
        out = back[1:].view(26, 4, 131)[..., 2:130].transpose(0, 1)
        D.attention_paged(p.ctx, p.pages, p.batch(rows), qt, out)
        p.compare(rows, p.lengths(), q, out)
        out.fill_(77.0)
        assert bool((back == 77.0).all())


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("rows", [[1, 1], [6, 3], [70, 33]])
def test_what_lies_behind_a_sequence_does_not_count(ctx, causal, rows):
    """NaN and infinities in the tokens behind a length, in its own last page too."""
    p = Pool(ctx, 8, 2, 128, 2, page=64, most=256, causal=causal, spare=0)
    bad = p.rows(512, 2)
    bad[:] = np.nan
    bad[:, ::3] = np.inf
    bad[:, 1::3] = -np.inf
    p.pages.append(p.batch([256, 256], [256, 256]), dev(bad), dev(bad))
    p.fill([150, 33])
    for dtype in (torch.float32, torch.float16):
        p.attend(rows, dtype=dtype)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_what_lies_behind_a_sequence_costs_nothing(ctx, d):
    """The path for values that are not finite is for those that rows see."""
    times = []
    for fill in (0.0, float("nan")):
        p = Pool(ctx, 4, 4, d, 1, page=256, most=2048, spare=0)
        bad = torch.full((4, 2048, d), fill, dtype=torch.float16, device="cuda")
        p.pages.append(p.batch([2048], [2048]), bad, bad)
        p.fill([1810])
        q = dev(p.rows(330, 4))
        out = torch.empty_like(q)
        b = p.batch([330])
        best = 1e9
        for _ in range(5):
            t = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            t[0].record()
            for _ in range(10):
                D.attention_paged(ctx, p.pages, b, q, out)
            t[1].record()
            torch.cuda.synchronize()
            best = min(best, t[0].elapsed_time(t[1]))
        times.append(best)
        assert bool(torch.isfinite(out).all())
    assert times[1] < 3 * times[0]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [[3], [7], [10], [40], [130]])
def test_wild_values_count_for_the_rows_that_see_them(ctx, d, rows):
    p = Pool(ctx, 4, 2, d, 1, page=16, most=160, seed=d)
    k, v = p.rows(160, 2), p.rows(160, 2)
    v[0, 158, 3], v[0, 159, 3], v[1, 157, 5], v[1, 40, 7], v[1, 130, 9] = np.inf, -np.inf, np.nan, np.inf, -np.inf
    p.put([160], k, v)
    for dtype in (torch.float32, torch.float16):
        p.attend(rows, dtype=dtype)


def test_wild_keys_and_queries(ctx):
    """NaN in a key makes NaN of the rows that see it, NaN in a query of its own row."""
    p = Pool(ctx, 4, 2, 128, 2, page=16, most=100)
    k, v = p.rows(150, 2), p.rows(150, 2)
    k[0, 95, 0] = np.nan
    p.put([100, 50], k, v)
    q = p.rows(60, 4)
    q[2, 11] = np.nan
    p.attend([40, 20], q=q)
    p.attend([2, 2], q=q[:, :4])


def test_scores_far_apart(ctx):
    """Large scales, rows of one key's weight, keys that outdo all before them."""
    p = Pool(ctx, 4, 1, 64, 2, most=300, scale=4.0)
    k, v = p.rows(500, 1), p.rows(500, 1)
    k *= np.linspace(0.1, 4.0, 500).astype(np.float16)[None, :, None]
    p.put([300, 200], k, v)
    for rows in ([1, 1], [4, 4], [64, 20]):
        p.attend(rows)


def test_shared_pages(ctx):
    """Two sequences over the same prefix pages, each with a last page of its own."""
    p = Pool(ctx, 8, 2, 128, 2, page=32, most=128)
    p.table[1, :3] = p.table[0, :3]
    k, v = p.rows(96, 2), p.rows(96, 2)
    p.put([96, 0], k, v)
    p.k[1], p.v[1] = p.k[0].copy(), p.v[0].copy()
    p.fill([10, 32])
    p.check_held()
    p.attend([1, 1])
    p.attend([12, 40], dtype=torch.float16)


def test_many_sequences(ctx):
    """1024 places, most of them short, some idle, some without rows; results do not depend on the batch."""
    p = Pool(ctx, 4, 2, 64, 1024, page=16, most=48, seed=3)
    n = [int(x) for x in p.rng.integers(0, 48, 1024)]
    n[1000] = 48
    p.fill(n)
    out = p.attend([1] * 1024)
    rows = [int(x) for x in p.rng.integers(0, 4, 1024)]
    p.attend(rows, dtype=torch.float16)
    again = torch.empty_like(out)
    q = p.rows(1024, 4)
    for x in (out, again):
        D.attention_paged(ctx, p.pages, p.batch([1] * 1024), dev(q), x)
    assert torch.equal(out, again)


# --- what the device finds wrong ---------------------------------------------------

def test_wrong_pages_lengths_and_offsets(ctx):
    p = Pool(ctx, 4, 2, 64, 3, page=16, most=64)
    p.fill([40, 30, 20])
    q, out = dev(p.rows(6, 4)), torch.full((4, 6, 64), 77.0, device="cuda")
    k = dev(p.rows(6, 2))

    def flawed():
        with pytest.raises(npu.NpuError):
            p.pages.check()
        p.pages.check()          # told once

    def others_right(rows, wrong):
        got = out.cpu().numpy()
        at = 0
        for s, n in enumerate(rows):
            if s != wrong and n:
                want = M.attention(q.cpu().numpy()[:, at:at + n], p.k[s], p.v[s], p.scale, p.k[s].shape[1] - n, True)
                assert np.abs(got[:, at:at + n] - want).max() < 1e-4
            at += n
    good = p.table.copy()
    for page in (-1, len(good) * good.shape[1] + 3, 2 ** 31 - 1, -2 ** 31):
        p.table = good.copy()
        p.table[1, 1] = page
        D.attention_paged(ctx, p.pages, p.batch([2, 2, 2]), q, out)
        flawed()
        others_right([2, 2, 2], 1)
        got = [torch.full((2, 6, 64), 77.0, dtype=torch.float16, device="cuda") for _ in range(2)]
        p.table[1, 1], p.table[2, 1] = good[1, 1], page
        b = p.batch([2, 2, 2])
        p.pages.read(b, *got)
        flawed()
        assert np.array_equal(got[0].cpu().numpy()[:, :2], p.k[0][:, -2:])
        assert bool((got[0][:, 4:] == 77.0).all()) and bool((got[1][:, 4:] == 77.0).all())
        p.pages.append(b, got[0], got[1])
        flawed()
    p.table = good
    # an entry no token needs is not read
    p.table[1, 2] = -5
    D.attention_paged(ctx, p.pages, p.batch([2, 2, 2]), q, out)
    p.pages.check()
    p.table = good
    for length in (-1, 65, 2 ** 31 - 1, -2 ** 31):
        b = p.batch([2, 2, 2], [40, length, 20], max_tokens=64)
        got = [torch.full((2, 6, 64), 77.0, dtype=torch.float16, device="cuda") for _ in range(2)]
        p.pages.read(b, *got)
        flawed()
        assert np.array_equal(got[1].cpu().numpy()[:, 4:], p.v[2][:, -2:]) and bool((got[0][:, 2:4] == 77.0).all())
        p.pages.append(b, *got)
        flawed()
        out.fill_(77.0)
        D.attention_paged(ctx, p.pages, p.batch([2, 2, 2], [40, length, 20], max_tokens=64), q, out)
        flawed()
        others_right([2, 2, 2], 1)
        assert bool((out[:, 2:4] == 0.0).all())
    for offsets in ([0, 2, 1, 6], [0, 2, 7, 6], [-1, 2, 4, 6], [0, 2, 2 ** 31 - 1, 6], [0, 2, -2 ** 31, 6], [0, 4, 5, 6]):
        b = D.PagedBatch(dev(p.table), ints(p.lengths()), ints(offsets), max_rows=3)
        D.attention_paged(ctx, p.pages, b, q, out)
        flawed()
        p.pages.read(b, k.clone(), k.clone())
        flawed()
    p.check_held()


def test_refusals(ctx):
    """Calls the host turns down before anything runs."""
    p = Pool(ctx, 4, 2, 64, 2, page=16, most=64)
    p.fill([20, 20])
    L, bad = F.lib(), F.RK_NPU_ERR_PARAM
    pool, ws = p.pages.handle.raw, ctx.attention_workspace(p.pages)
    table, lengths, offsets = dev(p.table), ints([20, 20]), ints([0, 1, 2])
    q, kv = torch.zeros(4, 2, 64, dtype=torch.float16, device="cuda"), torch.zeros(2, 2, 64, dtype=torch.float16, device="cuda")
    host = torch.zeros(4, 2, 64, dtype=torch.float16)

    def batch(**kw):
        x = dict(sequences=2, rows=2, max_rows=1, max_tokens=64, lengths=lengths.data_ptr(),
                 row_offsets=offsets.data_ptr(), table=table.data_ptr(), table_stride=4)
        x.update(kw)
        return ctypes.byref(F.rk_npu_hip_paged_batch(*(x[n] for n, _ in F.rk_npu_hip_paged_batch._fields_)))

    def heads(t, type=F.RK_NPU_HIP_F16, head=128, row=64, at=0):
        return ctypes.byref(F.rk_npu_hip_heads(t.data_ptr() + at if t is not None else None, type, head, row))

    def all_calls(b, q=heads(q), kv=heads(kv)):
        return (L.rk_npu_hip_attention_paged_run(ws.raw, pool, b, q, heads(out), None),
                L.rk_npu_hip_attention_paged_read(pool, b, kv, heads(kv2), None),
                L.rk_npu_hip_attention_paged_append(pool, b, kv, heads(kv2), None, None, None, None))
    out, kv2 = torch.zeros_like(q), torch.zeros_like(kv)
    assert all_calls(batch()) == (0, 0, 0)
    assert all_calls(batch(row_offsets=None)) == (0, 0, 0)
    for kw in (dict(sequences=0), dict(sequences=-1), dict(sequences=1025), dict(rows=0), dict(rows=-1), dict(rows=2 ** 23 + 1),
               dict(max_rows=0), dict(max_rows=3), dict(max_tokens=0), dict(max_tokens=65), dict(max_tokens=-1),
               dict(table_stride=0), dict(table_stride=3), dict(lengths=None), dict(table=None), dict(rows=1, row_offsets=None),
               dict(rows=2, max_rows=2, row_offsets=None), dict(lengths=lengths.data_ptr() + 2), dict(table=table.data_ptr() + 1),
               dict(lengths=host.data_ptr()), dict(table=host.data_ptr()), dict(row_offsets=host.data_ptr())):
        assert all_calls(batch(**kw)) == (bad,) * 3, kw
    assert (L.rk_npu_hip_attention_paged_run(ws.raw, pool, None, heads(q), heads(out), None),
            L.rk_npu_hip_attention_paged_read(pool, None, heads(kv), heads(kv), None)) == (bad, bad)
    for kw in (dict(type=2), dict(type=-1), dict(head=-1), dict(row=-64), dict(at=1)):
        assert all_calls(batch(), heads(q, **kw), heads(kv, **kw)) == (bad,) * 3, kw
    assert all_calls(batch(), heads(host), heads(host)) == (bad,) * 3
    assert all_calls(batch(), heads(None), heads(None)) == (bad,) * 3
    # outputs whose rows overlap
    for kw in (dict(row=32), dict(head=64, row=64), dict(head=0)):
        assert L.rk_npu_hip_attention_paged_run(ws.raw, pool, batch(), heads(q), heads(out, **kw), None) == bad
        assert L.rk_npu_hip_attention_paged_read(pool, batch(), heads(kv, **kw), None, None) == bad
        assert L.rk_npu_hip_attention_paged_append(pool, batch(), heads(kv), heads(kv2), None, heads(q), heads(out, **kw), None) == bad
    assert L.rk_npu_hip_attention_paged_read(pool, batch(), None, None, None) == bad
    assert L.rk_npu_hip_attention_paged_read(pool, batch(), None, heads(kv), None) == 0
    append = L.rk_npu_hip_attention_paged_append
    assert append(pool, batch(), None, heads(kv), None, None, None, None) == bad
    assert append(pool, batch(), heads(kv), heads(kv2), None, heads(q), None, None) == bad
    assert append(pool, batch(), heads(kv), heads(kv2), None, None, heads(q), None) == bad
    assert append(pool, batch(), heads(kv), heads(kv2), None, heads(q), heads(q), None) == 0
    wide = torch.zeros(4, 2, 128, dtype=torch.float16, device="cuda")
    assert append(pool, batch(), heads(kv), heads(kv2), None, heads(wide), heads(wide, head=256, row=128), None) == bad
    assert append(pool, batch(), heads(kv), heads(kv2), host.data_ptr(), None, None, None) == bad
    assert append(pool, batch(), heads(kv), heads(kv2), lengths.data_ptr() + 2, None, None, None) == bad
    # handles of other kinds and geometries
    other = D.KvPages(ctx, 4, 2, 64, 0.5, 8, page=16)
    assert L.rk_npu_hip_attention_paged_run(ctx.attention_workspace(other).raw, pool, batch(), heads(q), heads(out), None) == bad
    assert L.rk_npu_hip_attention_paged_run(pool, pool, batch(), heads(q), heads(out), None) == bad
    assert L.rk_npu_hip_attention_paged_run(ws.raw, ws.raw, batch(), heads(q), heads(out), None) == bad
    assert L.rk_npu_hip_attention_paged_status(ws.raw) == bad
    p.pages.check()
    for build in (dict(page=48), dict(page=512), dict(page=0), dict(pages=0), dict(pages=-1), dict(rotary_dim=8),
                  dict(rotary_dim=72), dict(rotary_dim=-16), dict(rotary_dim=16, rope_theta=0.0),
                  dict(rotary_dim=16, rope_theta=float("nan")), dict(rotary_dim=16, frequencies=[1.0] * 7),
                  dict(rotary_dim=16, frequencies=[1.0] * 7 + [float("inf")]), dict(capacity=0)):
        with pytest.raises(npu.NpuError):
            D.KvPages(ctx, 4, 2, 64, 0.125, **{**dict(pages=8, page=16), **build})
    with pytest.raises(npu.NpuError):
        D.KvPages(ctx, 4, 2, 96, 0.125, 8)
    with pytest.raises(npu.NpuError):
        D.KvPages(ctx, 4, 2, 64, 0.125, 2 ** 31 - 1, page=256)
    for t in (torch.zeros(2, 4, dtype=torch.int64, device="cuda"), torch.zeros(2, 4, dtype=torch.int32)):
        with pytest.raises(npu.NpuError):
            D.PagedBatch(t, lengths)
    with pytest.raises(npu.NpuError):
        D.PagedBatch(table, ints([1, 2, 3]))
    with pytest.raises(npu.NpuError):
        D.PagedBatch(table, lengths, ints([0, 1]))
    with pytest.raises(npu.NpuError):
        D.attention_paged(ctx, p.pages, D.PagedBatch(table, lengths, max_tokens=65), q, out)
    with pytest.raises(npu.NpuError):
        p.pages.append(D.PagedBatch(table, lengths), kv, kv, q=q)


# --- streams, graphs, a run of them together ----------------------------------------

def test_streams_with_workspaces_of_their_own(ctx):
    p = Pool(ctx, 8, 2, 128, 3, most=2000)
    p.fill([2000, 1500, 3])
    q = dev(p.rows(3, 8))
    b = p.batch([1, 1, 1])
    want = torch.empty((8, 3, 128), device="cuda")
    D.attention_paged(ctx, p.pages, b, q, want)
    torch.cuda.synchronize()
    runs = [(torch.cuda.Stream(), ctx.attention_workspace(p.pages, own=True), torch.empty_like(want)) for _ in range(3)]
    for _ in range(5):
        for s, ws, out in runs:
            with torch.cuda.stream(s):
                D.attention_paged(ctx, p.pages, b, q, out, ws=ws)
    torch.cuda.synchronize()
    p.pages.check()
    for _, _, out in runs:
        assert torch.equal(out, want)


def test_captured_step_follows_the_lengths(ctx):
    """One captured decode step, launched as the sequences grow, against eager calls."""
    p = Pool(ctx, 8, 2, 128, 4, page=16, most=1500, rotary_dim=128)
    n = [1, 700, 30, 0]
    k, v = p.rows(sum(n), 2), p.rows(sum(n), 2)
    p.pages.append(p.batch(n, n), dev(k), dev(v))
    ws = ctx.attention_workspace(p.pages, own=True)
    lengths = ints([x + 1 for x in n])
    b = D.PagedBatch(dev(p.table), lengths, max_tokens=1500)
    new = [torch.zeros(h, 4, 128, device="cuda") for h in (8, 2, 2)]
    turned, out = torch.zeros(8, 4, 128, dtype=torch.float16, device="cuda"), torch.zeros(8, 4, 128, device="cuda")

    def step(batch, turned, out):
        p.pages.append(batch, new[1], new[2], q=new[0], q_out=turned)
        D.attention_paged(ctx, p.pages, batch, turned, out, ws=ws)
    step(b, turned, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(b, turned, out)
    for i in range(40):
        for x in new:
            x.copy_(dev(p.rng.standard_normal(x.shape).astype(np.float32)))
        now = [x + 1 + i for x in n]
        now[2] = 0 if i % 3 == 0 else now[2]      # idle at times
        lengths.copy_(ints(now))
        out.fill_(77.0)
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        want, t2 = torch.full_like(out, 77.0), torch.zeros_like(turned)
        step(D.PagedBatch(dev(p.table), ints(now), max_tokens=1500), t2, want)
        torch.cuda.synchronize()
        assert torch.equal(got, want), f"launch {i}"
        if now[2] == 0:
            assert bool((got[:, 2] == 0.0).all())
    p.pages.check()


def test_every_launch_of_a_graph_is_told_of(ctx):
    """check() waits for each launch of a captured call, on a stream of its own, and not only for the first."""
    p = Pool(ctx, 4, 2, 64, 2, page=16, most=64, spare=1)
    p.fill([20, 20])
    table = dev(p.table)
    b = D.PagedBatch(table, ints([20, 20]))
    q, k, v = dev(p.rows(2, 4)), dev(p.rows(2, 2)), dev(p.rows(2, 2))
    out, ws = torch.empty_like(q), ctx.attention_workspace(p.pages, own=True)

    def step():
        p.pages.append(b, k, v)
        D.attention_paged(ctx, p.pages, b, q, out, ws=ws)
    step()
    p.pages.check()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        step()
    p.pages.check()
    for wrong in (True, False, True, True, False):
        table[1, 1] = -1 if wrong else int(p.table[1, 1])
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)     # (the launch waits here while check() is called)
            graph.replay()
        if wrong:
            with pytest.raises(npu.NpuError):
                p.pages.check()
        p.pages.check()
        assert side.query()


def test_prompt_then_decode(ctx):
    """Prompts in ragged pieces, then drafts, then single tokens, rotated on the way:
    attention over what the pages hold, and what they hold over the whole run."""
    p = Pool(ctx, 8, 2, 128, 3, page=32, most=400, rotary_dim=64, rope_theta=1e6)
    freq = M.frequencies(64, 1e6)
    keys = [np.zeros((2, 0, 128)) for _ in range(3)]
    for rows in ([100, 7, 250], [60, 0, 1], [3, 3, 3], [1, 1, 1], [1, 1, 1], [1, 0, 1]):
        before, total = p.lengths(), sum(rows)
        q, k, v = p.rows(total, 8, np.float32), p.rows(total, 2, np.float32), p.rows(total, 2, np.float32)
        now = [a + n for a, n in zip(before, rows)]
        b = p.batch(rows, now)
        turned = torch.empty(8, total, 128, dtype=torch.float16, device="cuda")
        p.pages.append(b, dev(k), dev(v), q=dev(q), q_out=turned)
        held = [torch.empty(2, total, 128, dtype=torch.float16, device="cuda") for _ in range(2)]
        p.pages.read(b, *held)
        out = torch.full((8, total, 128), 77.0, device="cuda")
        D.attention_paged(ctx, p.pages, b, turned, out)
        p.pages.check()
        at = 0
        for s, n in enumerate(rows):
            mine = slice(at, at + n)
            at += n
            p.k[s] = np.concatenate([p.k[s], held[0].cpu().numpy()[:, mine]], axis=1)
            p.v[s] = np.concatenate([p.v[s], held[1].cpu().numpy()[:, mine]], axis=1)
            want = M.rotate(k[:, mine], np.arange(before[s], now[s]), freq, False)
            assert np.all(np.abs(p.k[s][:, before[s]:] - want) <= M.rotate_bound(k[:, mine], want, True))
        p.compare(rows, now, turned.cpu().numpy(), out)
    p.check_held()
