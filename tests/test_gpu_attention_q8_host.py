"""The 8-bit KV cache's host-buffer calls, a run of its operators together as a
decode loop uses them, and its use from several threads, streams and graphs;
against tests/kv_model.py."""
import ctypes
import threading

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


def say(*words):
    print(*words, flush=True)


class HostPair:
    """A cache behind Backend.attention_q8 and its model."""

    def __init__(self, qh, kh, d, fmt="i8", block=32, context=4096, chunk=128, noncausal=False, seed=0, backend=None):
        say(f"qh={qh} kh={kh} d={d} {fmt} block={block} noncausal={noncausal} seed={seed}")
        self.be = backend or npu.Backend(npu.ModelOptions(chunk=chunk, context=context))
        self.scale = float(np.float32(d ** -0.5))
        self.qh, self.kh, self.d, self.noncausal, self.i8 = qh, kh, d, noncausal, fmt == "i8"
        self.att = self.be.attention_q8(qh, kh, d, d ** -0.5, fmt, block, noncausal)
        self.k, self.v = (kv_model.KvModel(kh, d, fmt, block) for _ in range(2))
        self.rng = np.random.default_rng(seed)

    def rows(self, n):
        return [self.rng.standard_normal((n, self.kh, self.d)).astype(np.float32) for _ in range(2)]

    def took(self, k, v):
        for m, x in ((self.k, k), (self.v, v)):
            m.append(x.transpose(1, 0, 2).astype(np.float16))

    def put(self, n, call=None):
        """rows through the C call itself: any number at once."""
        k, v = self.rows(n)
        self.took(k, v)
        bits = [np.ascontiguousarray(x.transpose(1, 0, 2).astype(np.float16)) for x in (k, v)]
        call = call or F.lib().rk_npu_hip_attention_q8_cache_append
        npu.check(call(self.be.ctx, self.att.cache.raw, bits[0].ctypes.data, bits[1].ctypes.data, n), "append")

    def truncate(self, n):
        self.att.truncate(n)
        self.k.truncate(n)
        self.v.truncate(n)

    def check_contents(self, first=0, n=None):
        n = self.k.length - first if n is None else n
        got = self.att.read(first, n)
        for name, g, m in zip("kv", got, (self.k, self.v)):
            want = m.values()[:, first:first + n].astype(np.float16).transpose(1, 0, 2)
            assert np.array_equal(g, want, equal_nan=True), f"{name} differs"
        assert self.att.info().length == self.k.length

    def close(self, q, out, position, f16=False):
        """q, out [qh][rows][d]."""
        k, v = self.k.values(), self.v.values()
        want = kv_model.attention(q, k, v, self.scale, position, not self.noncausal)
        most = kv_model.bound(q, k, v, self.scale, f16, self.i8) * np.abs(v).max()
        assert np.abs(out.astype(np.float64) - want).max() <= most


@pytest.mark.parametrize("flag", [0, 1])
@pytest.mark.parametrize("fmt,block,d", [("i8", 32, 64), ("e4m3", 128, 128), ("i8", 64, 256)])
def test_load_append_read_and_growth(flag, fmt, block, d):
    """Loads, appends past the capacity (which grows), pieces read back; with and
    without the call's completion word."""
    with D.plan_switch("HM_HOST_FLAG", flag):
        p = HostPair(4, 2, d, fmt, block, context=2000, seed=d)
        assert p.att.info().capacity == 128
        for n in (1, 40, 87, 1, 300, 129):
            p.put(n)
            p.check_contents()
        assert p.att.info().capacity >= p.k.length
        p.check_contents(3, 1)
        p.check_contents(block - 1, 70)
        before = p.att.info().generation
        p.k, p.v = (kv_model.KvModel(2, d, fmt, block) for _ in range(2))
        p.put(75, F.lib().rk_npu_hip_attention_q8_cache_load)
        p.check_contents()
        assert p.att.info().generation > before
        p.att.reset()
        assert p.att.info().length == 0
        p.k, p.v = (kv_model.KvModel(2, d, fmt, block) for _ in range(2))
        p.put(2000)
        p.check_contents()
        most = p.att.info().max_capacity - 2000
        x = np.zeros((2, most + 1, d), np.float16)
        assert F.lib().rk_npu_hip_attention_q8_cache_append(p.be.ctx, p.att.cache.raw, x.ctypes.data, x.ctypes.data,
                                                            most + 1) == F.RK_NPU_ERR_PARAM
        p.check_contents(1900, 100)


@pytest.mark.parametrize("held", [0, 10, 64, 77])
def test_long_host_appends_can_be_taken_back(held):
    """Rows for several pieces of the staging memory: the call's start is still exact."""
    p = HostPair(8, 8, 256, "i8", 64, context=8192, seed=held)
    if held:
        p.put(held)
    for n in (1100, 2600, 1025):  # (a piece is 1024 rows here)
        p.put(n)
        p.check_contents(held + n - 70, 70)
        for back in (held + n - 3, held + 2, held):
            p.truncate(back)
            if back:
                p.check_contents(max(0, back - 70), min(back, 70))
    p.put(5)
    p.check_contents()


@pytest.mark.parametrize("d,fmt,noncausal", [(64, "e4m3", False), (128, "i8", True), (256, "i8", False)])
def test_run_and_run_half(d, fmt, noncausal):
    """Both output types of the C calls, with and without timings, few rows and
    many; what is refused."""
    p = HostPair(8, 2, d, fmt, 32, noncausal=noncausal, seed=d)
    p.put(777)
    L, ws = F.lib(), p.be._attention.workspace
    for rows in (1, 9, 128):
        for half in (False, True):
            say(f"  rows={rows} half={half}")
            q = p.rng.standard_normal((8, rows, d)).astype(np.float16)
            run = L.rk_npu_hip_attention_q8_run_half if half else L.rk_npu_hip_attention_q8_run
            outs = []
            for timings in (None, F.rk_npu_attention_f16_timings()):
                outs.append(np.empty((8, rows, d), np.float16 if half else np.float32))
                npu.check(run(p.be.ctx, ws.raw, p.att.cache.raw, q.ctypes.data, rows, 777 - rows, outs[-1].ctypes.data,
                              ctypes.byref(timings) if timings else None), "run")
            assert timings.total_us > 0 and timings.device_us > 0
            assert np.array_equal(outs[0], outs[1])
            p.close(q, outs[0], 777 - rows, half)
    args = (p.be.ctx, ws.raw, p.att.cache.raw, q.ctypes.data)
    out = outs[0].ctypes.data
    for bad in ((args[0], None) + args[2:] + (1, 0, out), args[:2] + (None, args[3], 1, 0, out),
                args[:3] + (None, 1, 0, out), args + (1, 0, None), args + (0, 0, out), args + (129, 0, out),
                args + (1, -1, out), (None,) + args[1:] + (1, 0, out)):
        assert run(*bad, None) == F.RK_NPU_ERR_PARAM
    if not noncausal:
        assert run(*args, 2, 776, out, None) == F.RK_NPU_ERR_PARAM
    p.att.reset()
    assert run(*args, 1, 0, out, None) == F.RK_NPU_ERR_PARAM


@pytest.mark.parametrize("fmt,block", [("i8", 32), ("e4m3", 64)])
def test_decode_loop_of_the_host_calls(fmt, block):
    """A prompt in chunks, then steps, drafts that are partly rejected, a session
    cut back and continued: Attention's own calls over the 8-bit cache."""
    p = HostPair(8, 2, 64, fmt, block, context=1024, seed=5)
    position = 0
    for rows, keep in ((100, 100), (128, 128), (33, 33), (1, 1), (1, 1), (6, 2), (6, 6), (1, 1), (40, 3), (1, 1)):
        say(f"  rows={rows} position={position}")
        q = p.rng.standard_normal((rows, 8, 64)).astype(np.float32)
        k, v = p.rows(rows)
        out = np.empty((rows, 8, 64), np.float32)
        p.att.run(q, k, v, out, rows, position)
        p.took(k, v)
        p.close(q.transpose(1, 0, 2).astype(np.float16), out.transpose(1, 0, 2), position)
        position += keep
        if keep < rows:
            p.truncate(position)
    p.truncate(21)  # (deeper than the rows kept)
    k, v = p.rows(30)
    p.att.append(k, v, 30, 21)
    p.took(k, v)
    p.check_contents()
    with pytest.raises(npu.NpuError):
        p.att.append(k, v, 30, 21)
    small = npu.Backend.attention_cache_bytes(p.be.options, 8, 2, 64, 0.125, (fmt, block))
    assert small < 0.7 * npu.Backend.attention_cache_bytes(p.be.options, 8, 2, 64, 0.125)
    assert p.att.bytes() <= small


def test_shares_the_backend_workspace():
    """fp16 and 8-bit caches of one geometry on one backend; another geometry or
    mask is refused, as Backend.attention does."""
    be = npu.Backend(npu.ModelOptions(chunk=32, context=256))
    f16 = be.attention(4, 2, 64, 0.125)
    p = HostPair(4, 2, 64, context=256, chunk=32, backend=be)
    q = p.rng.standard_normal((20, 4, 64)).astype(np.float32)
    k, v = p.rows(20)
    outs = [np.empty((20, 4, 64), np.float32) for _ in range(2)]
    f16.run(q, k, v, outs[0], 20, 0)
    p.att.run(q, k, v, outs[1], 20, 0)
    p.took(k, v)
    p.close(q.transpose(1, 0, 2).astype(np.float16), outs[1].transpose(1, 0, 2), 0)
    assert np.abs(outs[0] - outs[1]).max() < 1e-2  # (20 rows: the open block, fp16 in both)
    for args in ((8, 2, 64, 0.125), (4, 2, 128, 0.125), (4, 2, 64, 0.25), (4, 2, 64, 0.125, "i8", 32, True)):
        with pytest.raises(npu.NpuError):
            be.attention_q8(*args)
    for args in ((4, 2, 64, 0.125, "i4"), (4, 2, 64, 0.125, "i8", 48)):
        with pytest.raises(npu.NpuError):
            be.attention_q8(*args)


def test_two_threads_on_one_cache():
    """Runs on a workspace of each thread while a third appends and cuts back rows
    behind theirs: results as alone."""
    p = HostPair(4, 2, 64, "i8", 32, context=1024, seed=12)
    p.put(331)
    L = F.lib()
    spaces = []
    for _ in range(2):
        raw = ctypes.c_void_p()
        npu.check(L.rk_npu_attention_f16_prepare(p.be.domain, ctypes.byref(p.be._attention.config), ctypes.byref(raw)),
                  "prepare")
        spaces.append(raw)
    q = p.rng.standard_normal((4, 16, 64)).astype(np.float16)
    outs, codes = [np.empty((4, 16, 64), np.float32) for _ in range(2)], []

    def runs(i):
        for _ in range(50):
            outs[i].fill(3.0)
            codes.append(L.rk_npu_hip_attention_q8_run(p.be.ctx, spaces[i], p.att.cache.raw, q.ctypes.data, 16, 300,
                                                       outs[i].ctypes.data, None))

    k, v = p.rows(90)
    bits = [np.ascontiguousarray(x.transpose(1, 0, 2).astype(np.float16)) for x in (k, v)]

    def appends():
        for _ in range(30):
            codes.append(L.rk_npu_hip_attention_q8_cache_append(p.be.ctx, p.att.cache.raw, bits[0].ctypes.data,
                                                                bits[1].ctypes.data, 90))
            codes.append(L.rk_npu_hip_attention_q8_cache_truncate(p.att.cache.raw, 331))

    threads = [threading.Thread(target=runs, args=(i,)) for i in range(2)] + [threading.Thread(target=appends)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert set(codes) == {F.RK_NPU_OK}
    for o in outs:
        p.close(q, o, 300)
    p.check_contents()
    for raw in spaces:
        L.rk_npu_attention_f16_workspace_free(raw)


# --- device calls ---------------------------------------------------------------

def test_device_and_host_calls_share_a_cache(ctx):
    """Host calls wait for device calls made before them, on the null stream and on
    another."""
    say("qh=4 kh=2 d=64")
    cache = D.KvCacheQ8(ctx, 4, 2, 64, 0.125, 512)
    models = [kv_model.KvModel(2, 64, "i8", 32) for _ in range(2)]
    rng = np.random.default_rng(3)
    L, side = F.lib(), torch.cuda.Stream()
    for i in range(4):
        rows = [rng.standard_normal((2, 45, 64)).astype(np.float16) for _ in range(2)]
        k, v = (torch.from_numpy(x).cuda() for x in rows)
        torch.cuda.synchronize()
        with torch.cuda.stream(side if i % 2 else torch.cuda.default_stream()):
            cache.append(k, v)
        for m, x in zip(models, rows):
            m.append(x)
        n = cache.length
        got = [np.empty((2, n, 64), np.float16) for _ in range(2)]
        npu.check(L.rk_npu_hip_attention_q8_cache_read(ctx.shared.ctx.raw, cache.handle.raw, 0, n, got[0].ctypes.data,
                                                       got[1].ctypes.data), "read")
        for m, g in zip(models, got):
            assert np.array_equal(m.values().astype(np.float16), g)


def test_two_graphs_and_two_streams(ctx):
    """Decode graphs of two caches of one geometry, each on a workspace of its own,
    launched side by side; and a capture that is refused."""
    scale, qh, kh, d = 0.125, 8, 2, 64
    rng = np.random.default_rng(8)
    caches, models, outs, graphs, qs = [], [], [], [], []
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(2):
        say(f"cache {i}")
        cache = D.KvCacheQ8(ctx, qh, kh, d, scale, 4096)
        rows = [rng.standard_normal((kh, 3000 + i, d)).astype(np.float16) for _ in range(2)]
        cache.append(*(torch.from_numpy(x).cuda() for x in rows))
        model = [kv_model.KvModel(kh, d, "i8", 32) for _ in range(2)]
        for m, x in zip(model, rows):
            m.append(x)
        ws = ctx.attention_workspace(cache, own=True)
        q = rng.standard_normal((qh, 4, d)).astype(np.float16)
        qt = torch.from_numpy(q).cuda()
        out = torch.zeros(qh, 4, d, device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[i]):
            for _ in range(5):
                D.attention_q8(ctx, cache, qt, out, 2990, ws=ws)
        caches.append((cache, ws, qt))
        models.append(model)
        outs.append(out)
        graphs.append(graph)
        qs.append(q)
    assert caches[0][1] is not caches[1][1] and ctx.attention_workspace(caches[0][0]) is not caches[0][1]
    for _ in range(4):
        for o in outs:
            o.fill_(2.0)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, q, (mk, mv) in zip(outs, qs, models):
            want = kv_model.attention(q, mk.values(), mv.values(), scale, 2990, True)
            most = kv_model.bound(q, mk.values(), mv.values(), scale, False) * np.abs(mv.values()).max()
            assert np.abs(o.cpu().numpy().astype(np.float64) - want).max() <= most
    cache = caches[0][0]
    cache.truncate(100)
    k = torch.zeros(kh, 1, d, device="cuda", dtype=torch.float16)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=s):
        k.add_(1.0)
        with pytest.raises(npu.NpuError):
            cache.append(k, k)
    assert cache.length == 100
    cache.append(k, k)
    assert cache.length == 101


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_offsets_past_32_bits(ctx, fmt):
    """A cache of more than 4 GiB of codes each of K and V, rows read into an array
    of more than 2^32 elements; the last head's last rows."""
    kh, d, n, block = 32, 256, 525000, 128
    say(f"kh={kh} d={d} rows={n} {fmt}")
    cache = D.KvCacheQ8(ctx, kh, kh, d, d ** -0.5, n, fmt=fmt, block=block, max_query_rows=16)
    x = torch.randn(kh, n, d, device="cuda", dtype=torch.float16)
    cache.append(x, x)
    tail0 = n // block * block
    model = kv_model.KvModel(kh, d, fmt, block)
    model.append(x[:, tail0 - 2 * block:].cpu().numpy())
    back = torch.empty_like(x)
    cache.read(0, back, x)  # (V back over the rows themselves)
    torch.cuda.synchronize()
    assert torch.equal(back, x)
    assert np.array_equal(x[:, tail0 - 2 * block:].cpu().numpy(), model.values().astype(np.float16))
    del back
    q = torch.randn(kh, 16, d, device="cuda", dtype=torch.float16)
    out = torch.empty(kh, 16, d, device="cuda")
    D.attention_q8(ctx, cache, q, out, n - 16)
    # heads 0 and the last, against 64 bits of what was read
    for g in (0, kh - 1):
        held = x[g].double()
        for r in (0, 15):
            seen = held[:n - 15 + r]
            p = torch.softmax((seen * q[g, r].double()).sum(1) * d ** -0.5, 0)
            want = (p[:, None] * seen).sum(0)
            # (the rows read are values rounded to fp16: half a step of each of K and V)
            s = float((seen.abs() * q[g, r].double().abs()).sum(1).max()) * d ** -0.5
            most = (2 * s + 2) * 2.0 ** -11 * float(seen.abs().max())
            assert float((out[g, r].double() - want).abs().max()) <= most
