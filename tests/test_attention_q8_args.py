"""The 8-bit KV cache's Python calls pass 32-bit numbers to the library: ones that
do not fit are refused, not cut to their low bits. No GPU: the library is a stub."""
import types

import pytest
import torch

from open_rknpu2_lm_infer_amd import _ffi as F
from open_rknpu2_lm_infer_amd import attention as A
from open_rknpu2_lm_infer_amd import device as D
from open_rknpu2_lm_infer_amd import npu

BIG = [2 ** 31, 2 ** 32, 2 ** 32 + 5, -2 ** 31 - 1, -2 ** 32]


class Stub:
    """Every call is noted and succeeds."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            return 0
        return call


@pytest.fixture
def stub(monkeypatch):
    s = Stub()
    monkeypatch.setattr(F, "lib", lambda: s)
    return s


def device_cache():
    c = object.__new__(D.KvCacheQ8)
    c.handle = types.SimpleNamespace(raw=64)
    c.ctx = types.SimpleNamespace(shared=types.SimpleNamespace(ctx=types.SimpleNamespace(raw=64)))
    c._kv = c._query = (1, 64)
    return c


class Rows:
    """A cuda tensor's attributes, [1][rows][64] fp16."""

    def __init__(self, rows):
        self.shape, self.is_cuda, self.dtype = (1, rows, 64), True, torch.float16

    def stride(self):
        return (0, 0, 1)

    def data_ptr(self):
        return 64


@pytest.mark.parametrize("n", BIG)
def test_device_calls(stub, n):
    c, r = device_cache(), Rows(1)
    ws = types.SimpleNamespace(raw=64)
    for call in (lambda: c.truncate(n), lambda: c.reserve(n), lambda: c.read(n, r, r, stream=0),
                 lambda: D.attention_q8(None, c, r, r, n, ws=ws, stream=0)):
        with pytest.raises(npu.NpuError):
            call()
    if n > 0:
        many = Rows(n)
        for call in (lambda: c.append(many, many, stream=0), lambda: c.read(0, many, many, stream=0),
                     lambda: D.attention_q8(None, c, many, many, 0, ws=ws, stream=0)):
            with pytest.raises(npu.NpuError):
                call()
    assert stub.calls == []
    c.truncate(5)
    c.reserve(2 ** 31 - 1)
    c.read(3, r, r, stream=0)
    D.attention_q8(None, c, r, r, 0, ws=ws, stream=0)
    assert len(stub.calls) == 4


@pytest.mark.parametrize("n", BIG)
@pytest.mark.parametrize("name", ["query_heads", "kv_heads", "head_dim", "capacity", "max_query_rows",
                                  "initial_capacity", "block"])
def test_device_cache_sizes(name, n):
    sizes = dict(query_heads=2, kv_heads=1, head_dim=64, softmax_scale=0.125, capacity=64)
    with pytest.raises(npu.NpuError, match=name):
        D.KvCacheQ8(None, **{**sizes, name: n})


@pytest.mark.parametrize("n", BIG)
def test_host_calls(stub, n):
    a = object.__new__(A.AttentionQ8)
    a.cache = types.SimpleNamespace(raw=64)
    a.backend = types.SimpleNamespace(ctx=64, options=types.SimpleNamespace(context=2 ** 40))
    a.kv_heads, a.dimension, a._lock = 1, 64, __import__("threading").Lock()
    for call in (lambda: a.truncate(n), lambda: a.reserve(n), lambda: a.read(n, 1)):
        with pytest.raises(npu.NpuError):
            call()
    assert stub.calls == []
    a.truncate(5)
    a.reserve(64)
    a.read(0, 1)
    assert len(stub.calls) == 3
    with pytest.raises(npu.NpuError):
        A.q8_config(F.rk_npu_attention_f16_config(), "i8", 2 ** 32 + 32)
