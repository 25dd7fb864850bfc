"""The 8-bit KV cache's C calls where no GPU is needed: the configuration's
defaults, the sizes, and what is refused before anything runs."""
import ctypes

import pytest

from open_rknpu2_lm_infer_amd import _ffi as F
from open_rknpu2_lm_infer_amd import npu


def config(qh=8, kh=2, d=128, fmt=F.RK_NPU_HIP_KV_I8, block=32):
    cfg = F.rk_npu_hip_attention_q8_config()
    F.lib().rk_npu_hip_attention_q8_config_init(ctypes.byref(cfg))
    a = cfg.attention
    a.query_heads, a.kv_heads, a.head_dim, a.softmax_scale = qh, kh, d, 0.125
    a.max_query_rows, a.max_capacity, a.initial_capacity = 16, 1000, 100
    cfg.format, cfg.block = fmt, block
    return cfg


def query(cfg, capacity=1000, rows=1):
    sizes = F.rk_npu_attention_f16_sizes()
    return F.lib().rk_npu_hip_attention_q8_query(ctypes.byref(cfg), capacity, rows, ctypes.byref(sizes)), sizes


def test_defaults():
    cfg, plain = F.rk_npu_hip_attention_q8_config(), F.rk_npu_attention_f16_config()
    F.lib().rk_npu_hip_attention_q8_config_init(ctypes.byref(cfg))
    F.lib().rk_npu_attention_f16_config_init(ctypes.byref(plain))
    assert bytes(cfg.attention) == bytes(plain)
    assert (cfg.format, cfg.block) == (F.RK_NPU_HIP_KV_I8, 32)
    F.lib().rk_npu_hip_attention_q8_config_init(None)


@pytest.mark.parametrize("block", [32, 64, 128])
def test_sizes(block):
    """Codes of whole blocks, 16 bytes of scales a block and head for K and V
    together, three fp16 blocks of each; the workspace is the fp16 family's."""
    for capacity in (0, 1, block, 1000):
        rc, s = query(config(block=block), capacity, 4)
        assert rc == F.RK_NPU_OK
        rows = -(-capacity // block) * block
        assert s.key_bytes == s.value_bytes == 2 * rows * 128 + 2 * (rows // block) * 8
        assert s.tail_bytes == 2 * 3 * 2 * block * 128 * 2
        plain = F.rk_npu_attention_f16_sizes()
        cfg = config(block=block)
        assert F.lib().rk_npu_attention_f16_query(ctypes.byref(cfg.attention), 0, 4, 0, ctypes.byref(plain)) == 0
        assert s.workspace_bytes == plain.workspace_bytes


def test_refused_configurations():
    assert query(config())[0] == F.RK_NPU_OK
    for fmt in (-1, 2):
        assert query(config(fmt=fmt))[0] == F.RK_NPU_ERR_PARAM
    for block in (0, -32, 16, 48, 256):
        assert query(config(block=block))[0] == F.RK_NPU_ERR_PARAM
    for bad in (dict(kh=0), dict(qh=7), dict(qh=1), dict(d=0), dict(d=40), dict(d=288), dict(kh=33, qh=33)):
        assert query(config(**bad))[0] == F.RK_NPU_ERR_PARAM
    for capacity in (-1, 2 ** 31 - 200):
        assert query(config(), capacity)[0] == F.RK_NPU_ERR_PARAM
    cfg = config()
    cfg.attention.max_capacity = 2 ** 31 - 100
    assert query(cfg)[0] == F.RK_NPU_ERR_PARAM
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        cfg = config()
        cfg.attention.softmax_scale = scale
        assert query(cfg)[0] == F.RK_NPU_ERR_PARAM
    assert F.lib().rk_npu_hip_attention_q8_query(ctypes.byref(config()), 1, 1, None) == F.RK_NPU_ERR_PARAM
    assert F.lib().rk_npu_hip_attention_q8_query(None, 1, 1, ctypes.byref(F.rk_npu_attention_f16_sizes())) \
        == F.RK_NPU_ERR_PARAM


def test_null_handles():
    """Every call on no cache, and on memory that is no cache."""
    L, cfg = F.lib(), config()
    raw = ctypes.c_void_p(1)
    assert L.rk_npu_hip_attention_q8_cache_create(None, ctypes.byref(cfg), ctypes.byref(raw)) == F.RK_NPU_ERR_PARAM
    assert raw.value is None
    other = (ctypes.c_uint64 * 64)()
    ctx = ctypes.addressof(other)
    heads = F.rk_npu_hip_heads(ctypes.addressof(other), F.RK_NPU_HIP_F16, 128, 128)
    h = ctypes.byref(heads)
    info = F.rk_npu_attention_f16_cache_info()
    for cache in (None, ctypes.addressof(other)):
        for rc in (L.rk_npu_hip_attention_q8_cache_reserve(ctx, cache, 10),
                   L.rk_npu_hip_attention_q8_cache_truncate(cache, 0),
                   L.rk_npu_hip_attention_q8_cache_get_info(cache, ctypes.byref(info)),
                   L.rk_npu_hip_attention_q8_cache_load(ctx, cache, None, None, 0),
                   L.rk_npu_hip_attention_q8_cache_append(ctx, cache, ctx, ctx, 1),
                   L.rk_npu_hip_attention_q8_cache_read(ctx, cache, 0, 1, ctx, ctx),
                   L.rk_npu_hip_attention_q8_run(ctx, None, cache, ctx, 1, 0, ctx, None),
                   L.rk_npu_hip_attention_q8_run_half(ctx, None, cache, ctx, 1, 0, ctx, None),
                   L.rk_npu_hip_attention_q8_device_append(cache, h, h, 1, None),
                   L.rk_npu_hip_attention_q8_device_read(cache, 0, 1, h, h, None),
                   L.rk_npu_hip_attention_q8_device_run(None, cache, h, 1, 0, h, None)):
            assert rc == F.RK_NPU_ERR_PARAM
        L.rk_npu_hip_attention_q8_cache_free(cache)


def test_cache_bytes_of_a_backend():
    opts = npu.ModelOptions(chunk=64, context=1000)
    plain = npu.Backend.attention_cache_bytes(opts, 16, 4, 64, 0.125)
    for fmt in ("i8", "e4m3"):
        small = npu.Backend.attention_cache_bytes(opts, 16, 4, 64, 0.125, (fmt, 32))
        assert small == 2 * (4 * 1024 * 64 + 4 * 32 * 8) + 2 * 3 * 4 * 32 * 64 * 2
        assert small < 0.6 * plain
    for bad in (("i4", 32), ("i8", 33)):
        with pytest.raises(npu.NpuError):
            npu.Backend.attention_cache_bytes(opts, 16, 4, 64, 0.125, bad)
