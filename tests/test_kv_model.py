"""The 8-bit KV cache without a GPU: its oracle against independent statements,
and the calls that need no device."""
import ctypes

import numpy as np
import pytest
import torch

from open_rknpu2_lm_infer_amd import _ffi as F
from tests import kv_model


def test_e4m3_rounding_is_the_formats():
    """Every finite e4m3 value is kept; values between two neighbours go to the
    nearer one, halfway to the even code; torch's conversion agrees."""
    codes = torch.arange(0, 0x7F, dtype=torch.uint8)
    grid = codes.view(torch.float8_e4m3fn).double().numpy()
    assert grid[-1] == 448.0 and np.array_equal(kv_model.e4m3_round(grid), grid)
    mid = (grid[1:] + grid[:-1]) / 2
    even = np.where(np.arange(len(mid)) % 2 == 0, grid[:-1], grid[1:])
    assert np.array_equal(kv_model.e4m3_round(mid), even)
    assert np.array_equal(kv_model.e4m3_round(mid * (1 + 1e-9)), grid[1:])
    assert np.array_equal(kv_model.e4m3_round(-mid * (1 - 1e-9)), -grid[:-1])
    x = np.random.default_rng(1).uniform(-448, 448, 20000).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(kv_model.e4m3_round(x.astype(np.float64)), want)


@pytest.mark.parametrize("fmt,step", [("i8", 0.5), ("e4m3", 16.0)])
def test_quantisation_error_is_half_a_step(fmt, step):
    x = np.random.default_rng(2).standard_normal((3, 32, 64)).astype(np.float16)
    x[1] = 0
    x[2, 5, 7] = np.inf
    codes, scales = kv_model.quantise(x, fmt)
    assert np.abs(codes[0]).max() == kv_model.TOP[fmt] and scales[0] > 0
    # (the widest step lies at the top: 1 of 127, 32 of 448)
    assert np.abs(codes[0] * scales[0] - x[0]).max() <= step * scales[0] * (1 + 1e-6)
    got = kv_model.values((codes, scales))
    assert not got[1].any() and np.isnan(got[2]).all()


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_contents_do_not_depend_on_the_calls(fmt):
    """One append, row by row, and with drafts appended and taken back."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((2, 200, 64)).astype(np.float16)
    whole = kv_model.KvModel(2, 64, fmt, 32)
    whole.append(x)
    for draft in (0, 1, 7, 40, 100):
        m = kv_model.KvModel(2, 64, fmt, 32)
        for i in range(200):
            if draft and i % 13 == 0:
                m.append(rng.standard_normal((2, draft, 64)))
                m.truncate(i)
            m.append(x[:, i:i + 1])
        assert np.array_equal(m.values(), whole.values())


def _config(**kw):
    cfg = F.rk_npu_hip_attention_q8_config()
    F.lib().rk_npu_hip_attention_q8_config_init(ctypes.byref(cfg))
    for name, value in kw.items():
        setattr(cfg if name in ("format", "block") else cfg.attention, name, value)
    return cfg


def test_query_counts_codes_scales_and_fp16_rows():
    L = F.lib()
    cfg, sizes = _config(), F.rk_npu_attention_f16_sizes()
    assert (cfg.format, cfg.block, cfg.attention.head_dim) == (F.RK_NPU_HIP_KV_I8, 32, 128)
    assert L.rk_npu_hip_attention_q8_query(ctypes.byref(cfg), 4097, 1, ctypes.byref(sizes)) == 0
    assert sizes.key_bytes == sizes.value_bytes == 8 * (4128 * 128 + 129 * 8)
    assert sizes.tail_bytes == 2 * 3 * 8 * 32 * 128 * 2
    f16 = F.rk_npu_attention_f16_sizes()
    assert L.rk_npu_attention_f16_query(ctypes.byref(cfg.attention), 4128, 1, 4128, ctypes.byref(f16)) == 0
    assert sizes.key_bytes < 0.51 * f16.key_bytes and sizes.workspace_bytes == f16.workspace_bytes


@pytest.mark.parametrize("bad", [dict(format=2), dict(format=-1), dict(block=0), dict(block=16), dict(block=48),
                                 dict(block=256), dict(kv_heads=0), dict(query_heads=12), dict(head_dim=33),
                                 dict(softmax_scale=0.0), dict(softmax_scale=float("nan")), dict(max_query_rows=257),
                                 dict(max_capacity=2 ** 31 - 1), dict(initial_capacity=8192), dict(mask_mode=2)])
def test_bad_configs_are_refused(bad):
    L = F.lib()
    cfg, sizes, out = _config(**bad), F.rk_npu_attention_f16_sizes(), ctypes.c_void_p(1)
    assert L.rk_npu_hip_attention_q8_query(ctypes.byref(cfg), 64, 1, ctypes.byref(sizes)) == F.RK_NPU_ERR_PARAM
    assert L.rk_npu_hip_attention_q8_cache_create(None, ctypes.byref(cfg), ctypes.byref(out)) == F.RK_NPU_ERR_PARAM
    assert not out.value


def test_null_handles_are_refused():
    L = F.lib()
    h = F.rk_npu_hip_heads(64, F.RK_NPU_HIP_F16, 128, 128)
    p = ctypes.byref(h)
    sizes = F.rk_npu_attention_f16_sizes()
    cfg = _config()
    assert L.rk_npu_hip_attention_q8_query(None, 64, 1, ctypes.byref(sizes)) == F.RK_NPU_ERR_PARAM
    assert L.rk_npu_hip_attention_q8_query(ctypes.byref(cfg), -1, 1, ctypes.byref(sizes)) == F.RK_NPU_ERR_PARAM
    assert L.rk_npu_hip_attention_q8_query(ctypes.byref(cfg), 64, 0, ctypes.byref(sizes)) == F.RK_NPU_ERR_PARAM
    assert L.rk_npu_hip_attention_q8_device_append(None, p, p, 1, None) == F.RK_NPU_ERR_PARAM
    assert L.rk_npu_hip_attention_q8_device_read(None, 0, 1, p, p, None) == F.RK_NPU_ERR_PARAM
    assert L.rk_npu_hip_attention_q8_device_run(None, None, p, 1, 0, p, None) == F.RK_NPU_ERR_PARAM
    assert L.rk_npu_hip_attention_q8_cache_load(None, None, None, None, 0) == F.RK_NPU_ERR_PARAM
    assert L.rk_npu_hip_attention_q8_cache_append(None, None, None, None, 1) == F.RK_NPU_ERR_PARAM
    assert L.rk_npu_hip_attention_q8_cache_read(None, None, 0, 1, None, None) == F.RK_NPU_ERR_PARAM
    assert L.rk_npu_hip_attention_q8_cache_reserve(None, None, 1) == F.RK_NPU_ERR_PARAM
    assert L.rk_npu_hip_attention_q8_cache_truncate(None, 0) == F.RK_NPU_ERR_PARAM
    assert L.rk_npu_hip_attention_q8_cache_get_info(None, None) == F.RK_NPU_ERR_PARAM
    assert L.rk_npu_hip_attention_q8_run(None, None, None, None, 1, 0, None, None) == F.RK_NPU_ERR_PARAM
    assert L.rk_npu_hip_attention_q8_run_half(None, None, None, None, 1, 0, None, None) == F.RK_NPU_ERR_PARAM
    L.rk_npu_hip_attention_q8_cache_free(None)
    L.rk_npu_hip_attention_q8_config_init(None)
