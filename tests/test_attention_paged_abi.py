"""The paged KV cache's C calls where no GPU is needed: the configuration's defaults,
the sizes, and what is refused before anything runs."""
import ctypes

import pytest
import torch

from open_rknpu2_lm_infer_amd import _ffi as F
from open_rknpu2_lm_infer_amd import device as D
from open_rknpu2_lm_infer_amd import npu


def config(qh=8, kh=2, d=128, page=64, pages=100, rotary=0, **more):
    cfg = F.rk_npu_hip_attention_paged_config()
    F.lib().rk_npu_hip_attention_paged_config_init(ctypes.byref(cfg))
    a = cfg.attention
    a.query_heads, a.kv_heads, a.head_dim, a.softmax_scale = qh, kh, d, 0.125
    a.max_query_rows, a.max_capacity, a.initial_capacity = 1, 1000, 0
    cfg.page, cfg.pages, cfg.rotary_dim = page, pages, rotary
    for name, value in more.items():
        setattr(cfg, name, value)
    return cfg


def query(cfg):
    sizes = F.rk_npu_attention_f16_sizes()
    return F.lib().rk_npu_hip_attention_paged_query(ctypes.byref(cfg), ctypes.byref(sizes)), sizes


def test_defaults():
    cfg, plain = F.rk_npu_hip_attention_paged_config(), F.rk_npu_attention_f16_config()
    F.lib().rk_npu_hip_attention_paged_config_init(ctypes.byref(cfg))
    F.lib().rk_npu_attention_f16_config_init(ctypes.byref(plain))
    assert bytes(cfg.attention) == bytes(plain)
    assert (cfg.page, cfg.pages, cfg.rotary_dim, cfg.interleaved, cfg.rope_theta) == (64, 0, 0, 0, 10000.0)
    assert not cfg.frequencies
    F.lib().rk_npu_hip_attention_paged_config_init(None)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_sizes(page):
    rc, s = query(config(page=page))
    assert rc == F.RK_NPU_OK
    assert s.key_bytes == s.value_bytes == 100 * page * 2 * 128 * 2 and s.tail_bytes == 0
    plain, cfg = F.rk_npu_attention_f16_sizes(), config()
    assert F.lib().rk_npu_attention_f16_query(ctypes.byref(cfg.attention), 0, 1, 0, ctypes.byref(plain)) == 0
    assert s.workspace_bytes == plain.workspace_bytes


def test_refused_configurations():
    assert query(config())[0] == F.RK_NPU_OK
    for bad in (dict(page=0), dict(page=8), dict(page=48), dict(page=512), dict(page=-16), dict(pages=0), dict(pages=-1),
                dict(pages=2 ** 31 - 1), dict(kh=0), dict(qh=7), dict(qh=1), dict(d=40), dict(kh=33, qh=33),
                dict(rotary=8), dict(rotary=144), dict(rotary=-16), dict(rotary=24), dict(interleaved=2),
                dict(interleaved=-1), dict(rotary=16, rope_theta=0.0), dict(rotary=16, rope_theta=-1.0),
                dict(rotary=16, rope_theta=float("inf")), dict(rotary=16, rope_theta=float("nan"))):
        assert query(config(**bad))[0] == F.RK_NPU_ERR_PARAM, bad
    assert query(config(rope_theta=0.0))[0] == F.RK_NPU_OK     # (no rotation)
    for value in (float("nan"), float("inf")):
        cfg = config(rotary=16)
        cfg.frequencies = (ctypes.c_double * 8)(*([1.0] * 7 + [value]))
        assert query(cfg)[0] == F.RK_NPU_ERR_PARAM
    cfg = config()
    cfg.attention.max_capacity = 2 ** 30 + 1
    assert query(cfg)[0] == F.RK_NPU_ERR_PARAM
    assert F.lib().rk_npu_hip_attention_paged_query(ctypes.byref(config()), None) == F.RK_NPU_ERR_PARAM
    assert F.lib().rk_npu_hip_attention_paged_query(None, ctypes.byref(F.rk_npu_attention_f16_sizes())) == F.RK_NPU_ERR_PARAM


def test_frequencies_whose_angles_pass_64_bits():
    """An angle that is not finite at a 32-bit position would make NaN of a row: refused. (2^31
    positions of 5.2e299 radians, in turns, are the largest number of 64 bits.)"""
    for theta in (5e-324, 1e-310, 1e-306):
        assert query(config(rotary=128, rope_theta=theta))[0] == F.RK_NPU_ERR_PARAM, theta
    for theta in (1e-301, 1e-3, 1.0, 1e300, 1.7e308):
        assert query(config(rotary=128, rope_theta=theta))[0] == F.RK_NPU_OK, theta
    assert query(config(rotary=16, rope_theta=1e-320))[0] == F.RK_NPU_OK    # (at most theta^(-7/8))
    for value, rc in ((1.7e308, F.RK_NPU_ERR_PARAM), (-1e300, F.RK_NPU_ERR_PARAM), (1e298, F.RK_NPU_OK), (-1e298, F.RK_NPU_OK)):
        cfg = config(rotary=16)
        cfg.frequencies = (ctypes.c_double * 8)(*([1.0] * 7 + [value]))
        assert query(cfg)[0] == rc, value


def test_null_handles():
    """Every call on no pool, and on memory that is no pool."""
    L, cfg = F.lib(), config()
    raw = ctypes.c_void_p(1)
    assert L.rk_npu_hip_attention_paged_pool_create(None, ctypes.byref(cfg), ctypes.byref(raw)) == F.RK_NPU_ERR_PARAM
    assert raw.value is None
    other = (ctypes.c_uint64 * 64)()
    at = ctypes.addressof(other)
    h = ctypes.byref(F.rk_npu_hip_heads(at, F.RK_NPU_HIP_F16, 128, 128))
    b = ctypes.byref(F.rk_npu_hip_paged_batch(1, 1, 1, 16, at, None, at, 1))
    for pool in (None, at):
        for rc in (L.rk_npu_hip_attention_paged_status(pool),
                   L.rk_npu_hip_attention_paged_append(pool, b, h, h, None, None, None, None),
                   L.rk_npu_hip_attention_paged_read(pool, b, h, h, None),
                   L.rk_npu_hip_attention_paged_run(None, pool, b, h, h, None),
                   L.rk_npu_hip_attention_paged_run(at, pool, b, h, h, None)):
            assert rc == F.RK_NPU_ERR_PARAM
        L.rk_npu_hip_attention_paged_pool_free(pool)


class Ints:
    """A cuda int32 tensor's attributes."""

    def __init__(self, *shape, dtype=torch.int32, stride=None, cuda=True):
        self.shape, self.dtype, self.is_cuda = shape, dtype, cuda
        self._stride = stride or tuple([1] if len(shape) == 1 else [shape[1], 1])

    def stride(self, i=None):
        return self._stride if i is None else self._stride[i]

    def data_ptr(self):
        return 64


def test_batches():
    """What a batch's tensors have to be, and the numbers it passes on."""
    b = D.PagedBatch(Ints(3, 5), Ints(3), Ints(4), max_rows=7)
    raw = b._raw(20, 16)
    assert (raw.sequences, raw.rows, raw.max_rows, raw.max_tokens, raw.table_stride) == (3, 20, 7, 80, 5)
    assert D.PagedBatch(Ints(3, 5, stride=(9, 1)), Ints(3), max_tokens=33)._raw(3, 16).table_stride == 9
    assert b._raw(20, 16, 50).max_tokens == 50      # (the pages' capacity)
    with pytest.raises(AttributeError):
        b.lengths = Ints(3)
    for build in (lambda: D.PagedBatch(Ints(3, 5), Ints(2)), lambda: D.PagedBatch(Ints(3, 5), Ints(3), Ints(3)),
                  lambda: D.PagedBatch(Ints(3, 5, stride=(1, 3)), Ints(3)),
                  lambda: D.PagedBatch(Ints(3, 5, stride=(4, 1)), Ints(3)),
                  lambda: D.PagedBatch(Ints(3, 5, dtype=torch.int64), Ints(3)),
                  lambda: D.PagedBatch(Ints(3, 5, cuda=False), Ints(3)),
                  lambda: D.PagedBatch(Ints(3, 5), Ints(3, stride=(2,))),
                  lambda: D.PagedBatch(Ints(3, 5), Ints(3), max_rows=2 ** 31),
                  lambda: D.PagedBatch(Ints(3, 5), Ints(3), max_tokens=2 ** 32 + 5),
                  lambda: D.PagedBatch(Ints(3, 5), Ints(3), max_tokens=81)._raw(3, 16),
                  lambda: D.PagedBatch(Ints(3, 5), Ints(3))._raw(2 ** 31, 16)):
        with pytest.raises(npu.NpuError):
            build()


def test_more_rows_allowed_than_there_are():
    """max_rows is a bound: the call's rows are another."""
    b = D.PagedBatch(Ints(3, 50), Ints(3), Ints(4), max_rows=512)
    assert [b._raw(n, 16).max_rows for n in (1, 300, 512, 700)] == [1, 300, 512, 512]
    for n in (0, -1):
        assert D.PagedBatch(Ints(3, 50), Ints(3), Ints(4), max_rows=n)._raw(300, 16).max_rows == n    # (refused by the call)


@pytest.mark.parametrize("n", [2 ** 31, 2 ** 32 + 5, -2 ** 31 - 1])
@pytest.mark.parametrize("name", ["query_heads", "kv_heads", "head_dim", "pages", "page", "capacity", "rotary_dim"])
def test_numbers_beyond_32_bits(name, n):
    sizes = dict(query_heads=2, kv_heads=1, head_dim=64, softmax_scale=0.1, pages=4, page=16, capacity=64, rotary_dim=16)
    with pytest.raises(npu.NpuError):
        D.KvPages(None, **{**sizes, name: n})
