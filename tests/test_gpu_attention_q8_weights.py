"""The 8-bit KV cache's attention where weights, V's scales or both lie far apart,
and where every key counts: each output within a bound of its own
(tests/kv_bound.py), in every kernel, for both output types."""
import numpy as np
import pytest
import torch

from open_rknpu2_lm_infer_amd import device as D
from tests import kv_bound, kv_cases, kv_model

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32
# Query rows per KV head and HM_Q8_TILE: one row group a wave, two (of head_dim 256
# with 2), and the kernel for much work.
KERNELS = [(2, 0), (80, 0), (80, 1), (80, 2)]


@pytest.fixture(scope="module")
def ctx():
    return D.DeviceContext(0)


def check(ctx, appends, dtype, fmt="i8", block=32, causal=False, rows=1, qh=2, tile=-1, seed=0, q=None, d=64):
    """Appends the rows, attends with `rows` rows per query head at the end."""
    print(f"{fmt} block={block} causal={causal} rows={rows} qh={qh} tile={tile} {dtype} seed={seed}", flush=True)
    kh = appends[0][0].shape[0]
    n = sum(k.shape[1] for k, _ in appends)
    scale = float(np.float32(d ** -0.5))
    cache = D.KvCacheQ8(ctx, qh, kh, d, scale, n, fmt=fmt, block=block, causal=causal, max_query_rows=rows)
    k, v = (kv_model.KvModel(kh, d, fmt, block) for _ in range(2))
    for a, b in appends:
        k.append(a)
        v.append(b)
        cache.append(torch.from_numpy(a).cuda(), torch.from_numpy(b).cuda())
    rng = np.random.default_rng(seed)
    q = rng.standard_normal((qh, rows, d)).astype(np.float16) if q is None else np.broadcast_to(q, (qh, rows, d)).copy()
    out = torch.full((qh, rows, d), 77.0, dtype=dtype, device="cuda")
    with D.plan_switch("HM_Q8_TILE", tile):
        D.attention_q8(ctx, cache, torch.from_numpy(q).cuda(), out, max(n - rows, 0))
    want, most = kv_bound.attention(q, k.values(), v.values(), kv_bound.steps(v), scale, n - rows, causal,
                                    dtype == F16)
    got = out.double().cpu().numpy()
    worst = np.abs(got - want) / most
    assert worst.max() <= 1.0, f"{worst.max()} of the bound at {np.unravel_index(worst.argmax(), worst.shape)}"
    return got


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("fmt,block", [("i8", 32), ("i8", 128), ("e4m3", 64)])
@pytest.mark.parametrize("large_first", [True, False])
@pytest.mark.parametrize("power", [12, 18, 22, 26])
def test_scales_far_apart(ctx, power, large_first, fmt, block, dtype):
    """Half of the keys with values 2^power times the other half's: both count in the
    sum of the weights. The tail's values are those of the half before it."""
    for rows, tile in KERNELS[:3]:
        rng = np.random.default_rng(power)
        check(ctx, kv_cases.far_apart(rng, 1, 64, power, large_first, tail=20), dtype, fmt, block, rows=rows // 2,
              tile=tile, causal=tile == 1)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("power", [18, 24])
def test_scales_far_apart_of_wide_heads(ctx, power, dtype):
    for rows, tile in KERNELS:
        rng = np.random.default_rng(power)
        check(ctx, kv_cases.far_apart(rng, 1, 256, power, True, tail=20), dtype, rows=rows // 2, tile=tile, d=256)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("gap", [10, 14, 16])
def test_a_strong_key_of_no_value(ctx, gap, dtype):
    """Nearly all of a row's weight on a key whose V is zero, in a block of larger
    values: the output is the other keys', each of a weight e^-gap."""
    for fmt in ("i8", "e4m3"):
        for rows, tile in KERNELS[:3] + [(2, 1)]:
            rng = np.random.default_rng(gap)
            q = rng.standard_normal(64).astype(np.float16)
            check(ctx, kv_cases.strong_key(rng, 1, 64, q, 0.125, gap), dtype, fmt, rows=rows // 2, tile=tile, q=q)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("fmt,block", [("i8", 32), ("i8", 128), ("e4m3", 64)])
@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -14, 1.0, 2000.0])
@pytest.mark.parametrize("zeros_first", [True, False])
def test_blocks_of_zeros(ctx, zeros_first, size, fmt, block, dtype):
    """Half of the keys, and the tail, have values of zero: they take their share of
    the weight and leave the others' values all of their bits, however small."""
    for rows, tile in KERNELS[:3]:
        rng = np.random.default_rng(3)
        check(ctx, kv_cases.zeros(rng, 1, 64, size, zeros_first, tail=20), dtype, fmt, block, rows=rows // 2, tile=tile)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_only_zeros(ctx, dtype):
    """No value anywhere: outputs of zero, exactly."""
    for n in (20, 32, 300):
        for rows, tile in KERNELS[:3]:
            got = check(ctx, [(np.ones((1, n, 64), np.float16), np.zeros((1, n, 64), np.float16))], dtype,
                        rows=rows // 2, tile=tile)
            assert not got.any()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_a_tail_of_no_value(ctx, dtype):
    """The last tokens' V are zero, beside ordinary values: their weight counts."""
    for fmt in ("i8", "e4m3"):
        for rows, tile in KERNELS[:3]:
            rng = np.random.default_rng(5)
            head = kv_cases.far_apart(rng, 1, 64, 26, False)
            k = rng.standard_normal((1, 24, 64)).astype(np.float16)
            check(ctx, head + [(k, np.zeros_like(k))], dtype, fmt, rows=rows // 2, tile=tile)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("qh,kh,d,rows,keys", [(1, 1, 128, 1, 9000), (4, 1, 128, 1, 2500), (8, 2, 64, 2, 5001),
                                               (16, 2, 256, 1, 4000), (8, 1, 128, 16, 4100), (4, 1, 256, 20, 3000)])
def test_every_unit_counts(ctx, qh, kh, d, rows, keys, fmt, dtype):
    """Each 32 keys name themselves in V, so that one left out or taken twice, in a
    wave, a split or a join, shows whole in its output."""
    rng = np.random.default_rng(keys)
    for tile in ((0, 1, 2) if qh // kh * rows > 16 else (0,)):
        check(ctx, kv_cases.marks(rng, kh, d, keys), dtype, fmt, rows=rows, qh=qh, tile=tile, causal=rows > 1, d=d)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("qh,kh,d,rows,keys", [(32, 8, 128, 1, 3980), (16, 8, 64, 8, 2000), (16, 2, 256, 2, 5000),
                                               (1, 1, 64, 1, 1), (4, 2, 128, 3, 45)])
def test_few_rows_of_f16_output_are_rounded_once(ctx, qh, kh, d, rows, keys, fmt):
    """Up to 16 query rows per KV head: fp16 outputs are the f32 ones, rounded."""
    print(f"{fmt} qh={qh} kh={kh} d={d} rows={rows} keys={keys}", flush=True)
    cache = D.KvCacheQ8(ctx, qh, kh, d, d ** -0.5, keys, fmt=fmt, max_query_rows=rows)
    g = torch.Generator("cuda").manual_seed(keys)
    k, v = (torch.randn(kh, keys, d, device="cuda", generator=g) for _ in range(2))
    cache.append(k, v)
    q = torch.randn(qh, rows, d, device="cuda", generator=g)
    outs = [torch.empty(qh, rows, d, device="cuda", dtype=t) for t in (F32, F16)]
    for o in outs:
        D.attention_q8(ctx, cache, q, o, keys - rows)
    assert torch.equal(outs[0].half(), outs[1])
