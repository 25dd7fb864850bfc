"""The bound of the 8-bit KV cache's attention finds the mistakes it is meant to
find, planted in its arithmetic, and passes that arithmetic."""
import numpy as np
import pytest

from tests import kv_bound, kv_cases, kv_model


def check(appends, f16, fmt="i8", d=64, plants=(), q=None):
    rng = np.random.default_rng(7)
    k, v = (kv_model.KvModel(1, d, fmt, 32) for _ in range(2))
    for a, b in appends:
        k.append(a)
        v.append(b)
    scale = float(np.float32(d ** -0.5))
    q = rng.standard_normal((1, 1, d)).astype(np.float16) if q is None else q[None, None]
    step = kv_bound.steps(v)
    x, y = k.values(), v.values()
    want, most = kv_bound.attention(q, x, y, step, scale, 0, False, f16)

    def off(plant=None):
        got = kv_bound.wave(q[0, 0], x[0], y[0], step[0], scale, f16, plant=plant)
        return float((np.abs(got - want[0, 0]) / most[0, 0]).max())

    assert off() <= 1.0
    for plant in plants:
        assert off(plant) > 1.0, plant


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("large_first", [False, True])
@pytest.mark.parametrize("power", [12, 18, 22, 26])
def test_scales_far_apart(power, large_first, f16):
    rng = np.random.default_rng(power)
    lost = f16 and large_first and power >= 22
    check(kv_cases.far_apart(rng, 1, 64, power, large_first, tail=20), f16, plants=("sum",) if lost else ())


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("size", [2.0 ** -18, 2.0 ** -14, 1.0, 2000.0])
@pytest.mark.parametrize("zeros_first", [False, True])
def test_blocks_of_zeros(zeros_first, size, f16):
    rng = np.random.default_rng(3)
    plants = ("zeros",) if zeros_first and size < 1e-3 and not f16 else ()
    if f16 and not zeros_first and size > 1.0:
        plants += ("sum",)
    check(kv_cases.zeros(rng, 1, 64, size, zeros_first, tail=20), f16, plants=plants)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("gap", [10, 14, 16])
def test_a_strong_key_of_no_value(gap, f16):
    rng = np.random.default_rng(gap)
    q = rng.standard_normal(64).astype(np.float16)
    check(kv_cases.strong_key(rng, 1, 64, q, 0.125, gap), f16, q=q, plants=("units", "offset") if f16 and gap >= 14 else ())


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_a_lost_unit(fmt, f16):
    rng = np.random.default_rng(9)
    check(kv_cases.marks(rng, 1, 64, 9000), f16, fmt, plants=("drop",))
