"""The bound of the paged attention finds the mistakes it is meant to find, planted in
its arithmetic, and passes that arithmetic."""
import numpy as np
import pytest

from tests import paged_bound as B


@pytest.mark.parametrize("one", [False, True])
@pytest.mark.parametrize("at", [1, 2, 7])
@pytest.mark.parametrize("high", [0.0, 5.875, 7.875])
@pytest.mark.parametrize("jump", [9, 16, 20, 23, 24, 25, 26, 31, 40])
def test_a_maximum_that_jumps(one, at, high, jump):
    """Weights of the unit before, which wait to be multiplied, keep their bits."""
    rng = np.random.default_rng(jump)
    q, k, v = B.jumps(rng, 64, 8, at, high, float(jump))
    want, most = B.attention(q[None], k[None], v[None], B.SCALE, 0, False, one, one)

    def off(plant=None):
        return max(float((np.abs(B.wave(q[r], k, v, B.SCALE, one, plant) - want[0, r]) / most[0, r]).max())
                   for r in range(0, 20, 3))

    assert off() <= 1.0
    # (a factor of 2^-25 is 0 in fp16; the unit's weights lie above the floor)
    before = np.ceil(high) if at == 1 or high > (6 if one else 8) else 0.0
    if jump - before >= 25 and jump - high <= 24:
        assert off("alpha") > 1.0
    if at > 1:
        assert off("drop") > 1.0 or (jump > 30 and at != 2)
