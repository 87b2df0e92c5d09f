"""Edge cases of the serving operators' host side (include/pyxis_serve.h) without a GPU."""
import math

import numpy as np
import pytest

import pyxis_b200 as px
from pyxis_b200 import _native


def yarn(rot, theta, factor, context, fast, slow):
    """The header's formula, index by index."""
    def at(turns):
        return rot * math.log(context / (2 * math.pi * turns)) / (2 * math.log(theta))

    low, high = max(0, math.floor(at(fast))), min(rot - 1, math.ceil(at(slow)))
    out = []
    for i in range(rot // 2):
        f = theta ** (-2 * i / rot)
        r = min(1.0, max(0.0, (i - low) / (high - low))) if high > low else float(i > low)
        out.append(f * (1 - r) + f / factor * r)
    return np.array(out)


@pytest.mark.parametrize("rot", [64, 128])
@pytest.mark.parametrize("theta,factor,context,fast,slow", [
    (1e6, 4.0, 32768, 32.0, 1.0), (1e4, 8.0, 65536, 32.0, 1.0), (1e4, 4.0, 131072, 32.0, 1.0), (1e4, 4.0, 1e6, 32.0, 1.0),
    (1e4, 2.0, 4096, 32.0, 1.0), (5e5, 8.0, 8192, 4.0, 1.0), (100.0, 3.0, 1e9, 32.0, 1.0), (1e4, 16.0, 100, 32.0, 1.0),
    (1e4, 2.0, 5.0, 32.0, 1.0), (1e4, 4.0, 131072, 16.5, 16.25)])
def test_every_yarn_frequency(rot, theta, factor, context, fast, slow):
    g, m = px.rope_frequencies(rot, theta, "yarn", factor=factor, original_context=context, beta_fast=fast, beta_slow=slow)
    np.testing.assert_allclose(g, yarn(rot, theta, factor, context, fast, slow), rtol=1e-13)  # a few u of 64 bits in pow and the mixture
    assert m == pytest.approx(0.1 * math.log(factor) + 1, rel=1e-15)


def test_yarn_leaves_frequencies_that_turn_often_alone_at_the_slow_end():
    # a context so long that the last frequency turns 18 times in it: it is in the ramp, not past it
    f, _ = px.rope_frequencies(128, 1e4)
    g, _ = px.rope_frequencies(128, 1e4, "yarn", factor=4.0, original_context=1e6)
    assert 1e6 * f[-1] / (2 * math.pi) > 18
    assert g[-1] > 0.8 * f[-1]


def test_a_table_that_was_freed_is_not_forked():
    pool = px.PagePool(8, 16)
    t = pool.allocate(40)
    stale, twice = list(t), [t[0], t[0], t[1]]
    with pytest.raises(px.PyxisError):
        pool.fork(twice, 40)
    with pytest.raises(px.PyxisError):
        pool.fork([0, 1, 99], 40)
    pool.free(t)
    assert pool.available == 8
    with pytest.raises(px.PyxisError):
        pool.fork(stale, 40)
    assert pool.available == 8
    a, b = pool.allocate(64), pool.allocate(64)
    assert sorted(a + b) == list(range(8))  # no page is given out twice


def test_sizes_past_32_bits_are_refused():
    for rot in ((1 << 32) + 2, 1 << 31, -(1 << 40)):
        with pytest.raises(px.PyxisError) as e:
            px.rope_frequencies(rot, 1e4)
        assert e.value.code == _native.PYXIS_EINVAL
