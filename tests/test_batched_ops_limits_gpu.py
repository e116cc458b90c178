"""The batched-step operators at the ends of their ranges, against the plain
64-bit implementations: scores and values of any finite size, the largest
vocabulary."""
import numpy as np
import pytest

import aaedn_b200 as ab
import batched_ops_ref as ref
from test_batched_ops_gpu import _call, _sample, _want

pytestmark = pytest.mark.gpu


def _flat_rows(B, V, rng):
    """Rows whose mass is near vocab times the largest: equal logits, two values a
    step apart, a high temperature over a narrow bulk; and a peaked one."""
    lg = np.full((B, V), 0.75, np.float32)
    lg[1::4] = np.where(rng.random(V) < 0.5, np.float32(2.0), np.float32(1.9999999))
    lg[2::4] = rng.integers(-3, 4, V).astype(np.float32) * 0.5
    lg[3::4] = rng.normal(0, 3, V).astype(np.float32)
    T = np.ones(B, np.float32)
    T[2::4] = 1e6
    return lg, T


@pytest.mark.parametrize("B,V", [(8, 1000000), (76, 1000000), (8, 524289), (76, 600001), (80, 524285)])
def test_sample_flat_rows_of_the_largest_vocabularies(B, V):
    """Few rows and more than four rounds of CTAs; draws over the whole range, the
    cuts one at a time. (A token's mass is rounded by 2^-45 of the largest, so a
    draw could differ from the 64-bit one only where its target lies within
    2^-25 of a token's border, relative to the row's mass.)"""
    rng = np.random.default_rng(B + V)
    lg, T = _flat_rows(B, V, rng)
    u = (rng.random(B) * (1 - 2.0 ** -24)).astype(np.float32)
    u[:8] = (0.0, 0.1, 0.3, 0.999, 1 - 2.0 ** -24, 0.6, 0.9, 0.45)
    p = rng.choice([1.0, 0.99, 0.9, 0.6], B).astype(np.float32)
    k = rng.choice([0, 0, 40, 530000, 300000], B)
    m = rng.choice([0.0, 0.0, 0.5], B).astype(np.float32)
    got, want = _sample(lg, T, k, p, m, u), _want(lg, T, k, p, m, u)
    assert np.array_equal(got, want), np.argwhere(got != np.array(want))[:5]
    few = slice(0, min(B, 8))  # no cut at all
    got, want = _sample(lg, T, None, None, None, u), _want(lg[few], T[few], None, None, None, u[few])
    assert np.array_equal(got[few], want)
