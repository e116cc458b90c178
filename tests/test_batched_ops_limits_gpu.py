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


def _far_case(H, KV, hd, rows, past, sign, bits, seed):
    """Scores of about sign * 2^(2 bits - 1) whose differences are whole
    multiples of their spacing in fp32. q and k are whole numbers with few
    bits, so every product and every sum of them
    is exact in fp32 in any order and in parts of 11 bits."""
    c = ref.Case(H, KV, hd, rows, past, seed=seed)
    rng = np.random.default_rng(seed)
    used = np.isfinite(c.k[:, 0, :, 0])
    big, step = 2.0 ** bits, 2.0 ** (2 * bits - 23)
    q = np.zeros((c.T, H, hd), np.float32)
    q[:, :, 0] = big / 2 + rng.integers(0, 2 ** (bits - 3), (c.T, H))
    q[:, :, 1:4] = step
    k = np.zeros_like(c.k)
    k[..., 0] = sign * big
    k[..., 1:4] = rng.integers(-1, 2, k.shape[:-1] + (3,))
    c.q = q.reshape(c.T, H * hd)
    c.k = np.where(used[:, None, :, None], k, c.k)
    c.scale = 1.0
    return c


def _check_far(c, kind, got, masks=None):
    """The scores are exact (above), so only the weights' arithmetic counts: a
    weight's argument x (in powers of two below the row's largest) passes a
    scale of 2^-23, up to four roundings of 2^-24 and an exponential of 2^-22.
    Weights from 2^-32 on count: 32 * 0.7 * (2^-23 + 4 * 2^-24) + 2^-22 <
    2^-17 of a weight, 2^-19 more as in ref.attention (its own bits, the sums),
    twice that of the mean of |v|, and 2^-37 of the largest |v|."""
    want, _ = ref.attention(kind, c.q, c.k, c.v, c.table, c.start, c.past, c.H, c.scale, masks)
    vabs, _ = ref.attention(kind, c.q, c.k, np.abs(c.v), c.table, c.start, c.past, c.H, c.scale, masks)
    top = np.abs(c.v[np.isfinite(c.v)]).max()
    tol = (2.0 ** -17 + 2.0 ** -19) * 2 * vabs + top * 2.0 ** -37
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (bad.mean(), np.argwhere(bad)[:3], got[bad][:3], want[bad][:3])


@pytest.mark.parametrize("hd", [48, 128, 160])
@pytest.mark.parametrize("sign,bits", [(1, 12), (1, 13), (-1, 13), (1, 15), (-1, 15)])
def test_scores_of_any_size(hd, sign, bits):
    """Scores of 2^23, 2^25 and 2^29, of either sign: over one unit of keys and over
    several, in tiles that the shares of the work cut and in whole ones."""
    for rows, past in (([40], [0]), ([70, 3, 100], [100, 200, 1]), ([1 + i % 3 for i in range(700)], [40] * 700)):
        c = _far_case(4, 2, hd, rows, past, sign, bits, seed=hd + bits)
        _check_far(c, "packed", _call(c, "packed"))


@pytest.mark.parametrize("hd", [64, 96, 132])
def test_scores_of_any_size_under_masks(hd):
    """Rows of huge and of ordinary scores in one tile, rows without a key, keys
    of the largest score masked."""
    c = _far_case(4, 2, hd, [30, 9], [0, 130], 1, 13, seed=hd)
    q = c.q.reshape(c.T, 4, hd)
    q[::3] = np.random.default_rng(1).normal(0, 1e-4, q[::3].shape)  # ordinary scores
    q[::3, :, 0] = 2.0 ** -13
    masks = ref.masks_of(ref.random_parents(np.random.default_rng(2), 39), 1)
    masks[30:] = ref.masks_of(ref.random_parents(np.random.default_rng(3), 9), 1)
    masks[4:7] = 0
    masks[11] = 0b100010
    got = _call(c, "tree", masks)
    want, tol = ref.attention("tree", c.q, c.k, c.v, c.table, c.start, c.past, c.H, c.scale, masks)
    ordinary = np.arange(c.T) % 3 == 0
    assert np.all(np.abs(got - want)[ordinary] <= tol[ordinary])
    assert np.all(got[4:7] == 0)
    c.q[ordinary] = 0.0  # compared above: uniform weights in what follows
    _check_far(c, "tree", _call(c, "tree", masks), masks)


def _check_scaled(c, kind, got, masks=None):
    want, tol = ref.attention(kind, c.q, c.k, c.v, c.table, c.start, c.past, c.H, c.scale, masks)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (bad.mean(), np.argwhere(bad)[:3], got[bad][:3], want[bad][:3])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size", [1e-33, 1e34, 5e37])
def test_values_near_the_ends_of_their_range(hd, size):
    """The mean of values that fp32 holds, where their sum and the sum of their
    scaled parts need not be: in tiles that the shares cut and in whole ones.
    (Values of up to 5 * 5e37 < 3.4e38; from 2^-112 up a value's parts lose
    nothing to its range, so the bounds are the usual ones.)"""
    for rows, past in (([200, 9], [57, 1000]), ([1 + i % 3 for i in range(700)], [90] * 700)):
        c = ref.Case(4, 2, hd, rows, past, seed=hd)
        c.v = (c.v.astype(np.float64) * size).astype(np.float32)
        _check_scaled(c, "packed", _call(c, "packed"))
    masks = ref.masks_of(ref.random_parents(np.random.default_rng(4), 20), 1)
    c = ref.Case(8, 2, hd, [20], [3000], seed=hd + 1)
    c.v = (c.v.astype(np.float64) * size).astype(np.float32)
    _check_scaled(c, "tree", _call(c, "tree", masks), masks)


@pytest.mark.parametrize("hd", [132, 256])
@pytest.mark.parametrize("size", [1e-33, 1e34, 5e37])
def test_wide_heads_values_near_the_ends_of_their_range(hd, size):
    test_values_near_the_ends_of_their_range(hd, size)


@pytest.mark.parametrize("hd", [48, 64, 128])
def test_factors_of_very_different_sizes_stay_within_the_stated_bound(hd):
    """K rows and dims of q that differ by up to 10^9 within a page and a row. What
    the parts of a factor cannot hold next to the largest one counts: 2^-38 of
    the largest K of the page times |q|, and of the largest q of the row times
    |k|, moves a score by up to scale * hd * 2^-38 * kmax * qmax each; a weight by
    twice that, and so the output (ref.attention's argument) by twice that of
    the mean of |v| again."""
    c = ref.Case(4, 2, hd, [60, 3], [100, 130], seed=hd)
    rng = np.random.default_rng(hd)
    with np.errstate(invalid="ignore"):
        c.k *= np.float32(10.0) ** rng.integers(-9, 1, (c.n_pages, 1, 64, 1)).astype(np.float32)
    c.q = (c.q.reshape(c.T, 4, hd) * np.float32(10.0) ** rng.integers(-9, 1, (c.T, 4, hd)).astype(np.float32)).reshape(c.T, -1)
    got = _call(c, "packed")
    want, tol = ref.attention("packed", c.q, c.k, c.v, c.table, c.start, c.past, c.H, c.scale)
    vabs, _ = ref.attention("packed", c.q, c.k, np.abs(c.v), c.table, c.start, c.past, c.H, c.scale)
    kmax = np.abs(c.k[np.isfinite(c.k)]).max()
    qmax = np.abs(c.q).reshape(c.T, 4, hd).max(2).repeat(hd, axis=1)
    tol = tol + 2 * (2 * 2 * c.scale * hd * 2.0 ** -38 * kmax * qmax) * vabs
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (bad.mean(), np.argwhere(bad)[:3])


@pytest.mark.parametrize("hd", [64, 128, 160])
def test_values_next_to_much_larger_ones_that_weigh_nothing(hd):
    """The first page holds values of 1e38 whose weights are exactly 0 (scores more
    than 1000 below the others'), the pages behind it values of 1e-32: the result
    is that of the pages behind it alone."""
    S = 400  # so that a share of the work has all pages of a sequence
    c = ref.Case(4, 2, hd, [1 + i % 2 for i in range(S)], [150] * S, seed=hd)
    first = c.table[:, 0].copy()
    with np.errstate(invalid="ignore"):
        c.v *= np.float32(1e-32)
    c.v[first] = np.float32(1e38) * np.sign(np.random.default_rng(1).normal(size=c.v[first].shape)).astype(np.float32)
    c.q[:] = np.abs(c.q) + 1.0
    c.k[first] = -40.0 * np.sqrt(hd)
    got = _call(c, "packed")
    c.table[:, 0] = -1  # left out
    _check_scaled(c, "packed", got)
