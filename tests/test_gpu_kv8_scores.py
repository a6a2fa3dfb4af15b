"""Attention over 8-bit caches where scores lie far apart: what a softmax in one pass may drop, and what it must not."""
import numpy as np
import pytest

from _gpu import lib, ok                       # noqa: F401
from _kv8 import attend, bf16_bits, bf16_value, read_rows, tolerance, write_rows
from test_gpu_kv8 import Case, rows_flat

pytestmark = pytest.mark.gpu

LN2 = float(np.log(2.0))


def levels(n, rows, place, level, value=None):
    """`rows` query rows over one cache, whose record i has a score of level[i] powers of two for every head (and a little
    noise); candidate j is record place[j].  `value`: the records' rows [len(level), d], or random ones of 512."""
    k = len(level)
    x = rows_flat(np.random.default_rng(9), k, 512) if value is None else value.astype(np.float32)
    d = x.shape[1]
    c = Case(71, n=n, d=d, seqs=rows, shared=True, na=0, nb=k, holes=0.0)
    x[:, d - 12] = level
    c.kv_b = write_rows(bf16_value(bf16_bits(x)), 64)[None]
    c.q *= np.float32(2.0 ** -8)
    c.q[:, :, :64] = 0
    c.q[:, :, d - 64:] = 0
    c.q[:, :, d - 12] = 1
    c.scale = LN2
    c.idx[:] = place
    return c


def check(c, got, some):
    """Case.check, and beside its tolerance what the one pass may drop.  A numerator is dropped below 2^-126, where the reference is
    48 powers of two above the largest score: a weight below 2^-78.  A part of a row, whose numerators are at most 2^64, is dropped
    where its factor is below 2^-126: weights below 2^-62, of which 2^-61 is a bound with all roundings."""
    val = read_rows(c.kv_b[0], c.d, c.rd)
    for r in some:
        o, wv, es = attend(c.q[r], val[c.idx[r]], np.ones(c.n, bool), c.scale, c.sink)
        off = np.abs(got[r] - o) / (tolerance(o, wv, es) + 2.0 ** -61 * np.abs(val[c.idx[r]]).sum(0))
        assert off.max() <= 1, (r, off.max())


# Most candidates weigh 2^-15 of the last one, hundreds or thousands of times, so that they count; they come where the
# running reference has not moved for long, and the last one moves it.  CTAs that have seen the first ones, all and the
# last one meet in a join.
@pytest.mark.parametrize("most", [15.5, 33.0, 47.5, 63.0, 79.5, 95.5, 111.5, 124.0])
@pytest.mark.parametrize("n,rows,lead", [(640, 1, 80), (640, 1, 450), (640, 160, 112), (640, 1024, 112), (8320, 1, 100), (8320, 1, 1800), (8320, 32, 450)])
def test_many_candidates_just_below_a_late_maximum(n, rows, lead, most):
    level = np.concatenate((np.zeros(16), np.full(16, most), [most + 15]))
    at = np.arange(n)
    c = levels(n, rows, np.where(at < lead, at % 16, np.where(at < n - 1, 16 + at % 16, 32)), level)
    x = rows_flat(np.random.default_rng(9), 33, 512)
    x[16:32, :64], x[32, :64], x[:, 500] = 1.0, 0.0, level
    c.kv_b = write_rows(x[None], 64)
    check(c, c.out(), sorted({0, rows - 1}))


# A sink above every score, where the scores have risen far above the first reference or stayed far below it.
@pytest.mark.parametrize("rise,sink", [(0.0, 10.0), (0.0, 50.0), (0.0, -40.0), (60.0, 100.0), (111.0, 121.0), (111.0, 160.0), (111.0, 60.0)])
@pytest.mark.parametrize("n,rows", [(640, 1), (640, 160), (8320, 2)])
def test_sinks_far_from_the_reference(n, rows, rise, sink):
    at = np.arange(n)
    c = levels(n, rows, np.where(at < n - 30, at % 16, 16 + at % 16), np.concatenate((np.zeros(16), np.full(16, rise))))
    c.sink[:] = sink * LN2
    check(c, c.out(), sorted({0, rows - 1}))


# Rows of any size that a record holds, in the codes (a scale byte far above the others') or in the rotated channels, behind
# scores that let the numerators grow: where the sums of the definition are numbers, so are these.
@pytest.mark.parametrize("rise", [0.0, 30.0, 47.5, 49.0, 63.0, 100.0, 111.5, 140.0])
@pytest.mark.parametrize("power,late", [(31, 300), (33, 300), (60, 1), (80, 1), (115, 300), (120, 1)])
@pytest.mark.parametrize("n,rows,d,channel", [(640, 1, 512, 3), (640, 160, 512, 3), (640, 160, 512, 450), (8320, 2, 512, 450), (640, 160, 192, 3), (640, 160, 192, 130)])
def test_large_values_behind_scores_that_rise(n, rows, d, channel, rise, power, late):
    level = np.concatenate((np.zeros(16), np.full(16, rise)))
    x = rows_flat(np.random.default_rng(9), 32, d)
    x[16:, channel] = -1.5 * 2.0 ** power
    at = np.arange(n)
    c = levels(n, rows, np.where(at < n - late, at % 16, 16 + at % 16), level, x)
    got = c.out()
    assert np.isfinite(got).all()
    check(c, got, sorted({0, rows - 1}))


# Every score is exact and thousands away from the next one, up to the end of f32, so that the result is the row of the largest
# one, or nothing beside a sink far above.
@pytest.mark.parametrize("n,rows", [(1, 1), (120, 1), (700, 1), (700, 160)])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("power", [20, 24, 31, 60, 90, 118])
def test_scores_up_to_the_largest_numbers(power, sign, n, rows):
    c = Case(41, n=n, holes=0.0, na=0, nb=128, seqs=rows, shared=True)
    x = rows_flat(np.random.default_rng(9), 128, 512)
    x[:, 500] = 1 + np.arange(128) / 128.0
    c.kv_b = write_rows(x, 64)[None]
    c.q[:] = 0
    c.q[:, :, 500] = 2.0 ** (np.arange(64) % 8)
    c.scale = sign * 2.0 ** power
    c.idx[:] = np.random.default_rng(5).integers(0, 128, (rows, n))
    best = c.idx.max(1) if sign > 0 else c.idx.min(1)
    want = np.broadcast_to(read_rows(c.kv_b[0, best], 512, 64)[:, None], (rows, 64, 512))
    assert np.array_equal(c.out(), want if sign > 0 else np.zeros_like(want))
    c.sink = None
    assert np.array_equal(c.out(), want)
