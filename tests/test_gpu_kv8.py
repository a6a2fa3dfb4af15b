"""The cache of latent rows held in 8 bits: rows written, read back and attended (apus_cuda_kv8_*_dev,
apus_cuda_sparse_attn_kv8_dev) against a plain restatement in 64 bits, at the sizes, masks and values where they can go wrong."""

import numpy as np
import pytest

from _gpu import P, lib, ok
from _kv8 import attend, bf16_bits, bf16_value, read_rows, row_bytes, tolerance, write_rows

pytestmark = pytest.mark.gpu


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def ptr(t):
    return None if t is None else t.data_ptr()


def stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


def rows(rng, *shape):
    """BF16 values of rows of very different sizes, with groups of zeros and tiny values."""
    x = rng.standard_normal(shape) * np.exp2(rng.integers(-12, 6, (*shape[:-1], 1)))
    x[..., 3::41] *= 2.0 ** -10
    if shape[-1] >= 128:
        x[rng.random(shape[:-1]) < 0.1, 64:128] = 0
    return bf16_value(bf16_bits(x.astype(np.float32)))


def write(x, rd, pos, cap, ring, counts=None, before=None, bf16=False, gap=0):
    """The caches' bytes after a call, [n_seq, cap + gap, row_bytes]."""
    import torch
    n, s, d = x.shape
    cache = dev(before if before is not None else np.full((n, cap + gap, row_bytes(d, rd)), 0xA5, np.uint8))
    xd = dev(bf16_bits(x).view(np.int16)) if bf16 else dev(x)
    pd, cd = dev(np.asarray(pos, np.int64)), None if counts is None else dev(np.asarray(counts, np.int32))
    ok(lib().apus_cuda_kv8_write_dev(ptr(xd), int(bf16), d, rd, n, s, ptr(pd), ptr(cd), int(ring), ptr(cache), cap, cap + gap, stream()), "kv8_write")
    torch.cuda.synchronize()
    return cache.cpu().numpy()


def read(rec, d, rd, cap=None, idx=None, first=0, s=None, bf16=False):
    import torch
    n, stride = rec.shape[:2]
    cap = stride if cap is None else cap
    s = idx.shape[1] if idx is not None else s
    cache, i = dev(rec), None if idx is None else dev(idx.astype(np.int32))
    out = torch.full((n, s, d), 7.0, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    ok(lib().apus_cuda_kv8_read_dev(ptr(cache), d, rd, cap, stride, n, s, ptr(i), first, ptr(out), int(bf16), stream()), "kv8_read")
    torch.cuda.synchronize()
    return out.float().cpu().numpy()


def same(a, b):
    return np.array_equal(np.ascontiguousarray(a, np.float32).view(np.uint32), np.ascontiguousarray(b, np.float32).view(np.uint32))


SHAPES = [(512, 64), (512, 0), (448, 64), (192, 64), (128, 0), (128, 64), (64, 0)]


@pytest.mark.parametrize("d,rd", SHAPES)
@pytest.mark.parametrize("n,s", [(1, 1), (3, 37), (65, 9)])
def test_write_is_the_definition_byte_for_byte(d, rd, n, s):
    x = rows(np.random.default_rng(d + s), n, s, d)
    pos = np.arange(n) % 3
    got = write(x, rd, pos, s + 5, False, gap=2)
    want = np.full_like(got, 0xA5)
    for b in range(n):
        want[b, pos[b]:pos[b] + s] = write_rows(x[b], rd)
    assert np.array_equal(got, want)
    assert np.array_equal(write(x, rd, pos, s + 5, False, gap=2, bf16=True), want)


@pytest.mark.parametrize("pos", [0, 127, 1000, (1 << 40) + 5])
@pytest.mark.parametrize("s", [1, 7, 128, 300])
def test_ring_keeps_the_last_rows(pos, s):
    x = rows(np.random.default_rng(s), 2, s, 128)
    got = write(x, 64, [pos, pos + 50], 128, True)
    want = np.full_like(got, 0xA5)
    for b in range(2):
        for t in range(s):
            want[b, (pos + 50 * b + t) % 128] = write_rows(x[b, t], 64)
    assert np.array_equal(got, want)


def test_rows_without_an_entry_and_padding_change_nothing():
    x = rows(np.random.default_rng(1), 6, 10, 192)
    pos, counts = [0, 5, 12, -4, 8, 1 << 50], [10, 0, 10, 10, -3, 99]
    got = write(x, 64, pos, 12, False, counts=counts, gap=1)
    want = np.full_like(got, 0xA5)
    for b in range(6):
        for t in range(min(max(counts[b], 0), 10)):
            if 0 <= pos[b] + t < 12:
                want[b, pos[b] + t] = write_rows(x[b, t], 64)
    assert np.array_equal(got, want) and (got[:, 12] == 0xA5).all()
    ring = write(x, 64, [0, 3, 2, -4, 8, 7], 4, True, counts=[10, 0, 3, 10, -3, 99])
    want = np.full_like(ring, 0xA5)
    for b, (p, c) in enumerate(zip([0, 3, 2, -4, 8, 7], [10, 0, 3, 10, 0, 10])):
        for t in range(c):
            if p + t >= 0:
                want[b, (p + t) % 4] = write_rows(x[b, t], 64)
    assert np.array_equal(ring, want)


def test_values_at_the_borders():
    """Zeros, subnormals, the largest values, ties, exact powers, and groups that are not finite."""
    x = np.zeros((1, 12, 128), np.float32)
    x[0, 1, :] = 1e-42
    x[0, 2, :64] = 3e38
    x[0, 3, :64] = np.linspace(-448, 448, 64)
    x[0, 4, :] = 448 * 2.0 ** -30
    x[0, 5, 0], x[0, 5, 1:64] = 448.0, (np.arange(63) + 0.5) / 2           # ties of the 4-bit significand among them
    x[0, 6, 7] = np.nan
    x[0, 7, 70] = -np.inf
    x[0, 8, :] = np.nextafter(np.float32(448), np.float32(500))
    x[0, 9, :64], x[0, 9, 64:] = -0.0, 2.0 ** -9
    x[0, 10, :64] = np.arange(64) * 2.0 ** -16
    x[0, 11, :] = 1e-4
    got = write(x, 0, [0], 12, False)
    assert np.array_equal(got[0], write_rows(x[0], 0))
    back = read(got, 128, 0, s=12)
    want = read_rows(got, 128, 0)
    assert np.array_equal(back, want.astype(np.float32), equal_nan=True)
    assert np.isnan(back[0, 6, :64]).all() and not back[0, 6, 64:].any() and np.isnan(back[0, 7, 64:]).all()
    tail = np.zeros((1, 1, 128), np.float32)
    tail[0, 0, 64:70] = [np.inf, -np.inf, np.nan, 3.4e38, -0.0, 1e-40]
    t = read(write(tail, 64, [0], 1, False), 128, 64, s=1)[0, 0, 64:70]
    assert np.array_equal(t, bf16_value(bf16_bits(tail[0, 0, 64:70])), equal_nan=True)


@pytest.mark.parametrize("d,rd", SHAPES)
def test_reading_gives_the_rounded_rows_and_writing_them_again_the_same_bytes(d, rd):
    x = rows(np.random.default_rng(5), 2, 23, d)
    rec = write(x, rd, [0, 0], 23, False)
    back = read(rec, d, rd, s=23)
    sim = np.ascontiguousarray(x.reshape(46, d))
    ok(lib().apus_cuda_fp8_qat_sim(P(sim), d, d - rd, 46), "qat")
    assert same(back.reshape(46, d), sim)                     # what the model's rows have been through
    assert same(read(rec, d, rd, s=23, bf16=True), back)
    assert np.array_equal(read_rows(write(back, rd, [0, 0], 23, False), d, rd), back.astype(np.float64))


def test_read_by_index_with_holes_and_a_shared_cache():
    import torch
    rng = np.random.default_rng(2)
    rec = write_rows(rows(rng, 3, 50, 512), 64)
    val = read_rows(rec, 512, 64).astype(np.float32)
    idx = rng.integers(-2, 55, (3, 77))
    got = read(rec, 512, 64, idx=idx)
    want = np.zeros((3, 77, 512), np.float32)
    for b in range(3):
        for t in range(77):
            if 0 <= idx[b, t] < 50:
                want[b, t] = val[b, idx[b, t]]
    assert same(got, want)
    assert same(read(rec, 512, 64, cap=40, first=-3, s=60)[:, 3:43], val[:, :40]) and not read(rec, 512, 64, cap=40, first=-3, s=60)[:, [0, 2, 43, 59]].any()
    out, cache = torch.empty(5, 4, 512, device="cuda"), dev(rec)
    ok(lib().apus_cuda_kv8_read_dev(ptr(cache), 512, 64, 50, 0, 5, 4, None, 9, ptr(out), 0, stream()), "kv8_read")
    assert same(out.cpu().numpy(), np.broadcast_to(val[0, 9:13], (5, 4, 512)))


# ---- attention -------------------------------------------------------------------------------------------
class Case:
    def __init__(self, seed, h=64, d=512, rd=64, n=640, seqs=1, per=1, na=128, nb=700, peak=1.0, holes=0.1, sink=True, shared=False):
        rng = np.random.default_rng(seed)
        R = seqs * per
        self.h, self.d, self.rd, self.n, self.rows, self.per, self.na, self.nb = h, d, rd, n, R, per, na, nb
        k = 1 if shared else seqs
        self.kv_a = write_rows(rows_flat(rng, k, na, d), rd)
        self.kv_b = write_rows(rows_flat(rng, k, nb, d), rd)
        self.shared = shared
        q = rng.standard_normal((R, h, d))
        q[:, ::5] *= peak
        self.q = bf16_value(bf16_bits(q.astype(np.float32)))
        self.idx = rng.integers(0, max(1, na + nb), (R, n)).astype(np.int32)
        self.idx[rng.random((R, n)) < holes] = -1
        self.sink = (rng.standard_normal(h) * 0.7).astype(np.float32) if sink else None
        self.scale = d ** -0.5

    def put(self):
        self.dq, self.di, self.ds = dev(self.q), dev(self.idx), None if self.sink is None else dev(self.sink)
        self.da, self.db = dev(self.kv_a), dev(self.kv_b)
        return self

    def call(self, out, st=None, qt=None):
        q, bf = (self.dq, 0) if qt is None else (qt, 1)
        st8 = 0 if self.shared else 1
        import torch
        return lib().apus_cuda_sparse_attn_kv8_dev(ptr(q), bf, ptr(self.ds), self.h, self.d, self.rd, ptr(self.di), self.n, self.rows, self.per, self.scale,
                                                   ptr(self.da) if self.na else None, self.na, st8 * self.na, ptr(self.db) if self.nb else None, self.nb,
                                                   st8 * self.nb, ptr(out), int(out.dtype == torch.bfloat16), stream() if st is None else st)

    def out(self, bf16=False, q_bf16=False):
        import torch
        self.put()
        o = torch.full((self.rows, self.h, self.d), 9.0, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
        qt = dev(bf16_bits(self.q).view(np.int16)) if q_bf16 else None
        ok(self.call(o, qt=qt), "sparse_attn_kv8")
        torch.cuda.synchronize()
        assert lib().apus_cuda_kernel_status(1) == 0
        return o.float().cpu().numpy()

    def want(self, r):
        seq = 0 if self.shared else r // self.per
        i = self.idx[r]
        val = np.concatenate((read_rows(self.kv_a[seq], self.d, self.rd), read_rows(self.kv_b[seq], self.d, self.rd)))
        valid = (i >= 0) & (i < self.na + self.nb)
        return attend(self.q[r], val[np.where(valid, i, 0)], valid, self.scale, self.sink)

    def check(self, got, some=None):
        assert same(got, bf16_value(bf16_bits(got)))         # BF16 values
        for r in range(self.rows) if some is None else some:
            o, wv, es = self.want(r)
            off = np.abs(got[r] - o) / tolerance(o, wv, es)
            assert off.max() <= 1, (r, off.max())


def rows_flat(rng, *shape):
    x = rng.standard_normal(shape)
    x *= 1 + 3 * (rng.random((*shape[:-1], 1)) < 0.1)
    return bf16_value(bf16_bits(x.astype(np.float32)))


# lengths around the sizes at which a tile, a 16-row step or a cluster's share ends
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 255, 257, 511, 640, 1025, 2049, 4100])
def test_lengths(n):
    c = Case(n, n=n, peak=3.0, nb=3000)
    c.check(c.out())


@pytest.mark.parametrize("h", [1, 2, 5, 8, 16, 31, 32, 33, 48, 63, 64, 65, 100, 128, 130])
def test_head_counts(h):
    c = Case(h, h=h, n=200, seqs=2)
    c.check(c.out())


@pytest.mark.parametrize("d,rd", SHAPES + [(256, 64), (320, 0), (384, 64), (256, 0)])
@pytest.mark.parametrize("n,seqs", [(333, 1), (1500, 3)])
def test_row_shapes(d, rd, n, seqs):
    c = Case(d + rd, h=64, d=d, rd=rd, n=n, seqs=seqs)
    c.check(c.out())


@pytest.mark.parametrize("seqs,per", [(1, 1), (2, 1), (5, 1), (9, 1), (19, 1), (33, 1), (75, 1), (150, 1), (1, 6), (3, 50), (2, 200)])
def test_batches_and_chunks(seqs, per):
    c = Case(seqs * 7 + per, n=300, seqs=seqs, per=per, nb=400)
    got = c.out()
    some = sorted({0, 1 % c.rows, c.rows // 2, c.rows - 1, *range(0, c.rows, 17)})
    c.check(got, some)


@pytest.mark.parametrize("n", [40, 640, 3000])
def test_types_of_queries_and_output_are_the_same_values(n):
    c = Case(3, n=n, seqs=3)
    a = c.out()
    assert same(c.out(bf16=True), a) and same(c.out(q_bf16=True), a) and same(c.out(bf16=True, q_bf16=True), a)
    keep = c.q
    c.q = keep + np.float32(2.0 ** -12) * keep * (np.arange(512) % 3 - 1).astype(np.float32)   # rounds back to the same BF16 values
    assert same(bf16_value(bf16_bits(c.q)), keep) and same(c.out(), a)


@pytest.mark.parametrize("n", [1, 100, 129, 2000])
@pytest.mark.parametrize("sink", [True, False])
def test_masks(n, sink):
    """Rows of holes only, one entry at the first or the last place, whole tiles of holes, ids behind the caches."""
    c = Case(8, n=n, seqs=8, sink=sink, holes=0.0)
    c.idx[0] = -1
    c.idx[1] = -1
    c.idx[1, 0] = 5
    c.idx[2] = -1
    c.idx[2, n - 1] = 777
    c.idx[3, n // 2:] = -1
    c.idx[4, :n // 2] = -1
    c.idx[5] = 828 + np.arange(n)                             # at the end of both caches and behind it
    c.idx[5, 0] = 827
    c.idx[6] = np.iinfo(np.int32).max
    c.idx[7] = np.iinfo(np.int32).min
    c.kv_a[:, 0, :] = 255                                     # a record full of NaN that nothing but holes could reach
    c.idx[c.idx == 0] = 1
    got = c.out()
    assert not got[0].any() and not got[6].any() and not got[7].any()
    c.check(got)


def test_no_ids_and_no_caches_give_zeros():
    c = Case(1, n=0, seqs=3)
    assert not c.out().any()
    c = Case(2, n=9, seqs=2, na=0, nb=0, holes=0.0)
    assert not c.out().any()


@pytest.mark.parametrize("na,nb", [(128, 0), (0, 50), (1, 1)])
def test_one_cache_only(na, nb):
    c = Case(4, n=150, seqs=2, na=na, nb=nb)
    c.check(c.out())


def test_the_same_entry_many_times_and_one_cache_for_all():
    c = Case(5, n=300, seqs=4, shared=True)
    c.idx[1] = 3
    c.idx[2] = 200
    c.check(c.out())


@pytest.mark.parametrize("sink", [-np.inf, np.inf, -1e30, 80.0, 3e38])
def test_sinks(sink):
    c = Case(6, n=200, seqs=2)
    c.sink[::2] = sink
    got = c.out()
    if sink == np.inf:
        assert not got[:, ::2].any()
        c.sink[::2] = 1e30                                    # as good as infinite
    with np.errstate(over="ignore", under="ignore"):
        c.check(got)


@pytest.mark.parametrize("n", [129, 700, 4000])
@pytest.mark.parametrize("order", ["rising", "falling", "late"])
def test_scores_far_apart(n, order):
    """Scores of some hundreds in rising order move the reference of the running softmax again and again."""
    c = Case(7, n=n, holes=0.0, nb=n, na=0, sink=True)
    c.scale = 1.0
    u = np.zeros(512, np.float32)
    u[100] = 1.0
    x = rows_flat(np.random.default_rng(9), 1, n, 512) * 0.25
    ramp = {"rising": np.linspace(-300, 300, n), "falling": np.linspace(300, -300, n), "late": np.where(np.arange(n) >= n - 3, 250.0, -200.0)}[order]
    x[0, :, 100] = ramp
    c.kv_b = write_rows(bf16_value(bf16_bits(x.astype(np.float32))), 64)
    c.q = bf16_value(bf16_bits((c.q * 0.02 + u).astype(np.float32)))
    c.q[:, 1::4] *= -1
    c.idx[:] = np.arange(n)
    c.check(c.out())


@pytest.mark.parametrize("n,sign", [(1, 1), (120, 1), (120, -1), (700, 1), (700, -1)])
def test_scores_of_hundreds_of_thousands(n, sign):
    """Every score is exact and a thousand or more away from the next one, so that the result is the row of the largest one."""
    c = Case(41, n=n, holes=0.0, na=0, nb=128)
    x = rows_flat(np.random.default_rng(9), 1, 128, 512)
    x[0, :, 500] = 1 + np.arange(128) / 128.0               # BF16 holds these, and 1,024 powers of e times them are apart
    c.kv_b = write_rows(bf16_value(bf16_bits(x.astype(np.float32))), 64)
    c.q[:] = 0
    c.q[:, :, 500] = sign * 2.0 ** 10 * 2.0 ** (np.arange(64) % 8)
    c.scale = 2.0 ** 7
    c.idx[0] = np.random.default_rng(5).integers(0, 128, n)
    got = c.out()
    best = c.idx[0].max() if sign > 0 else c.idx[0].min()
    row = np.broadcast_to(read_rows(c.kv_b[0, best], 512, 64), got.shape)    # BF16 values
    if sign > 0:
        assert np.array_equal(got, row)
    else:                                                     # the sink is far above every score
        assert not got.any()
    c.sink = None
    assert np.array_equal(c.out(), row)


def test_ends_of_the_numbers():
    """Positions whose rows run past the largest number are dropped, an id list may be as long as the sizes allow."""
    import torch
    x = rows(np.random.default_rng(3), 1, 6, 128)
    cache, xd = torch.zeros(1, 8, 208, dtype=torch.uint8, device="cuda"), dev(x)
    for pos, ring in (((1 << 63) - 3, 0), ((1 << 63) - 3, 1), (-(1 << 63), 1)):
        cache.zero_()
        ok(lib().apus_cuda_kv8_write_dev(ptr(xd), 0, 128, 64, 1, 6, ptr(dev(np.array([pos], np.int64))), None, ring, ptr(cache), 8, 8, stream()), "kv8_write")
        got, want = cache.cpu().numpy(), np.zeros((1, 8, 208), np.uint8)
        if pos > 0 and ring:
            for t in range(3):
                want[0, (pos + t) % 8] = write_rows(x, 64)[0, t]
        assert same(got, want)
    out = torch.full((1, 6, 128), 3.0, device="cuda")
    ok(lib().apus_cuda_kv8_read_dev(ptr(cache), 128, 64, 8, 8, 1, 6, None, (1 << 63) - 3, ptr(out), 0, stream()), "kv8_read")
    assert not out.any()


# rows for which a CTA has 16, 32 and 64 heads, with and without others at its row
@pytest.mark.parametrize("rows", [1, 6, 12, 30, 60, 160])
@pytest.mark.parametrize("n", [150, 700])
def test_masks_and_scores_far_apart_for_any_number_of_rows(rows, n):
    """Rows in turn: scores that rise by hundreds, fall, rise at the end; holes up to the last entry, behind the first, only."""
    c = Case(17, n=n, holes=0.0, nb=n, na=0, seqs=rows, shared=True)
    c.scale = 1.0
    u = np.zeros(512, np.float32)
    u[100] = 1.0
    x = rows_flat(np.random.default_rng(9), 1, n, 512) * 0.25
    x[0, :, 100] = np.linspace(-300, 300, n)
    c.kv_b = write_rows(bf16_value(bf16_bits(x.astype(np.float32))), 64)
    c.q = bf16_value(bf16_bits((c.q * 0.02 + u).astype(np.float32)))
    c.q[:, 1::4] *= -1
    up = np.arange(n)
    for r in range(rows):
        c.idx[r] = [up, up[::-1], np.where(up >= n - 3, up, up // 4), np.where(up == n - 1, up, -1), np.where(up == 0, up, -1), up * 0 - 1][r % 6]
    got = c.out()
    c.check(got, [r for r in range(rows) if r < 6 or r >= rows - 6])


def test_large_and_small_rows():
    """Scale bytes up to the largest that BF16 holds the values of, and down to the smallest that is written."""
    c = Case(11, n=100, holes=0.0, nb=60, na=0)
    x = rows_flat(np.random.default_rng(9), 1, 60, 512)
    x[0, 20:40] *= 2.0 ** 30
    x[0, 40:] *= 2.0 ** -40
    c.kv_b = write_rows(bf16_value(bf16_bits(x.astype(np.float32))), 64)
    c.scale = 2.0 ** -34
    c.check(c.out())


def test_a_row_that_is_not_finite_reaches_the_queries_that_ask_for_it():
    c = Case(12, n=150, seqs=2, holes=0.0)
    c.kv_b[0, 10, :] = write_rows(np.full((1, 512), np.nan, np.float32), 64)
    c.idx[c.idx == 138] = 3
    c.idx[0, 149] = 138
    got = c.out()
    assert np.isnan(got[0]).all()
    c.check(got, [1])


def test_entries_behind_four_gigabytes():
    import torch
    nb, rng = 7_600_000, np.random.default_rng(3)            # 4.5 GB of records
    c = Case(13, n=300, nb=64, na=16, holes=0.05)
    small = c.kv_b[0].copy()
    c.put()
    big = torch.zeros(nb, 592, dtype=torch.uint8, device="cuda")
    at = np.sort(rng.choice(np.arange(nb - 400_000, nb), 64, replace=False))
    at[-1] = nb - 1
    big[torch.from_numpy(at).cuda()] = dev(small)
    ids = np.where(c.idx < 16, c.idx, 16 + at[np.clip(c.idx - 16, 0, 63)]).astype(np.int32)
    di, o = dev(ids), torch.empty(1, 64, 512, device="cuda")
    ok(lib().apus_cuda_sparse_attn_kv8_dev(ptr(c.dq), 0, ptr(c.ds), 64, 512, 64, ptr(di), 300, 1, 1, c.scale, ptr(c.da), 16, 16, ptr(big), nb, nb, ptr(o), 0,
                                           stream()), "sparse_attn_kv8")
    c.check(o.cpu().numpy())
    x = rows(rng, 1, 3, 512)
    xd, pd, out = dev(x), dev(np.array([nb - 3], np.int64)), torch.empty(1, 3, 512, device="cuda")
    ok(lib().apus_cuda_kv8_write_dev(ptr(xd), 0, 512, 64, 1, 3, ptr(pd), None, 0, ptr(big), nb, nb, stream()), "kv8_write")
    ok(lib().apus_cuda_kv8_read_dev(ptr(big), 512, 64, nb, nb, 1, 3, None, nb - 3, ptr(out), 0, stream()), "kv8_read")
    assert same(out.cpu().numpy(), read_rows(write_rows(x, 64), 512, 64))
    del big


def test_streams_graphs_and_repeats_give_the_same_bits():
    import torch
    a, b = Case(20, n=640, seqs=3).put(), Case(21, n=333, seqs=40, h=8).put()
    outs = [torch.empty(c.rows, c.h, c.d, device="cuda") for c in (a, b)]
    for c, o in zip((a, b), outs):
        ok(c.call(o), "attn")
    torch.cuda.synchronize()
    want = [o.cpu().numpy() for o in outs]
    s = [torch.cuda.Stream() for _ in range(3)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s[2]):
        ok(a.call(outs[0], s[2].cuda_stream), "attn")
    many = [torch.empty_like(outs[1]) for _ in range(10)]
    outs[0].fill_(3)
    torch.cuda.synchronize()
    for k in range(10):
        with torch.cuda.stream(s[0]):
            graph.replay()
        ok(b.call(many[k], s[1].cuda_stream), "attn")
    torch.cuda.synchronize()
    assert same(outs[0].cpu().numpy(), want[0]) and all(same(m.cpu().numpy(), want[1]) for m in many)
    del graph


@pytest.mark.parametrize("n,h,rows,per", [(300, 130, 200, 50), (40, 1024, 20, 20), (700, 1000, 2, 1)])
def test_many_heads_and_more_rows_than_the_gpu_holds(n, h, rows, per):
    c = Case(h, h=h, n=n, seqs=rows // per, per=per, nb=300)
    got = c.out()
    c.check(got, [0, rows // 2, rows - 1])


@pytest.mark.parametrize("n", [100, 700])
@pytest.mark.parametrize("out_bf16", [False, True])
def test_pointers_on_16_byte_boundaries_only(n, out_bf16):
    """Queries, caches and output 16 bytes behind a coarser boundary, the bytes around the output as they were."""
    import torch
    c = Case(51, n=n, seqs=3, h=33)
    want = c.out(bf16=out_bf16)
    def shifted(t):
        raw = torch.zeros(t.numel() * t.element_size() + 4096, dtype=torch.uint8, device="cuda")
        at = (-raw.data_ptr()) % 1024 + 16
        v = raw[at:at + t.numel() * t.element_size()]
        v.copy_(t.reshape(-1).view(torch.uint8))
        return raw, v
    keep = [shifted(t) for t in (c.dq, c.da, c.db)]
    c.dq, c.da, c.db = (v for _, v in keep)
    es = 2 if out_bf16 else 4
    raw = torch.full((c.rows * c.h * c.d * es + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
    at = (-raw.data_ptr()) % 1024 + 16
    o = raw[at:at + c.rows * c.h * c.d * es].view(torch.bfloat16 if out_bf16 else torch.float32)
    ok(c.call(o), "attn")
    assert same(o.float().cpu().numpy().reshape(want.shape), want)
    assert (raw[:at] == 0x5A).all() and (raw[at + o.numel() * es:] == 0x5A).all()


def test_graphs_and_threads_side_by_side():
    """Two graphs whose rows are shared by several SMs, replayed on two streams at once, while two threads call on a third stream
    and on one each, with sizes that make the scratch of a stream grow."""
    import threading
    import torch
    cases = [Case(60 + i, n=n, seqs=s).put() for i, (n, s) in enumerate([(640, 2), (1500, 5), (300, 1), (2500, 9)])]
    want = []
    for c in cases:
        o = torch.empty(c.rows, c.h, c.d, device="cuda")
        ok(c.call(o), "attn")
        want.append(o)
    streams = [torch.cuda.Stream() for _ in range(5)]
    graphs, outs = [], [torch.empty_like(w) for w in want[:2]]
    for c, o, s in zip(cases, outs, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ok(c.call(o, s.cuda_stream), "attn")
        graphs.append(g)
    torch.cuda.synchronize()
    got, rcs = [[], []], []

    def calls(k):
        for i in range(12):
            c, w = cases[(i + k) % 4], want[(i + k) % 4]
            s = streams[2] if i & 1 else streams[3 + k]
            with torch.cuda.stream(s):
                o = torch.empty_like(w)
            rcs.append(c.call(o, s.cuda_stream))
            got[k].append((o, w))

    ts = [threading.Thread(target=calls, args=(k,)) for k in range(2)]
    for t in ts:
        t.start()
    for _ in range(12):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    for t in ts:
        t.join()
    torch.cuda.synchronize()
    assert not any(rcs)
    for o, w in [*got[0], *got[1], *zip(outs, want)]:
        assert torch.equal(o, w)
    del graphs


def test_the_first_call_of_a_process_may_be_recorded():
    import subprocess
    import sys
    code = """
import sys
sys.path[:0] = %r
import numpy as np, torch
from test_gpu_kv8 import Case, lib, ok
c = Case(3, n=640, seqs=2).put()
o = torch.zeros(2, 64, 512, device="cuda")
g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
torch.cuda.synchronize()
with torch.cuda.graph(g, stream=s):
    ok(c.call(o, s.cuda_stream), "attn")
g.replay()
torch.cuda.synchronize()
c.check(o.cpu().numpy())
""" % (sys.path,)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_a_decode_loop_over_8_bit_caches_is_the_loop_over_bf16_rows():
    """Written, attended and read back as a token loop does: a ring of the last positions and a cache that grows by an entry
    every few of them, beside apus_cuda_sparse_attn_batch_dev over the same rows in BF16."""
    import torch
    B, win, cap, d, rd, h, ratio = 3, 16, 40, 512, 64, 64, 4
    rng = np.random.default_rng(31)
    L = lib()
    ring8, cache8 = (torch.zeros(B, n, 592, dtype=torch.uint8, device="cuda") for n in (win, cap))
    ring16, cache16 = (torch.zeros(B, n, d, dtype=torch.bfloat16, device="cuda") for n in (win, cap))
    sink = dev((rng.standard_normal(h) * 0.5).astype(np.float32))
    entries = 0
    for pos in range(50):
        x = rows_flat(rng, B, 1, d)
        sim = np.ascontiguousarray(x.reshape(B, d))
        ok(L.apus_cuda_fp8_qat_sim(P(sim), d, d - rd, B), "qat")
        xd, p = dev(sim), dev(np.full(B, pos, np.int64))
        ok(L.apus_cuda_kv8_write_dev(ptr(xd), 0, d, rd, B, 1, ptr(p), None, 1, ptr(ring8), win, win, stream()), "kv8_write")
        ring16[:, pos % win] = xd.bfloat16()
        if pos % ratio == ratio - 1:
            p = dev(np.full(B, entries, np.int64))
            ok(L.apus_cuda_kv8_write_dev(ptr(xd), 0, d, rd, B, 1, ptr(p), None, 0, ptr(cache8), cap, cap, stream()), "kv8_write")
            cache16[:, entries] = xd.bfloat16()
            entries += 1
        q = dev(bf16_value(bf16_bits(rng.standard_normal((B, h, d)).astype(np.float32))))
        idx = np.full((B, win + cap), -1, np.int32)
        idx[:, :min(win, pos + 1)] = np.arange(min(win, pos + 1))
        idx[:, win:win + entries] = win + np.arange(entries)
        di = dev(idx)
        o8, o16 = torch.empty(B, h, d, device="cuda"), torch.empty(B, h, d, device="cuda")
        ok(L.apus_cuda_sparse_attn_kv8_dev(ptr(q), 0, ptr(sink), h, d, rd, ptr(di), win + cap, B, 1, d ** -0.5, ptr(ring8), win, win, ptr(cache8), cap, cap,
                                           ptr(o8), 0, stream()), "sparse_attn_kv8")
        ok(L.apus_cuda_sparse_attn_batch_dev(ptr(q), ptr(sink), h, d, ptr(di), win + cap, B, d ** -0.5, ptr(ring16), win, win, ptr(cache16), cap, cap, ptr(o16),
                                             stream()), "sparse_attn_batch")
        kv = torch.cat((ring16, cache16), 1).double().cpu().numpy()
        g8, g16 = o8.cpu().numpy(), o16.cpu().numpy()
        for b in range(B):                                    # both within the bound of the exact result
            o, wv, es = attend(q[b].cpu().numpy(), kv[b][np.where(idx[b] >= 0, idx[b], 0)], idx[b] >= 0, d ** -0.5, sink.cpu().numpy())
            t = tolerance(o, wv, es)
            assert (np.abs(g8[b] - o) <= t).all() and (np.abs(g16[b] - o) <= t).all()
    out = torch.empty(B, entries, d, device="cuda")
    ok(L.apus_cuda_kv8_read_dev(ptr(cache8), d, rd, cap, cap, B, entries, None, 0, ptr(out), 0, stream()), "kv8_read")
    assert same(out.cpu().numpy(), cache16[:, :entries].float().cpu().numpy())
