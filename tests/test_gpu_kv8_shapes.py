"""Attention over 8-bit caches at every row shape where a CTA has 64, 32 and 16 heads and several tiles (the numbers of rows and
candidates are those at which the rule takes them), at strides of their own, and to the norm of the difference."""
import numpy as np
import pytest

from _gpu import lib, ok
from _kv8 import bf16_bits, bf16_value, read_rows, write_rows
from _kv8_norm import norms
from test_gpu_kv8 import SHAPES, Case, dev, ptr, read, rows, same, stream, write

pytestmark = pytest.mark.gpu

ALL = SHAPES + [(256, 64), (320, 0), (384, 64), (256, 0)]
# candidates, query rows: 64 heads and 3 tiles, 64 in 2 CTAs per row and 7 tiles, 32 in 4 and 5, 32 in 16 and 4, 16 in 16 and 5
SIZES = [(333, 160), (1500, 40), (2000, 16), (6000, 3), (8320, 1)]


def flat(n, seqs, d=512, rd=64, h=64, nb=None, q=2.0 ** -4, holes=0.1):
    """Rows of much the same length and queries so small that all candidates weigh alike."""
    c = Case(n + d, h=h, d=d, rd=rd, n=n, seqs=seqs, shared=True, na=128, nb=nb or max(700, n), holes=holes)
    rng = np.random.default_rng(n)
    c.kv_a, c.kv_b = (write_rows(rng.standard_normal((1, k, d)).astype(np.float32), rd) for k in (c.na, c.nb))
    c.q *= np.float32(q)
    return c


def check_norm(c, got, some):
    val = np.concatenate((read_rows(c.kv_a[0], c.d, c.rd), read_rows(c.kv_b[0], c.d, c.rd)))
    for r in some:
        kv = val[c.idx[r][c.idx[r] >= 0]]
        off, bound = norms(got[r], c.q[r], kv, c.scale, c.sink)
        assert off <= bound, (r, off, bound)
        # one candidate less would be seen
        off, bound = norms(got[r], c.q[r], np.delete(kv, len(kv) // 3, 0), c.scale, c.sink)
        assert off > bound, (r, off, bound)


@pytest.mark.parametrize("d,rd", ALL)
@pytest.mark.parametrize("n,seqs", SIZES)
def test_every_candidate_counts_once(n, seqs, d, rd):
    c = flat(n, seqs, d, rd)
    got = c.out()
    c.check(got, sorted({0, seqs // 2, seqs - 1}))
    check_norm(c, got, sorted({0, seqs // 2, seqs - 1}))


@pytest.mark.parametrize("n,seqs,h", [(640, 1, 64), (640, 32, 64), (640, 32, 16), (100, 5, 20), (3000, 9, 128), (128, 300, 64)])
def test_every_candidate_counts_once_for_other_heads_and_rows(n, seqs, h):
    c = flat(n, seqs, h=h)
    got = c.out()
    check_norm(c, got, sorted({0, seqs // 2, seqs - 1}))
    assert same(c.out(bf16=True, q_bf16=True), got)


@pytest.mark.parametrize("d,rd", ALL)
@pytest.mark.parametrize("n,seqs", SIZES)
def test_scores_far_apart_at_every_row_shape(n, seqs, d, rd):
    """Scores that rise and fall by 300 move the references in every CTA; whole tiles of holes in between."""
    c = flat(n, seqs, d, rd, nb=n, q=0.02, holes=0.0)
    c.scale = 1.0
    x = 0.25 * np.random.default_rng(n).standard_normal((1, n, d))
    x[0, :, 36] = np.linspace(-150, 150, n)
    c.kv_b = write_rows(bf16_value(bf16_bits(x.astype(np.float32))), rd)
    c.q[:, :, 36] = np.where(np.arange(64) % 2, -1.0, 1.0)
    up = 128 + np.arange(n)
    gap = np.where(np.arange(n) // 120 % 3 == 1, -1, up)
    for r in range(seqs):
        c.idx[r] = [up, up[::-1], gap, gap[::-1]][r % 4]
    got = c.out()
    c.check(got, sorted({0, 1 % seqs, 2 % seqs, seqs - 1}))


@pytest.mark.parametrize("n,seqs,per", [(300, 3, 1), (300, 40, 4), (1500, 20, 2)])
def test_caches_further_apart_than_they_are_long(n, seqs, per):
    import torch
    c = Case(77, n=n, seqs=seqs, per=per, h=33)
    c.put()
    wide = []
    for rec, gap in ((c.kv_a, 3), (c.kv_b, 11)):
        w = np.full((seqs, rec.shape[1] + gap, rec.shape[2]), 255, np.uint8)    # records of NaN in between
        w[:, :rec.shape[1]] = rec
        wide.append(dev(w))
    o = torch.full((c.rows, c.h, c.d), 9.0, device="cuda")
    ok(lib().apus_cuda_sparse_attn_kv8_dev(ptr(c.dq), 0, ptr(c.ds), c.h, c.d, c.rd, ptr(c.di), c.n, c.rows, c.per, c.scale, ptr(wide[0]), c.na, c.na + 3,
                                           ptr(wide[1]), c.nb, c.nb + 11, ptr(o), 0, stream()), "sparse_attn_kv8")
    got = o.cpu().numpy()
    c.check(got, sorted({0, 1, c.rows // 2, c.rows - 1}))
    assert same(c.out(), got)


@pytest.mark.parametrize("d,rd", [(512, 64), (128, 0)])
@pytest.mark.parametrize("s,cap", [(1, 128), (300, 128), (37, 37)])
def test_a_ring_of_bf16_rows(s, cap, d, rd):
    x = rows(np.random.default_rng(s), 3, s, d)
    pos, counts = [5, 1000, 127], [s, max(1, s - 20), s]
    got = write(x, rd, pos, cap, True, counts=counts, bf16=True, gap=2)
    want = np.full_like(got, 0xA5)
    for b in range(3):
        for t in range(counts[b]):
            want[b, (pos[b] + t) % cap] = write_rows(x[b, t], rd)
    assert same(got, want)


@pytest.mark.parametrize("d,rd", [(512, 64), (192, 64), (64, 0)])
def test_reading_by_index_into_bf16_rows(d, rd):
    rng = np.random.default_rng(d)
    rec = write_rows(rows(rng, 3, 50, d), rd)
    idx = rng.integers(-2, 55, (3, 77))
    want = np.where(((idx >= 0) & (idx < 50))[..., None], read_rows(rec, d, rd)[np.arange(3)[:, None], np.clip(idx, 0, 49)], 0)
    assert same(read(rec, d, rd, idx=idx, bf16=True), want) and same(read(rec, d, rd, idx=idx), want)


@pytest.mark.parametrize("per,entries", [(200, 0), (6, 0), (200, 1000), (90, 7)])
def test_chunks_of_window_layers_and_of_heavily_compressed_ones(per, entries):
    """Two prompts; row t attends rows t .. t + 127 of its window buffer and the entries that were complete at its position."""
    seqs, win = 2, 128
    c = Case(per + entries, n=win + entries, seqs=seqs, per=per, na=win - 1 + per, nb=entries, holes=0.0)
    t = np.tile(np.arange(per), seqs)[:, None]
    have = entries - 4 + t * 4 // per                         # some complete within the chunk
    e = np.arange(entries)
    c.idx[:] = np.concatenate((t + np.arange(win), np.where(e < have, c.na + e, -1)), 1)
    c.check(c.out(), sorted({0, 1, per - 1, per, c.rows // 2 + 1, c.rows - 1}))
