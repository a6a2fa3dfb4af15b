"""The cache of latent rows held in 8 bits at further ends: positions at the last number, other strides, types and row shapes."""
import numpy as np
import pytest

from _gpu import lib, ok
from _kv8 import attend, bf16_bits, bf16_value, read_rows, tolerance, write_rows
from test_gpu_kv8 import Case, dev, ptr, read, rows, rows_flat, same, stream, write
from test_gpu_wait_status import plant

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("back,cap,s", [(3, 2, 6), (3, 1, 6), (1, 4, 9), (5, 5, 20), (6, 4, 6)])
def test_a_ring_at_the_end_of_the_numbers_keeps_the_last_row_that_has_an_entry(back, cap, s):
    x = rows(np.random.default_rng(s), 1, s, 128)
    got = write(x, 64, [(1 << 63) - back], cap, True)
    want = np.full_like(got, 0xA5)
    for t in range(min(s, back)):
        want[0, ((1 << 63) - back + t) % cap] = write_rows(x, 64)[0, t]
    assert same(got, want)


@pytest.mark.parametrize("code", [51, 57])
def test_a_code_in_the_status_word_stays_until_it_is_read(code):
    """Planted by the host, as the attention's waits (51 to 56) and its look at its own layout (57) would leave it: a call that only
    enqueues neither takes nor covers it."""
    import torch
    L, c = lib(), Case(3, n=200, seqs=2).put()
    o = torch.empty(c.rows, c.h, c.d, device="cuda")
    plant(code)
    try:
        ok(c.call(o), "attn")
        torch.cuda.synchronize()
        assert L.apus_cuda_kernel_status(0) == code
    finally:
        left = L.apus_cuda_kernel_status(1)
    assert left == code and L.apus_cuda_kernel_status(0) == 0
    c.check(c.out())


@pytest.mark.parametrize("scale", [3, 120, 127, 140])
def test_codes_of_nan_count_as_480_where_the_scale_is_a_number(scale):
    """In reading, where the scale is one that BF16 products hold or not, and in attention."""
    c = Case(9, n=100, seqs=2, nb=60, na=0, holes=0.0)
    c.kv_b[:, :, 5::7] = 0x7f
    c.kv_b[:, :, 3::64] = 0xff
    c.kv_b[:, :, 448:576] = 0
    c.kv_b[:, :, 576:583] = scale
    val = read_rows(c.kv_b, 512, 64)
    assert np.abs(val).max() == 480 * 2.0 ** (scale - 127)
    for bf16 in (False, True):
        assert same(read(c.kv_b, 512, 64, s=60, bf16=bf16), val)
    if scale > 16:                                            # else the values are below what an attention has to see
        c.scale *= 2.0 ** (127 - scale - 9)
        c.check(c.out())


def test_chunks_of_positions_over_a_ring_that_is_as_long_as_window_and_chunk():
    """Prompts in chunks of several lengths, a verify batch that is taken back and repeated, steps: every position attends its own
    window and the entries complete by then, whatever was written behind it in the same chunk."""
    import torch
    B, win, d, rd, h, ratio, s_max, cap = 2, 16, 512, 64, 64, 4, 40, 64
    L, rng, n = win - 1 + s_max, np.random.default_rng(6), 110
    x = rows_flat(rng, B, n, d)                               # of all positions; an entry is that of its last position, halved
    val = read_rows(write_rows(x, rd), d, rd)
    ent = read_rows(write_rows(0.5 * x[:, ratio - 1::ratio], rd), d, rd)
    q = bf16_value(bf16_bits(rng.standard_normal((B, n, h, d)).astype(np.float32)))
    sink = (rng.standard_normal(h) * 0.5).astype(np.float32)
    ring, cache = (torch.zeros(B, k, 592, dtype=torch.uint8, device="cuda") for k in (L, cap))
    dsink, at = dev(sink), 0
    for s in (40, 7, 6, 6, 1, 1, 33, 16, 6):
        if s == 6 and at == 53:
            at = 47                                           # the verify batch again, other rows kept of it
        p = at + np.arange(s)
        e0, e1 = at // ratio, (at + s) // ratio
        xd, pos = dev(x[:, at:at + s]), dev(np.full(B, at, np.int64))
        ok(lib().apus_cuda_kv8_write_dev(ptr(xd), 0, d, rd, B, s, ptr(pos), None, 1, ptr(ring), L, L, stream()), "kv8_write")
        if e1 > e0:
            ed, epos = dev(0.5 * x[:, ratio - 1::ratio][:, e0:e1]), dev(np.full(B, e0, np.int64))
            ok(lib().apus_cuda_kv8_write_dev(ptr(ed), 0, d, rd, B, e1 - e0, ptr(epos), None, 0, ptr(cache), cap, cap, stream()), "kv8_write")
        back = p[:, None] - win + 1 + np.arange(win)
        entries = np.where(np.arange(cap) < (p[:, None] + 1) // ratio, L + np.arange(cap), -1)
        ids = np.concatenate((np.where(back >= 0, back % L, -1), entries), 1)
        di, dq = dev(np.broadcast_to(ids, (B, *ids.shape)).astype(np.int32)), dev(q[:, at:at + s])
        o = torch.empty(B, s, h, d, device="cuda")
        ok(lib().apus_cuda_sparse_attn_kv8_dev(ptr(dq), 0, ptr(dsink), h, d, rd, ptr(di), win + cap, B * s, s, d ** -0.5, ptr(ring), L, L, ptr(cache), cap, cap,
                                               ptr(o), 0, stream()), "sparse_attn_kv8")
        got = o.cpu().numpy()
        for b in range(B):
            for t in range(s):
                i = at + t
                kv = np.concatenate((val[b, max(0, i - win + 1):i + 1], ent[b, :(i + 1) // ratio]))
                want, wv, es = attend(q[b, i], kv, np.ones(len(kv), bool), d ** -0.5, sink)
                assert (np.abs(got[b, t] - want) <= tolerance(want, wv, es)).all(), (at, b, t)
        at += s
    assert at == n
