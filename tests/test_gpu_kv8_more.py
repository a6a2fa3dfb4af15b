"""The cache of latent rows held in 8 bits at further ends: positions at the last number, other strides, types and row shapes."""
import numpy as np
import pytest

from _gpu import lib, ok
from _kv8 import read_rows, write_rows
from test_gpu_kv8 import Case, read, rows, same, write
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
