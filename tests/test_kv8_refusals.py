"""What the entry points of the 8-bit cache refuse, asked on the CPU: arguments are looked at before any device is, and no
pointer given here is ever followed."""
import pytest

import apus_b200

X, CACHE, POS, OUT, IDX = 0x1000, 0x2000, 0x3000, 0x4000, 0x5000
WRITE = dict(x=X, bf16=0, d=512, rd=64, n_seq=2, s=3, pos=POS, counts=None, ring=1, cache=CACHE, cap=128, stride=128, st=None)
READ = dict(cache=CACHE, d=512, rd=64, cap=128, stride=128, n_seq=2, s=3, idx=IDX, first=0, out=OUT, bf16=0, st=None)
ATTN = dict(q=X, q_bf16=0, sink=None, h=64, d=512, rd=64, idxs=IDX, idxw=640, rows=6, per=3, scale=0.04, kv_a=CACHE, na=128, sa=128,
            kv_b=CACHE, nb=1000, sb=1000, o=OUT, o_bf16=1, st=None)


def refused(fn, base, change, word):
    L = apus_b200.lib()
    rc = getattr(L, fn)(*dict(base, **change).values())
    assert rc == 1 and word in L.apus_cuda_last_error().decode(), (rc, L.apus_cuda_last_error())


@pytest.mark.parametrize("d,rd", [(0, 0), (-64, 0), (63, 0), (576, 64), (512, 32), (512, 128), (64, 64), (512, -64)])
def test_row_shapes(d, rd):
    L = apus_b200.lib()
    assert L.apus_cuda_kv8_row_bytes(d, rd) == 0
    for fn, base in (("apus_cuda_kv8_write_dev", WRITE), ("apus_cuda_kv8_read_dev", READ), ("apus_cuda_sparse_attn_kv8_dev", ATTN)):
        refused(fn, base, dict(d=d, rd=rd), "d=")


def test_row_bytes():
    L = apus_b200.lib()
    assert L.apus_cuda_kv8_row_bytes(512, 64) == 592 and L.apus_cuda_kv8_row_bytes(512, 0) == 528 and L.apus_cuda_kv8_row_bytes(128, 64) == 208


@pytest.mark.parametrize("change,word", [
    (dict(n_seq=-1), "sequences"), (dict(s=-1), "sequences"), (dict(cap=-1), "cap"), (dict(stride=-1), "stride"), (dict(stride=127), "apart"),
    (dict(cache=None), "no cache"), (dict(cache=CACHE + 8), "16-byte"), (dict(x=None), "rows"), (dict(x=X + 16), "32-byte"), (dict(x=X + 4, bf16=1), "16-byte"),
    (dict(pos=None), "positions"), (dict(n_seq=1 << 20, s=1 << 20), "too many")])
def test_write(change, word):
    refused("apus_cuda_kv8_write_dev", WRITE, change, word)


@pytest.mark.parametrize("change,word", [
    (dict(n_seq=-1), "sequences"), (dict(cap=-1), "cap"), (dict(stride=-2), "stride"), (dict(cache=None), "no cache"), (dict(cache=CACHE + 1), "16-byte"),
    (dict(out=None), "output"), (dict(out=OUT + 16), "32-byte"), (dict(out=OUT + 4, bf16=1), "16-byte"), (dict(n_seq=1 << 20, s=1 << 20), "too many")])
def test_read(change, word):
    refused("apus_cuda_kv8_read_dev", READ, change, word)


@pytest.mark.parametrize("change,word", [
    (dict(h=0), "h="), (dict(h=1025), "h="), (dict(rows=-1), "rows"), (dict(idxw=-1), "ids"), (dict(idxw=(1 << 30) + 1), "ids"), (dict(per=0), "sequences"), (dict(per=4), "sequences"),
    (dict(na=-1), "na="), (dict(nb=-1), "nb="), (dict(nb=1 << 31), "nb="), (dict(sa=-1), "stride"), (dict(sb=-1), "stride"), (dict(kv_a=None), "no cache"),
    (dict(kv_b=None), "no cache"), (dict(kv_a=CACHE + 8), "16-byte"), (dict(kv_b=CACHE + 4), "16-byte"), (dict(q=None), "queries"), (dict(o=None), "output"),
    (dict(idxs=None), "ids"), (dict(q=X + 4), "16-byte"), (dict(o=OUT + 2), "16-byte")])
def test_attention(change, word):
    refused("apus_cuda_sparse_attn_kv8_dev", ATTN, change, word)


def test_nothing_to_do_needs_no_device():
    L = apus_b200.lib()
    for fn, base, change in (("apus_cuda_kv8_write_dev", WRITE, dict(s=0)), ("apus_cuda_kv8_write_dev", WRITE, dict(n_seq=0)),
                             ("apus_cuda_kv8_write_dev", WRITE, dict(cap=0, cache=None)), ("apus_cuda_kv8_read_dev", READ, dict(s=0)),
                             ("apus_cuda_sparse_attn_kv8_dev", ATTN, dict(rows=0, per=1, q=None, o=None))):
        assert getattr(L, fn)(*dict(base, **change).values()) == 0, L.apus_cuda_last_error()


@pytest.mark.parametrize("na,nb", [((1 << 63) - 1, (1 << 63) - 1), (1 << 62, 1 << 62), ((1 << 62) + 5, (1 << 63) - (1 << 62)), (1 << 31, 0), (1, (1 << 31) - 1)])
def test_cache_sizes_whose_sum_leaves_its_type(na, nb):
    refused("apus_cuda_sparse_attn_kv8_dev", ATTN, dict(na=na, nb=nb), "na=")
