"""The 8-bit cache's record and the attention over it, restated in numpy and in 64 bits."""
import numpy as np

GROUP = 64


def row_bytes(d, rd):
    return d + rd + 16


def bf16_bits(x):
    """Nearest BF16 value, ties to even, as 16 bits (NaN stays NaN)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where((u & 0x7fffffff) > 0x7f800000, (u >> 16).astype(np.uint16), r)


def bf16_value(b):
    return (np.ascontiguousarray(b).astype(np.uint32) << 16).view(np.float32)


_CODES = np.array([(8 + m) * 2.0 ** (e - 10) if e else m * 2.0 ** -9 for e in range(16) for m in range(8)])   # code 127 = 480


def e4m3(v):
    """Nearest of the 127 magnitudes up to 448, ties to the even code."""
    a, sign = np.abs(v), np.signbit(v)
    hi = np.clip(np.searchsorted(_CODES[:127], a), 1, 126)
    lo = hi - 1
    dl, dh = a - _CODES[lo], _CODES[hi] - a
    c = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return (c + 128 * sign).astype(np.uint8)


def write_rows(x, rd):
    """x [..., d] f32 -> records [..., row_bytes]."""
    x = np.asarray(x, np.float32)
    d = x.shape[-1]
    nq = d - rd
    g = x[..., :nq].reshape(*x.shape[:-1], nq // GROUP, GROUP)
    rec = np.zeros((*x.shape[:-1], row_bytes(d, rd)), np.uint8)
    amax = np.abs(g).max(-1)
    odd = ~np.isfinite(amax)
    p = np.maximum(np.where(odd, 1.0, amax), np.float32(1e-4)).astype(np.float32) * np.float32(1.0 / 448.0)
    m, e = np.frexp(p)
    e = e - (m == 0.5)
    codes = e4m3(np.where(np.isfinite(g), g, 0).astype(np.float64) * np.exp2(-e.astype(np.float64))[..., None])
    codes[odd] = 0x7f
    rec[..., :nq] = codes.reshape(*x.shape[:-1], nq)
    if rd:
        rec[..., nq:d + rd] = np.ascontiguousarray(bf16_bits(x[..., nq:])).view(np.uint8)
    rec[..., d + rd:d + rd + nq // GROUP] = np.where(odd, 255, e + 127).astype(np.uint8)
    return rec


def read_rows(rec, d, rd):
    """Records -> f64 values."""
    nq = d - rd
    c = rec[..., :nq]
    b = rec[..., d + rd:d + rd + nq // GROUP].astype(np.float64)
    s = np.where(b == 255, np.nan, np.exp2(np.maximum(b, 0) - 127))
    v = _CODES[c & 127] * np.where(c & 128, -1.0, 1.0) * np.repeat(s, GROUP, -1)
    if not rd:
        return v
    tail = bf16_value(np.ascontiguousarray(rec[..., nq:d + rd]).view(np.uint16)).astype(np.float64)
    return np.concatenate((v, tail), -1)


def attend(q, kv, valid, scale, sink):
    """One query row: q [h, d], kv [n, d], valid [n], sink [h] or None -> (o, sum of w |v|, largest |error| that the f32 sums of a
    score may have, over the heads) in 64 bits."""
    q, kv = np.asarray(q, np.float64), np.asarray(kv, np.float64)[valid]
    h, d = q.shape
    if not len(kv):
        z = np.zeros((h, d))
        return z, z, np.zeros((h, 1))
    x = q @ kv.T * scale
    m = x.max(1) if sink is None else np.maximum(x.max(1), sink)
    p = np.exp(x - m[:, None])
    w = p / (p.sum(1) + (0 if sink is None else np.exp(sink - m)))[:, None]
    # a score is a sum of d products in f32 (any order: each partial sum rounds by 2^-24 of at most the sum of magnitudes),
    # then a multiplication, a subtraction of a reference and an exponential of it (2^-22 with the argument's own rounding)
    mag = np.abs(q) @ np.abs(kv).T * abs(scale)
    es = (d + 2) * 2.0 ** -24 * mag.max(1) + 4 * 2.0 ** -24 * (np.abs(x).max(1) + np.abs(m)) + 2.0 ** -21
    return w @ kv, w @ np.abs(kv), es[:, None]


def tolerance(o, wv, es):
    """A numerator is rounded to BF16 (half a step: 2^-8), and so is the result; the weights' sum is that of the rounded
    numerators, so it is off by 2^-8 too.  With A = sum w |v| and es the relative error of a numerator from its score:
    |error| <= (2^-8 + es) A + (2^-8 + es) |o| + 2^-8 |o|, times the second order (1 + 2^-6), and the f32 sums of the
    output, 2^-24 per term of at most some ten thousand terms (2^-10 A is far above them for the sizes here: 2^-24 n <= 2^-11)."""
    u = 2.0 ** -8
    return (1 + 2.0 ** -6) * ((u + es + 2.0 ** -11) * (wv + np.abs(o)) + u * np.abs(o)) + 1e-30
