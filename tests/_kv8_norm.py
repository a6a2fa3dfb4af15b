"""A bound on the norm of what an attention over 8-bit caches is off by, sharp enough to see one candidate too few or too many."""
import numpy as np

U = 2.0 ** -8                                                # half a BF16 step at the low end of a binade


def norms(got, q, kv, scale, sink):
    """One query row: (norm of got - o, bound), o in 64 bits.

    With weights w_j and v_j the rows: the numerators' roundings d_j move the result by sum_j w_j d_j (v_j - o), their sum being that
    of the rounded ones; the result's rounding by r o.  |d|, |r| <= U, spread over at most half a step to each side: variance U^2 / 3
    at most.  A score is a sum of d products in f32, every partial one rounded by at most 2^-24 of the sum of magnitudes M, and is
    then scaled, subtracted and put into an exponential (4 * 2^-24 of the score and 2^-21): variance (d + 2) (2^-24 M)^2 and the
    square of the rest.  The roundings are as good as independent, so the square of the norm over all heads and channels is

        sum over heads of  sum_j w_j^2 |v_j - o|^2 (U^2 / 3 + e^2)  +  |o|^2 U^2 / 3

    in the mean; the bound is twice the root of it, which a sum over 16 or more heads does not reach by chance."""
    q, kv = np.asarray(q, np.float64), np.asarray(kv, np.float64)
    d = q.shape[1]
    x = q @ kv.T * scale
    m = x.max(1) if sink is None else np.maximum(x.max(1), sink)
    p = np.exp(x - m[:, None])
    w = p / (p.sum(1) + (0 if sink is None else np.exp(sink - m)))[:, None]
    o = w @ kv
    mag = (np.abs(q) @ np.abs(kv).T * abs(scale)).max(1)
    e2 = (d + 2) * (2.0 ** -24 * mag) ** 2 + (4 * 2.0 ** -24 * (np.abs(x).max(1) + np.abs(m)) + 2.0 ** -21) ** 2
    oo = (o * o).sum(1)
    vo = (kv * kv).sum(1)[None] - 2 * o @ kv.T + oo[:, None]                 # |v_j - o|^2
    var = ((w * w * vo).sum(1) * (U * U / 3 + e2) + oo * U * U / 3).sum()
    return np.sqrt(((got - o) ** 2).sum()), 2 * np.sqrt(var)
