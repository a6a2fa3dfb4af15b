"""The cache of latent rows held in 8 bits, as measurable cases: rows quantised as they are written into it, read back
from it, and attended where they lie.

A cache row is one token's (or one compressed entry's) latent vector, key and value at once, shared by all heads.  It
is kept as a record of d - rd E4M3 codes, rd BF16 values (the rotated channels) and one UE8M0 scale byte for every 64
codes, padded to a multiple of 16 bytes.  Sizes are those of DeepSeek-V4-Flash (64 heads, 512 channels of which 64
rotated, a window of 128, the top 512 of the compressed entries) over the contexts and batches of this repository's
benchmark, with smaller heads and head counts beside them.
"""
import math

import torch

own = False

HEADS, HEAD_DIM, ROPE_DIM, WINDOW, TOPK, GROUP = 64, 512, 64, 128, 512, 64
MOST_ATTN = 1024 * (WINDOW + TOPK) * HEADS          # query rows x candidates x heads of the largest listed attention


def listed():
    return [
        # a decode step's rows into the window rings of 32 sequences that are past the first turn
        {"name": "write_step_b32", "op": "write", "B": 32, "s": 1, "d": 512, "rd": 64, "ring": True, "bf16": False, "cap": 128, "pos": 1501, "ragged": False},
        # the entries of eight prompts of odd lengths, appended
        {"name": "write_prompts", "op": "write", "B": 8, "s": 511, "d": 512, "rd": 64, "ring": False, "bf16": False, "cap": 1024, "pos": 130, "ragged": True},
        # a long context handed over as BF16 rows, all at once
        {"name": "write_context", "op": "write", "B": 4, "s": 16384, "d": 512, "rd": 64, "ring": False, "bf16": True, "cap": 16384, "pos": 0, "ragged": False},
        # the rows that one step selected, for a host that keeps f32 state; some are holes
        {"name": "read_selected", "op": "read", "B": 3, "s": 641, "d": 512, "rd": 64, "cap": 2001, "gather": True, "bf16": False},
        # whole caches back to BF16 rows
        {"name": "read_caches", "op": "read", "B": 8, "s": 8192, "d": 512, "rd": 64, "cap": 8192, "gather": False, "bf16": True},
        # sliding-window layers, where a shard holds eight of the heads
        {"name": "attn_window_b5_h8", "op": "attn", "form": "window", "ctx": 700, "B": 5, "s": 1, "h": 8, "d": 512, "rd": 64, "bf16": False},
        # one query against a million tokens of context: window and the chosen 512 entries
        {"name": "attn_csa_1m_b1", "op": "attn", "form": "csa", "ctx": 1 << 20, "B": 1, "s": 1, "h": 64, "d": 512, "rd": 64, "bf16": True},
        # a decode batch at an everyday context
        {"name": "attn_csa_8k_b32", "op": "attn", "form": "csa", "ctx": 8192, "B": 32, "s": 1, "h": 64, "d": 512, "rd": 64, "bf16": False},
        # a heavily compressed layer attends every entry a sequence has; odd batch, every sequence of its own length
        {"name": "attn_hca_100k_b7", "op": "attn", "form": "hca", "ctx": 100003, "B": 7, "s": 1, "h": 64, "d": 512, "rd": 64, "bf16": True},
        # the same at a full batch and a million tokens
        {"name": "attn_hca_1m_b32", "op": "attn", "form": "hca", "ctx": 1 << 20, "B": 32, "s": 1, "h": 64, "d": 512, "rd": 64, "bf16": True},
        # the verify batch of speculative decoding: six positions of one sequence
        {"name": "attn_verify_s6", "op": "attn", "form": "csa", "ctx": 4001, "B": 1, "s": 6, "h": 64, "d": 512, "rd": 64, "bf16": False},
        # a chunk of two prompts, every position with its own window and its own choice
        {"name": "attn_prompt_b2_s512", "op": "attn", "form": "csa", "ctx": 4096, "B": 2, "s": 512, "h": 64, "d": 512, "rd": 64, "bf16": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("write", "read", "attn", "attn", "attn"))
    d, rd = rng.choice(((512, 64), (512, 64), (512, 64), (512, 0), (256, 64), (192, 64), (128, 0)))
    if op == "write":
        B = _log(rng, 1, 64)
        s = _log(rng, 1, 65536 // B)
        ring, pos = rng.random() < 0.5, rng.randint(0, 3000)
        return {"op": op, "B": B, "s": s, "d": d, "rd": rd, "ring": ring, "bf16": rng.random() < 0.5, "cap": rng.randint(64, 300) if ring else pos + s + rng.randint(0, 9),
                "pos": pos, "ragged": rng.random() < 0.5}
    if op == "read":
        B = _log(rng, 1, 64)
        s = _log(rng, 1, 65536 // B)
        return {"op": op, "B": B, "s": s, "d": d, "rd": rd, "cap": s + rng.randint(0, 99), "gather": rng.random() < 0.5, "bf16": rng.random() < 0.5}
    form, h = rng.choice(("window", "csa", "csa", "hca")), rng.choice((64, 64, 64, 32, 16, 8, 5, 128))
    if rng.random() < 0.3 and form != "hca":                # several positions of each sequence in one call
        B, s = _log(rng, 1, 4), _log(rng, 2, 512)
        ctx = _log(rng, 600, 16384)
    else:
        B, s = _log(rng, 1, 32), 1
        ctx = _log(rng, 600, 1 << 20)
    n = WINDOW + (0 if form == "window" else min(TOPK, ctx // 4) if form == "csa" else ctx // 128)
    B = max(1, min(B, MOST_ATTN // (n * h * s)))
    return {"op": op, "form": form, "ctx": ctx, "B": B, "s": s, "h": h, "d": d, "rd": rd, "bf16": rng.random() < 0.5}


# ---- the record of a row ---------------------------------------------------------------------------
def _row_bytes(d, rd):
    return (d - rd + 2 * rd + (d - rd) // GROUP + 15) // 16 * 16


def _parts(cache, d, rd):
    """A cache's codes, rotated channels and scales, as views of the types that they are held in."""
    n, t, g = d - rd, d - rd + 2 * rd, (d - rd) // GROUP
    return cache[..., :n].view(torch.float8_e4m3fn), cache[..., n:t].view(torch.bfloat16), cache[..., t:t + g].view(torch.float8_e8m0fnu)


def _quantise(x, rd):
    """Rows [..., d] in 32 bits -> codes, rotated channels and scale bytes."""
    n = x.shape[-1] - rd
    g = x[..., :n].unflatten(-1, (-1, GROUP))
    m, e = torch.frexp(g.abs().amax(-1).clamp_min(1e-4) * (1.0 / 448.0))
    e = e - (m == 0.5).int()                                 # the least power of two that is not below
    codes = torch.ldexp(g, -e[..., None]).to(torch.float8_e4m3fn).flatten(-2)
    return codes, x[..., n:].bfloat16(), (e + 127).to(torch.uint8)


def _dequantise(cache, d, rd):
    codes, tail, scales = _parts(cache, d, rd)
    x = codes.float().unflatten(-1, (-1, GROUP)) * scales.float()[..., None]
    return torch.cat((x.flatten(-2), tail.float()), -1)


# ---- what a program has in hand before the call ----------------------------------------------------
def _dev():
    return torch.device("cuda", torch.cuda.current_device())


def _rows(g, *shape):
    """Latent rows as the norm before the cache leaves them: N(0, 1) BF16 values, one row in 64 eight times as large,
    some channels nearly silent."""
    x = torch.randn(*shape, generator=g, device=_dev())
    x *= 1 + 7 * (torch.rand(*shape[:-1], 1, generator=g, device=_dev()) < 1 / 64)
    x[..., 5::97] *= 2.0 ** -9
    return x.bfloat16()


def _cache(g, B, cap, d, rd):
    """Caches of B sequences: every row is one of some thousand quantised ones."""
    some = _rows(g, 4096, d).float()
    rec = torch.zeros(4096, _row_bytes(d, rd), dtype=torch.uint8, device=_dev())
    codes, tail, scales = _quantise(some, rd)
    n, t = d - rd, d - rd + 2 * rd
    rec[:, :n], rec[:, n:t], rec[:, t:t + scales.shape[-1]] = codes.view(torch.uint8), tail.view(torch.uint8), scales
    return rec[torch.randint(0, 4096, (B, cap), generator=g, device=_dev())]


def _choice(g, rows, n, k):
    """k different numbers below n for each row, in an order of their own."""
    return torch.rand(rows, n, generator=g, device=_dev()).topk(k, -1).indices.int()


def _positions(c):
    """Of a write: first position and number of rows of every sequence."""
    b = torch.arange(c["B"], device=_dev())
    pos = c["pos"] + (b * 17 % 61 if c["ring"] else b * 0)
    return pos, (c["s"] - (b * 13) % max(1, c["s"] // 3) if c["ragged"] else b * 0 + c["s"]).int()


def prepare(case, seed):
    c, g, dev = dict(case), torch.Generator(device=_dev()).manual_seed(seed), _dev()
    d, rd, B, s = c["d"], c["rd"], c["B"], c["s"]
    if c["op"] == "write":
        x = _rows(g, B, s, d)
        c["x"] = x if c["bf16"] else x.float()
        c["first"], c["counts"] = _positions(c)
        c["cache"] = _cache(g, B, c["cap"], d, rd)           # what the caches hold so far
    elif c["op"] == "read":
        c["cache"] = _cache(g, B, c["cap"], d, rd)
        c["idx"] = None
        if c["gather"]:
            c["idx"] = torch.randint(-c["cap"] // 16 - 1, c["cap"], (B, s), generator=g, device=dev, dtype=torch.int32).clamp_min(-1)
        c["out"] = torch.empty(B, s, d, dtype=torch.bfloat16 if c["bf16"] else torch.float32, device=dev)
    else:
        h, T, form = c["h"], B * s, c["form"]
        na = WINDOW + s - 1                                  # the ring, or the rows of the window before a chunk and its own
        nb = 0 if form == "window" else c["ctx"] // (4 if form == "csa" else 128)
        k = min(TOPK, nb) if form == "csa" else nb
        q = torch.randn(T, h, d, generator=g, device=dev)
        q[:, ::7] *= 4                                       # a few heads look for something
        c["q"] = q.bfloat16() if c["bf16"] else q.bfloat16().float()
        c["sink"] = torch.randn(h, generator=g, device=dev) * 0.5
        c["na"], c["nb"] = na, nb
        c["ring"], c["cache"] = _cache(g, B, na, d, rd), _cache(g, B, nb, d, rd) if nb else None
        t = torch.arange(T, device=dev)[:, None] % s
        idx = torch.empty(T, WINDOW + k, dtype=torch.int32, device=dev)
        idx[:, :WINDOW] = t + torch.arange(WINDOW, device=dev)
        if form == "csa":
            idx[:, WINDOW:] = na + _choice(g, T, nb, k)
        elif form == "hca":                                  # every sequence has entries of its own number
            e = torch.arange(nb, device=dev, dtype=torch.int32)
            have = nb - (torch.arange(B, device=dev)[:, None] * 37) % max(1, nb // 8)
            idx[:, WINDOW:] = torch.where(e < have, na + e, -1)
        if c["ctx"] < 1000:                                  # a young sequence: the window is not full yet
            idx[:, :WINDOW] = torch.where(torch.arange(WINDOW, device=dev) < 128 - c["ctx"] % 100, idx[:, :WINDOW], -1)
        c["idx"], c["o"] = idx, torch.empty(T, h, d, dtype=torch.bfloat16, device=dev)
    return c


# ---- one pass -----------------------------------------------------------------------------------------
def run(c):
    d, rd, B, s = c["d"], c["rd"], c["B"], c["s"]
    if own:
        import apus_b200
        L, st = apus_b200.lib(), torch.cuda.current_stream().cuda_stream
        if c["op"] == "write":
            apus_b200.check(L.apus_cuda_kv8_write_dev(c["x"].data_ptr(), int(c["bf16"]), d, rd, B, s, c["first"].data_ptr(), c["counts"].data_ptr(),
                                                      int(c["ring"]), c["cache"].data_ptr(), c["cap"], c["cap"], st))
        elif c["op"] == "read":
            idx = c["idx"].data_ptr() if c["gather"] else None
            apus_b200.check(L.apus_cuda_kv8_read_dev(c["cache"].data_ptr(), d, rd, c["cap"], c["cap"], B, s, idx, 0, c["out"].data_ptr(), int(c["bf16"]), st))
        else:
            kv_b = c["cache"].data_ptr() if c["nb"] else None
            apus_b200.check(L.apus_cuda_sparse_attn_kv8_dev(c["q"].data_ptr(), int(c["bf16"]), c["sink"].data_ptr(), c["h"], d, rd, c["idx"].data_ptr(),
                                                            c["idx"].shape[1], B * s, s, d ** -0.5, c["ring"].data_ptr(), c["na"], c["na"], kv_b, c["nb"],
                                                            c["nb"], c["o"].data_ptr(), 1, st))
    elif c["op"] == "write":
        codes, tail, scales = _quantise(c["x"].float(), rd)
        row = torch.cat((codes.view(torch.uint8), tail.contiguous().view(torch.uint8), scales), -1)
        t = torch.arange(s, device=row.device)
        at = c["first"][:, None] + t
        use = (t < c["counts"][:, None]) & (t >= c["counts"][:, None] - c["cap"] if c["ring"] else at < c["cap"])
        b, t = use.nonzero(as_tuple=True)                     # a ring keeps the last of the rows that share a place
        c["cache"][b, at[b, t] % c["cap"], :row.shape[-1]] = row[b, t]
    elif c["op"] == "read":
        if c["gather"]:
            rows = c["cache"].gather(1, c["idx"].clamp_min(0).long()[..., None].expand(-1, -1, c["cache"].shape[-1]))
            c["out"] = (_dequantise(rows, d, rd) * (c["idx"] >= 0)[..., None]).to(c["out"].dtype)
        else:
            c["out"] = _dequantise(c["cache"][:, :s], d, rd).to(c["out"].dtype)
    else:
        idx, seq = c["idx"], torch.arange(B * s, device=c["q"].device)[:, None] // s
        both = c["ring"] if not c["nb"] else torch.cat((c["ring"], c["cache"]), 1) if c["nb"] < 65536 else None
        if both is not None:
            rows = both[seq, idx.clamp_min(0).long()]
        else:                                                 # not a copy of a long cache
            rows = torch.cat((c["ring"][seq, idx[:, :WINDOW].clamp_min(0).long()], c["cache"][seq, idx[:, WINDOW:].long() - c["na"]]), 1)
        kv = _dequantise(rows, d, rd)
        x = torch.baddbmm(torch.where(idx >= 0, 0.0, -math.inf)[:, None, :], c["q"].float(), kv.transpose(1, 2), alpha=d ** -0.5)
        m = torch.maximum(x.amax(-1), c["sink"])[..., None]
        p = torch.exp(x - m)
        o = torch.bmm(p, kv) / (p.sum(-1, keepdim=True) + torch.exp(c["sink"][:, None] - m))
        c["o"] = o.bfloat16()
    if c["op"] == "write":
        codes, tail, scales = _parts(c["cache"], d, rd)
        return {"codes": codes, "tail": tail, "scales": scales}
    return c["out"] if c["op"] == "read" else c["o"]


# ---- the definition in 64 bits ---------------------------------------------------------------------------
def _values(cache, d, rd):
    """What records stand for, worked out from their bits."""
    u = cache.to(torch.int32)
    n, t, g = d - rd, d - rd + 2 * rd, (d - rd) // GROUP
    c = u[..., :n]
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e > 0, (8 + m) * torch.exp2(e.double() - 10), m * 2.0 ** -9) * (1 - 2 * (c >> 7))
    v = v * torch.exp2(u[..., t:t + g].double() - 127).repeat_interleave(GROUP, -1)
    tail = ((u[..., n:t:2] + (u[..., n + 1:t:2] << 8)) << 16).view(torch.float32).double()
    return torch.cat((v, tail), -1)


def exact(case, seed):
    c = prepare(case, seed)
    d, rd, B, s = c["d"], c["rd"], c["B"], c["s"]
    if c["op"] == "write":
        codes, tail, scales = [v.double() for v in _parts(c["cache"], d, rd)]
        n, cap = d - rd, c["cap"]
        for b in range(B):
            p0, cnt = int(c["first"][b]), int(c["counts"][b])
            t0 = max(0, cnt - cap) if c["ring"] else 0
            t1 = cnt if c["ring"] else min(cnt, cap - p0)
            if t1 <= t0:
                continue
            at = (p0 + torch.arange(t0, t1, device=codes.device)) % cap
            x = c["x"][b, t0:t1].double()
            grp = x[:, :n].reshape(t1 - t0, -1, GROUP)
            sc = torch.exp2(torch.ceil(torch.log2(torch.clamp(grp.abs().max(-1).values, min=1e-4) / 448)))
            codes[b, at] = (grp / sc[..., None]).reshape(t1 - t0, n)
            tail[b, at] = x[:, n:]
            scales[b, at] = sc
        return {"codes": codes, "tail": tail, "scales": scales}
    if c["op"] == "read":
        if not c["gather"]:
            return _values(c["cache"][:, :s], d, rd)
        out = torch.zeros(B, s, d, dtype=torch.float64, device=c["cache"].device)
        b, t = torch.nonzero(c["idx"] >= 0, as_tuple=True)
        out[b, t] = _values(c["cache"][b, c["idx"][b, t].long()], d, rd)
        return out
    o = torch.empty(B * s, c["h"], d, dtype=torch.float64, device=c["q"].device)
    for r in range(B * s):
        i = c["idx"][r][c["idx"][r] >= 0].long()
        rec = c["ring"][r // s][i[i < c["na"]]]
        if c["nb"]:
            rec = torch.cat((rec, c["cache"][r // s][i[i >= c["na"]] - c["na"]]))
        kv = _values(rec, d, rd)
        x = (c["q"][r].double() @ kv.T) * d ** -0.5
        x = torch.cat((x, c["sink"].double()[:, None]), 1)   # the sink is one more candidate, without a value
        o[r] = torch.softmax(x, 1)[:, :-1] @ kv
    return o


# ---- what a pass cannot do without --------------------------------------------------------------------------
def work(case):
    d, rd, B, s = case["d"], case["rd"], case["B"], case["s"]
    rec, esz = d - rd + 2 * rd + (d - rd) // GROUP, 2 if case.get("bf16") else 4
    if case["op"] == "write":
        rows = B * min(s, case["cap"]) if case["ring"] else B * s
        if case["ragged"]:
            rows = sum(min(s - (b * 13) % max(1, s // 3), case["cap"] if case["ring"] else s) for b in range(B))
        return {"bytes": rows * (d * esz + rec) + 12 * B, "flops": rows * d}
    if case["op"] == "read":
        return {"bytes": B * s * (rec + d * esz + (4 if case["gather"] else 0)), "flops": B * s * d}
    h, T, form = case["h"], B * s, case["form"]
    nb = 0 if form == "window" else case["ctx"] // (4 if form == "csa" else 128)
    k = min(TOPK, nb) if form == "csa" else nb
    win = 128 - case["ctx"] % 100 if case["ctx"] < 1000 else WINDOW
    have = [k - (b * 37) % max(1, nb // 8) if form == "hca" else k for b in range(B)]
    n = sum(win + v for v in have) * s                       # candidates over all query rows
    rows = sum(win + s - 1 + min(nb, v * s) for v in have)   # different cache rows
    return {"bytes": rows * rec + T * h * d * (esz + 2) + 4 * T * (WINDOW + k) + 4 * h, "flops": 4.0 * n * h * d}
