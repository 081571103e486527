"""CPU restatement of the 4-bit key/value cache: its record layout, quantisation, attention and page selection (numpy,
64 bits; the quantisation in the fp32 steps that define it).  Used by the tests only."""
import numpy as np

PAGE = 64


def record_bytes(d, g):
    return 68 * d + 512 * (d // g)


def places(d, g):
    """For row r and element e of a record: byte and shift of the key's and of the value's code, byte of the key's and of
    the value's scale (the minimum lies 8 bytes behind it)."""
    out = {n: np.zeros((PAGE, d), dtype=np.int64) for n in ("kb", "ks", "vb", "vs", "ksm", "vsm")}
    for r in range(PAGE):
        for word in range(d // 8):
            chunk, w = divmod(word, d // 32)
            for n in range(8):
                e = 64 * (w // 2) + 32 * (n % 2) + 8 * chunk + 4 * (n // 2 % 2) + 2 * (w % 2) + n // 4
                out["kb"][r, e] = r * (d // 2) + 4 * word + n // 2
                out["ks"][r, e] = 4 * (n % 2)
                e = 16 * n + word if d == 128 else 16 * (n % 4) + 8 * (n // 4) + word
                out["vb"][r, e] = 32 * d + (r // 4) * 2 * d + 16 * word + 4 * (r % 4) + n // 2
                out["vs"][r, e] = 4 * (n % 2)
        e = np.arange(d)
        out["ksm"][r] = 64 * d + (e // g) * 256 + (r // 4) * 16 + (r % 4) * 2
        out["vsm"][r] = out["ksm"][r] + 256 * (d // g)
    return out


def _half(rec, at):
    return rec[..., np.stack([at, at + 1], -1)].copy().view(np.float16)[..., 0]


def read(rec, d, g):
    """Records uint8 [..., record] -> dict of codes (int), scales and minima (fp16), [..., 64, D] each, and bounds."""
    p = places(d, g)
    rec = np.ascontiguousarray(rec)
    return {"kc": (rec[..., p["kb"]].astype(np.int32) >> p["ks"]) & 15, "vc": (rec[..., p["vb"]].astype(np.int32) >> p["vs"]) & 15,
            "ks": _half(rec, p["ksm"]), "km": _half(rec, p["ksm"] + 8), "vs": _half(rec, p["vsm"]), "vm": _half(rec, p["vsm"] + 8),
            "bounds": rec[..., -4 * d:].copy().view(np.float16).reshape(rec.shape[:-1] + (2, d))}


def quantise(x, g):
    """fp16 [..., D] -> codes, scales, minima (the latter two fp16, repeated over their group)."""
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        y = np.asarray(x, dtype=np.float16).astype(np.float32).reshape(x.shape[:-1] + (-1, g))
        lo, hi = y.min(-1, keepdims=True), y.max(-1, keepdims=True)
        s = ((hi - lo) / np.float32(15)).astype(np.float16)
        c = np.rint((y - lo) / s.astype(np.float32))
        c = np.where((s > 0) & ~np.isnan(c), np.clip(c, 0, 15), 0)
    rep = lambda t: np.broadcast_to(t, y.shape).reshape(x.shape)
    return c.reshape(x.shape).astype(np.int32), rep(s), rep(lo.astype(np.float16))


def values(c, s, m):
    return s.astype(np.float64) * c + m.astype(np.float64)


class Rows:
    """The rows of one sequence and key/value head: K and V in 64 bits, and what the tolerance needs of them."""

    def __init__(self, pool, pages, n, head, d, g):
        f = read(pool[np.asarray(pages, dtype=np.int64), head], d, g)
        flat = lambda t: t.reshape(-1, d)[:n]
        self.k, self.v = flat(values(f["kc"], f["ks"], f["km"])), flat(values(f["vc"], f["vs"], f["vm"]))
        self.k_abs = flat(f["ks"].astype(np.float64) * f["kc"] + np.abs(f["km"].astype(np.float64)))
        self.v_mid = flat(np.abs(f["vs"].astype(np.float64) * (f["vc"] - 8)))
        self.v_rest = flat(np.abs(f["vs"].astype(np.float64) * 8 + f["vm"].astype(np.float64)))


def attend(rows, q, scale, seen, middles=0.0):
    """q fp64 [D] over the rows named by `seen` (indices, with repetition): (out, tolerance) [D] in 64 bits.

    Tolerance.  P' = P s is rounded to fp16 before it meets code - 8: eps/2 = 2^-11 of every term (no allowance is made for
    denormal ones, below 2^-25 of the largest scale).  A probability is off by
    twice the error of its exponent (numerator and sum): the score's fp32 sums of D + 16 terms, each rounding (also towards
    zero) 2^-23 of sum |q| (s code + |m|), and 2^-20 for the exponential, its argument in base 2 and the joining of partial
    sums.  fp32 sums of the result: the terms P s (code - 8) of every 32 rows are added to what there is, 33 additions
    that each round (towards zero as well) 2^-23 of a partial sum of at most sum P s |code - 8| over those rows; the sums are in
    one chain of n / 32, 8 additions join partial sums.  The output's own rounding is 2^-11 of it, or 2^-25
    where it is denormal.  middles: what m + 8 s is rounded by, of itself (2^-11
    for fp16), where it is held in fewer bits."""
    if len(seen) == 0:
        return np.zeros(rows.k.shape[1]), np.zeros(rows.k.shape[1])
    d = rows.k.shape[1]
    k, v = rows.k[seen], rows.v[seen]
    s = k @ q * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    out = p @ v
    mid, rest = p @ rows.v_mid[seen], p @ rows.v_rest[seen]
    dscore = (d + 16) * 2.0 ** -23 * np.max(rows.k_abs[seen] @ np.abs(q)) * abs(scale) + 2.0 ** -20
    chain = (8 + min(len(seen), 4096) / 32) * 2.0 ** -23
    tol = 2.0 ** -11 * (np.abs(out) + mid) + (2 * dscore + chain) * (mid + rest) + 2.0 ** -24
    return out, tol + 33 * 2.0 ** -23 * mid + middles * rest


def select(bounds, q, count, keep_first, keep_last):
    """bounds fp16 [pages, 2, D], q fp16 [heads, D] of one key/value head -> places, ascending."""
    n = bounds.shape[0]
    if n <= count:
        return list(range(n))
    hi, lo = bounds[:, 0].astype(np.float64), bounds[:, 1].astype(np.float64)
    q = q.astype(np.float64)
    with np.errstate(invalid="ignore"):
        score = (np.maximum(q, 0) @ hi.T + np.minimum(q, 0) @ lo.T)
    score = np.where(np.isnan(score), -np.inf, score).max(0)
    key = lambda j: (0 if j < keep_first or j >= n - keep_last else 1, -score[j], j)
    return sorted(sorted(range(n), key=key)[:count])
