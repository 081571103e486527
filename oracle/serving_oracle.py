"""Plain restatements in 64 bits of what a decoder over fp16 caches is served with (numpy; used by the tests only):
attention behind a shared prefix, the cache that evicts by accumulated attention weight, rules on logits."""
import numpy as np


def _softmax(s):
    """Rows of scores (-inf: not seen); a row that sees nothing gives 0."""
    m = s.max(-1, keepdims=True) if s.shape[-1] else np.zeros(s.shape[:-1] + (1,))
    p = np.exp(s - np.where(np.isfinite(m), m, 0.0))
    total = p.sum(-1, keepdims=True)
    return p / np.where(total == 0, 1.0, total)


def prefix_attention(q, kp, vp, kc, vc, lens, new, scale, k_new=None, v_new=None):
    """q [T, heads, D]; new: tokens of each sequence.  Returns (out, sum P |v|, caches after): tokens behind the last
    sequence's are NaN in out."""
    q, kp, vp = (x.astype(np.float64) for x in (q, kp, vp))
    kc, vc = kc.copy(), vc.copy()
    t, heads, d = q.shape
    b, h, room = kc.shape[:3]
    share = heads // h
    out, size = np.full(q.shape, np.nan), np.zeros(q.shape)
    at = 0
    for i in range(b):
        before = max(lens[i], 0) - new[i]
        if k_new is not None:
            for j in range(new[i]):
                if 0 <= before + j < room:
                    kc[i, :, before + j], vc[i, :, before + j] = k_new[at + j], v_new[at + j]
        for j in range(new[i]):
            seen = min(max(before + j + 1, 0), room)
            for g in range(heads):
                k = np.concatenate([kp[g // share], kc[i, g // share, :seen].astype(np.float64)])
                v = np.concatenate([vp[g // share], vc[i, g // share, :seen].astype(np.float64)])
                p = _softmax((k @ q[at + j, g] * scale)[None])[0]
                out[at + j, g], size[at + j, g] = p @ v, p @ np.abs(v)
        at += new[i]
    return out, size, kc, vc


def order(weight):
    """Weights in the order that they are compared in: a NaN is the lowest."""
    return np.where(np.isnan(weight), -np.inf, weight), ~np.isnan(weight)


def evict_step(q, k_new, v_new, kc, vc, weight, position, seen, scale, first, last):
    """Returns (out, sum P |v|, slot, kc, vc, weight, position) after one token of each sequence."""
    kc, vc, weight, position = kc.copy(), vc.copy(), weight.astype(np.float64), position.copy()
    b, heads, d = q.shape
    h, room = kc.shape[1:3]
    share = heads // h
    out, size, slot = np.zeros(q.shape), np.zeros(q.shape), np.full((b, h), -1, np.int32)
    for i in range(b):
        n = int(seen[i])
        if n <= 0:
            continue
        for j in range(h):
            at = n - 1
            if n > room:
                free = (position[i, j] >= first) & (position[i, j] < n - last)
                value, number = order(weight[i, j])
                rank = sorted((bool(number[r]), value[r], r) for r in range(room) if free[r])
                at = rank[0][2] if rank else 0
            slot[i, j] = at
            kc[i, j, at], vc[i, j, at], weight[i, j, at], position[i, j, at] = k_new[i, j], v_new[i, j], 0.0, n - 1
            used = min(n, room)
            qs = q[i, j * share:(j + 1) * share].astype(np.float64)
            p = _softmax(qs @ kc[i, j, :used].astype(np.float64).T * scale)
            v = vc[i, j, :used].astype(np.float64)
            out[i, j * share:(j + 1) * share], size[i, j * share:(j + 1) * share] = p @ v, p @ np.abs(v)
            weight[i, j, :used] += p.sum(0)
    return out, size, slot, kc, vc, weight, position


def attention_weights(q, k, lens, scale, window=None):
    b, heads, s, d = q.shape
    h = k.shape[1]
    share = heads // h
    w = np.zeros((b, h, s))
    for i in range(b):
        n = min(max(int(lens[i]), 0), s)
        first = max(0, n - window) if window else 0
        hidden = np.arange(n)[None] > np.arange(first, n)[:, None]
        for g in range(heads):
            x = q[i, g, first:n].astype(np.float64) @ k[i, g // share, :n].astype(np.float64).T * scale
            w[i, g // share, :n] += _softmax(np.where(hidden, -np.inf, x)).sum(0) if n else 0.0
    return w


def keep_rows(weight, n, room, first, last):
    """The rows of one head that stay, ascending."""
    if n <= room:
        return list(range(n))
    value, number = order(weight[:n])
    forced = [r for r in range(n) if r < first or r >= n - last]
    others = sorted((r for r in range(n) if first <= r < n - last), key=lambda r: (not number[r], -value[r], r))
    return sorted((forced + others)[:room])


def logit_rules(x, ids=None, lengths=None, generated=None, repetition=None, presence=None, frequency=None, bias_ids=None, bias=None,
                mask=None, dtype=np.float64):
    """The rules in `dtype` (np.float32: step by step as the kernel rounds; np.float64: exactly)."""
    out = x.astype(dtype)
    m, v = x.shape
    for i in range(m):
        if ids is not None and (repetition is not None or presence is not None or frequency is not None):
            n = ids.shape[1] if lengths is None else min(max(int(lengths[i]), 0), ids.shape[1])
            start = 0 if generated is None else int(generated[i])
            text = [(int(t), j >= start) for j, t in enumerate(ids[i, :n]) if 0 <= t < v]
            count = {}
            for t, made in text:
                count[t] = count.get(t, 0) + made
            for t, c in count.items():
                if repetition is not None:
                    r = dtype(repetition[i])
                    out[i, t] = out[i, t] / r if out[i, t] > 0 else out[i, t] * r
                if c and frequency is not None:
                    out[i, t] = out[i, t] - dtype(dtype(frequency[i]) * dtype(c))
                if c and presence is not None:
                    out[i, t] = out[i, t] - dtype(presence[i])
        if bias is not None:
            for t, value in {int(t): value for t, value in zip(bias_ids[i], bias[i]) if 0 <= t < v}.items():
                out[i, t] = out[i, t] + dtype(value)
        if mask is not None:
            words = mask[i if mask.shape[0] > 1 else 0].view(np.uint32)
            e = np.arange(v)
            out[i, ((words[e // 32] >> (e % 32).astype(np.uint32)) & 1) == 0] = -np.inf
    return out


def best_token(y):
    """The lowest of the largest (-inf among them), NaN never; 0 where all are."""
    best = []
    for row in y.astype(np.float64):
        tokens = np.flatnonzero(~np.isnan(row))
        best.append(tokens[row[tokens].argmax()] if len(tokens) else 0)
    return np.array(best, dtype=np.int64)
