"""A key/value cache held in 4 bits, and what reads and writes it, as cases that can be timed one by one.

The cache is a pool of pages of 64 rows.  pool [pages, kv_heads, record] uint8 holds one record per page and head:

    keys      64 x D codes of 4 bits, row by row: uint32 [64][4][D / 32]; nibble n (from the least significant) of
              word w of chunk c is element 64 (w / 2) + 32 (n % 2) + 8 c + 4 (n / 2 % 2) + 2 (w % 2) + n / 4
    values    64 x D codes, uint32 [16][D / 8][4]: row 4 a + t, word w; nibble n is element 16 n + w for D = 128 and
              16 (n % 4) + 8 (n / 4) + w for D = 64
    scales    fp16 [D / g][16][2][4] of the keys, then of the values: scale and minimum of row 4 a + t by group of g
    bounds    fp16 [2][D]: the largest and the smallest key of the page, element by element, as it was given

A row's group reads as scale * code + minimum, minimum = min(x), scale = fp16((max(x) - min(x)) / 15), code =
round((x - minimum) / scale) in 0..15, all in fp32.  pages int32 [sequences, width] names the pages of a sequence in
their order, lengths int32 [sequences] counts its rows, those of the present call among them.

Kinds of cases (a case is a dict of plain values):

    append   quantise the keys and values of new tokens into the cache
    attend   causal attention of each sequence's last tokens over its cached rows
    sparse   for one token of each sequence: score every page by the bound that its largest and smallest keys give
             the query, keep the best, attend over those
    copy     copy pages inside the pool of every layer (a fork's last page, a pool made compact)

listed() holds the cases themselves, draw() makes more over the same ranges.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
PAGE = 64


def _kv4():
    package = os.path.join(os.getcwd(), "sparse-quant_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from sqamd import kv4
    return kv4


def listed():
    return [
        # a decode step of 8 sequences of 32 heads writes its rows: launch latency
        {"name": "append_step_8", "kind": "append", "batch": 8, "kv_heads": 32, "dim": 128, "group": 64, "tokens": 1,
         "rows": 640, "ragged": False},
        # prompts of different lengths into the cache, some behind rows that are there
        {"name": "append_prompts", "kind": "append", "batch": 12, "kv_heads": 8, "dim": 128, "group": 32, "tokens": 2048,
         "rows": 2500, "ragged": True},
        # interactive decoding: one sequence, shared heads
        {"name": "attend_1x640", "kind": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "dim": 128, "group": 64,
         "tokens": 1, "rows": 640, "ragged": False},
        # the decode step of an OPT-6.7B layer at batch 8
        {"name": "attend_8x640", "kind": "attend", "batch": 8, "heads": 32, "kv_heads": 32, "dim": 128, "group": 64,
         "tokens": 1, "rows": 640, "ragged": False},
        # serving: 64 sequences of very different lengths
        {"name": "attend_64_ragged", "kind": "attend", "batch": 64, "heads": 32, "kv_heads": 8, "dim": 128, "group": 128,
         "tokens": 1, "rows": 8192, "ragged": True},
        # one long context
        {"name": "attend_1x131072", "kind": "attend", "batch": 1, "heads": 64, "kv_heads": 8, "dim": 128, "group": 64,
         "tokens": 1, "rows": 131072, "ragged": False},
        # drafted tokens verified together, heads of 64
        {"name": "attend_16x5tok", "kind": "attend", "batch": 16, "heads": 16, "kv_heads": 4, "dim": 64, "group": 32,
         "tokens": 5, "rows": 3333, "ragged": False},
        # a long prompt in chunks: the chunk's rows see what came before them
        {"name": "attend_chunk_2x1024", "kind": "attend", "batch": 2, "heads": 32, "kv_heads": 8, "dim": 128, "group": 64,
         "tokens": 1024, "rows": 16384, "ragged": True},
        # one sequence decoding over the pages that matter to it
        {"name": "sparse_1x8000", "kind": "sparse", "batch": 1, "heads": 32, "kv_heads": 8, "dim": 128, "group": 64,
         "rows": 8000, "ragged": False, "count": 16},
        # a batch of long contexts
        {"name": "sparse_8x32768", "kind": "sparse", "batch": 8, "heads": 32, "kv_heads": 8, "dim": 128, "group": 64,
         "rows": 32768, "ragged": True, "count": 64},
        # a fork: its last, part-filled page in all layers
        {"name": "copy_fork", "kind": "copy", "layers": 32, "pool": 16, "kv_heads": 8, "dim": 128, "group": 64, "moved": 1},
        # a pool made compact
        {"name": "copy_compact", "kind": "copy", "layers": 8, "pool": 384, "kv_heads": 8, "dim": 128, "group": 64,
         "moved": 160},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "sparse", "copy"])
    dim = rng.choice([64, 128, 128])
    case = {"kind": kind, "dim": dim, "group": rng.choice([g for g in (32, 64, 128) if g <= dim])}
    if kind == "copy":
        case["kv_heads"] = rng.choice([1, 2, 4, 8, 8, 32])
        case["layers"] = rng.randint(1, 32)
        case["pool"] = max(4, min(_log_int(rng, 4, 384), 8 * 384 * 8 // (case["layers"] * case["kv_heads"])))
        case["moved"] = rng.randint(1, case["pool"] // 2)
        return case
    case["ragged"] = rng.random() < 0.5
    case["kv_heads"] = rng.choice([1, 2, 3, 4, 8, 8, 32])
    if kind == "append":
        case["tokens"] = rng.choice([1, _log_int(rng, 1, 2048)])
        case["batch"] = min(_log_int(rng, 1, 128), max(1, 12 * 2048 * 8 // (case["tokens"] * case["kv_heads"])))
        case["rows"] = case["tokens"] + _log_int(rng, 1, 4096) - 1
        return case
    case["heads"] = case["kv_heads"] * rng.choice([1, 2, 4, 4, 5, 8] if case["kv_heads"] <= 8 else [1, 2])
    if kind == "sparse":
        case["rows"] = _log_int(rng, 64, 65536)
        case["batch"] = max(1, min(_log_int(rng, 1, 64), 8 * 32768 * 8 // (case["rows"] * case["kv_heads"])))
        case["count"] = _log_int(rng, 2, 64)
        return case
    case["tokens"] = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 8, 1024)])
    most = 16384 - 1024 if case["tokens"] > 8 else 65536 if case["kv_heads"] <= 8 else 32768
    case["rows"] = case["tokens"] + _log_int(rng, 1, most) - 1
    room = 131072 * 8 // (case["rows"] * case["kv_heads"])
    if case["tokens"] > 8:
        room = min(room, 16, 32 * 1024 * 16384 // (case["tokens"] * case["rows"] * case["heads"]))
    case["batch"] = max(1, min(_log_int(rng, 1, 128), room))
    return case


def _sizes(case):
    """Rows and new tokens of every sequence: by the case alone."""
    b, rows, tokens = case["batch"], case["rows"], case.get("tokens", 1)
    if not case["ragged"]:
        return [rows] * b, [tokens] * b
    rng = random.Random("%d %d %d" % (b, rows, tokens))
    new = [tokens if i == 0 or tokens == 1 else _log_int(rng, 1, tokens) for i in range(b)]
    lens = [rows if i == 0 else max(new[i], _log_int(rng, max(1, rows // 16), rows)) for i in range(b)]
    return lens, new


def _record(case):
    return 68 * case["dim"] + 512 * (case["dim"] // case["group"])


def _pool(case, shape, gen):
    """A pool of random records: codes of all values, scales and minima as of rows of normal numbers."""
    d, groups = case["dim"], case["dim"] // case["group"]
    pool = torch.randint(0, 256, shape + (_record(case),), dtype=torch.uint8, device=DEV, generator=gen)
    s = torch.rand(shape + (2 * groups * 16, 1, 4), device=DEV, generator=gen) * 0.2 + 0.2
    m = torch.randn(shape + (2 * groups * 16, 1, 4), device=DEV, generator=gen) * 0.3 - 7.5 * s
    pool[..., 64 * d:64 * d + 512 * groups] = torch.cat([s, m], -2).half().flatten(-3).view(torch.uint8)
    hi = 2.0 + 0.5 * torch.randn(shape + (1, d), device=DEV, generator=gen)
    lo = -2.0 + 0.5 * torch.randn(shape + (1, d), device=DEV, generator=gen)
    pool[..., 64 * d + 512 * groups:] = torch.cat([torch.maximum(hi, lo), torch.minimum(hi, lo)], -2).half().flatten(
        -2).view(torch.uint8)
    return pool


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    state = {"case": case}
    if case["kind"] == "copy":
        state["pool"] = _pool(case, (case["layers"], case["pool"], case["kv_heads"]), gen)
        order = torch.randperm(case["pool"], device=DEV, generator=gen).int()
        state["src"], state["dst"] = order[:case["moved"]].clone(), order[case["moved"]:2 * case["moved"]].clone()
        return state
    lens, new = _sizes(case)
    counts = [(n + PAGE - 1) // PAGE for n in lens]
    total = sum(counts)
    state["pool"] = _pool(case, (total + 3, case["kv_heads"]), gen)
    order = torch.randperm(total + 3, device=DEV, generator=gen).int()
    width = max(counts)
    pages = torch.zeros((case["batch"], width), dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(counts):
        pages[i, :n] = order[at:at + n]
        at += n
    state["pages"], state["host_lengths"], state["host_new"] = pages, lens, new
    state["lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state["host_starts"] = starts
    equal = min(new) == max(new)
    state["starts"] = None if equal else torch.tensor(starts, dtype=torch.int32, device=DEV)
    t, d = starts[-1], case["dim"]
    if case["kind"] == "append":
        # keys and values as a fused projection leaves them; keys have a few large elements
        kv = torch.randn((t, 2, case["kv_heads"], d), device=DEV, generator=gen)
        kv[:, 0] *= 1.0 + 4.0 * (torch.rand((case["kv_heads"], d), device=DEV, generator=gen) > 0.97)
        kv = kv.half()
        state["k"], state["v"] = kv[:, 0], kv[:, 1]
    else:
        state["q"] = torch.randn((t, case["heads"], d), device=DEV, generator=gen).half()
        state["scale"] = 1.0 / math.sqrt(d)
    return state


# ---------------------------------------------------------------------------------------------- the plain forms

def _codes(rec, d):
    """Codes of keys and values of records uint8 [..., record] -> int32 [..., 64, D] each."""
    shift = torch.arange(0, 32, 4, dtype=torch.int32, device=rec.device)
    lead = rec.shape[:-1]
    k = rec[..., :32 * d].contiguous().view(torch.int32).view(lead + (64, 4, d // 64, 2, 1))
    k = ((k >> shift) & 15).view(lead + (64, 4, d // 64, 2, 2, 2, 2))  # [row, c, w / 2, w % 2, n / 4, n / 2 % 2, n % 2]
    n = len(lead)
    k = k.permute(tuple(range(n + 1)) + (n + 2, n + 6, n + 1, n + 5, n + 3, n + 4)).reshape(lead + (64, d))
    v = rec[..., 32 * d:64 * d].contiguous().view(torch.int32).view(lead + (16, d // 8, 4, 1))
    v = (v >> shift) & 15  # [a, w, t, n]
    if d == 128:
        v = v.permute(tuple(range(n + 1)) + (n + 2, n + 3, n + 1))
    else:
        v = v.view(lead + (16, 8, 4, 2, 4)).permute(tuple(range(n + 1)) + (n + 2, n + 4, n + 3, n + 1))
    return k, v.reshape(lead + (64, d))


def _scales(rec, d, g):
    """Scales and minima of keys and values, fp32 [..., 64, D] each."""
    lead, groups = rec.shape[:-1], d // g
    sm = rec[..., 64 * d:64 * d + 512 * groups].contiguous().view(torch.float16).view(lead + (2, groups, 16, 2, 4)).float()
    n = len(lead)
    sm = sm.permute(tuple(range(n + 1)) + (n + 3, n + 2, n + 4, n + 1)).reshape(lead + (2, 2, 64, groups))
    sm = sm.repeat_interleave(g, -1)
    return [sm[..., i, j, :, :] for i in (0, 1) for j in (0, 1)]


def _values(rec, d, g):
    k, v = _codes(rec, d)
    ks, km, vs, vm = _scales(rec, d, g)
    return ks * k + km, vs * v + vm


def _quantise(x, g):
    """fp16 [T, H, D] -> codes int32 [T, H, D], scale and minimum fp16 [T, H, D / g]."""
    y = x.float().unflatten(-1, (-1, g))
    low = y.amin(-1, keepdim=True)
    # (a tensor of 15: torch multiplies by the rounded reciprocal of a plain number)
    s = ((y.amax(-1, keepdim=True) - low) / torch.full_like(low, 15.0)).half()
    c = torch.where(s > 0, (y - low) / s.float(), torch.zeros_like(y)).round().clamp(0, 15).int()
    return c.flatten(-2), s[..., 0], low[..., 0].half()


def _words(nibbles):
    """int32 [..., 8] nibbles from the least significant -> uint8 [..., 4]."""
    pairs = nibbles.view(nibbles.shape[:-1] + (4, 2))
    return (pairs[..., 0] | (pairs[..., 1] << 4)).to(torch.uint8)


def _append_plain(st):
    case, pool, k, v = st["case"], st["pool"], st["k"], st["v"]
    d, g, h = case["dim"], case["group"], case["kv_heads"]
    groups, dev = d // g, pool.device
    page, slot = [], []
    for b, (n, new) in enumerate(zip(st["host_lengths"], st["host_new"])):
        pos = torch.arange(n - new, n, device=dev)
        page.append(st["pages"][b].long()[pos // PAGE])
        slot.append(pos % PAGE)
    page, slot = torch.cat(page), torch.cat(slot)
    kc, ks, km = _quantise(k, g)
    vc, vs, vm = _quantise(v, g)
    t = k.shape[0]
    # keys: a row is d / 2 adjacent bytes
    kw = _words(kc.view(t, h, d // 64, 2, 4, 2, 2, 2).permute(0, 1, 4, 2, 6, 7, 5, 3).reshape(t, h, -1, 8)).flatten(2)
    view = pool.as_strided((pool.shape[0], h, 64, d // 2), (pool.stride(0), pool.stride(1), d // 2, 1))
    view[page, :, slot] = kw
    # values: word w of row 4 a + t
    if d == 128:
        vw = _words(vc.view(t, h, 8, 16).permute(0, 1, 3, 2))
    else:
        vw = _words(vc.view(t, h, 4, 2, 8).permute(0, 1, 4, 3, 2).reshape(t, h, 8, 8))
    view = pool.as_strided((pool.shape[0], h, 16, d // 8, 4, 4), (pool.stride(0), pool.stride(1), 2 * d, 16, 4, 1),
                           pool.storage_offset() + 32 * d)
    view[page, :, slot // 4, :, slot % 4] = vw
    half = pool.view(torch.float16)
    for i, (s, m) in enumerate(((ks, km), (vs, vm))):
        view = half.as_strided((half.shape[0], h, groups, 16, 2, 4), (half.stride(0), half.stride(1), 128, 8, 4, 1),
                               half.storage_offset() + 32 * d + 128 * groups * i)
        view[page, :, :, slot // 4, 0, slot % 4] = s
        view[page, :, :, slot // 4, 1, slot % 4] = m
    # bounds: a page that gets its row 0 starts anew
    fresh = page[slot == 0]
    view = half.as_strided((half.shape[0], h, 2, d), (half.stride(0), half.stride(1), d, 1),
                           half.storage_offset() + 32 * d + 256 * groups)
    bounds = view.float()
    bounds[fresh, :, 0], bounds[fresh, :, 1] = -math.inf, math.inf
    index = page.view(-1, 1, 1).expand(t, h, d)
    bounds[:, :, 0] = bounds[:, :, 0].scatter_reduce(0, index, k.float(), "amax")
    bounds[:, :, 1] = bounds[:, :, 1].scatter_reduce(0, index, k.float(), "amin")
    view[page] = bounds.half()[page]
    out = [(s.float().repeat_interleave(g, -1) * c + m.float().repeat_interleave(g, -1)).half()
           for c, s, m in ((kc, ks, km), (vc, vs, vm))]
    return {"k": out[0], "v": out[1], "pool": pool}


def _softmax_product(q, k, v, scale, seen):
    """q [H, R, D], k and v [H, N, D] fp32, seen [R, N] or None: softmax(q k^T scale) v, 0 where nothing is seen."""
    s = torch.matmul(q, k.transpose(-1, -2)) * scale
    if seen is not None:
        s = s.masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    l = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(l == 0, torch.ones_like(l), l)


def _attend_plain(st):
    case, q = st["case"], st["q"]
    d, g, h = case["dim"], case["group"], case["kv_heads"]
    share = case["heads"] // h
    out = torch.empty_like(q)
    for b, (n, new) in enumerate(zip(st["host_lengths"], st["host_new"])):
        rec = st["pool"][st["pages"][b, :(n + PAGE - 1) // PAGE].long()].transpose(0, 1)
        k, v = (x.flatten(1, 2)[:, :n] for x in _values(rec, d, g))
        at = st["host_starts"][b]
        rows = q[at:at + new].float().view(new, h, share, d).permute(1, 0, 2, 3).reshape(h, new * share, d)
        seen = None
        if new > 1:
            pos = torch.arange(n - new, n, device=q.device).repeat_interleave(share)
            seen = torch.arange(n, device=q.device)[None] <= pos[:, None]
        o = _softmax_product(rows, k, v, st["scale"], seen)
        out[at:at + new] = o.view(h, new, share, d).permute(1, 0, 2, 3).reshape(new, -1, d).half()
    return out


def _select_plain(st, b, first=1, last=1):
    case, n = st["case"], st["host_lengths"][b]
    d, groups, h = case["dim"], case["dim"] // case["group"], case["kv_heads"]
    count, total = case["count"], (n + PAGE - 1) // PAGE
    rec = st["pool"][st["pages"][b, :total].long()]
    hi, lo = rec[..., 64 * d + 512 * groups:].contiguous().view(torch.float16).view(total, h, 1, 2, d).double().unbind(-2)
    q = st["q"][b].double().view(1, h, -1, d)
    score = torch.maximum(q * hi, q * lo).sum(-1).amax(-1)  # [pages, kv heads], in 64 bits: neighbours in rank differ little
    score[:first] = math.inf
    score[total - last:] = math.inf
    best = torch.sort(score, dim=0, descending=True, stable=True).indices[:count].sort(0).values
    chosen = torch.full((h, count), -1, dtype=torch.int32, device=rec.device)
    chosen[:, :best.shape[0]] = best.t().int()
    return chosen


def _sparse_plain(st):
    case, q = st["case"], st["q"]
    d, g, h = case["dim"], case["group"], case["kv_heads"]
    out, chosen = torch.empty_like(q), []
    for b, n in enumerate(st["host_lengths"]):
        sel = _select_plain(st, b)
        chosen.append(sel)
        used = min(case["count"], (n + PAGE - 1) // PAGE)
        sel = sel[:, :used].long()
        rec = st["pool"][st["pages"][b].long()[sel], torch.arange(h, device=q.device)[:, None]]  # [h, used, record]
        k, v = (x.flatten(1, 2) for x in _values(rec, d, g))
        inside = (sel[..., None] * PAGE + torch.arange(PAGE, device=q.device)).flatten(1) < n
        o = _softmax_product(q[b].float().view(h, -1, d), k, v, st["scale"], inside[:, None])
        out[b] = o.view(-1, d).half()
    return {"pages": torch.stack(chosen), "out": out}


def _copy_plain(st):
    st["pool"][:, st["dst"].long()] = st["pool"][:, st["src"].long()]
    return st["pool"]


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"append": _append_plain, "attend": _attend_plain, "sparse": _sparse_plain, "copy": _copy_plain}[kind](state)
    kv4 = _kv4()
    if kind == "append":
        k, v = kv4.append(state["k"], state["v"], state["pool"], state["pages"], state["lengths"], starts=state["starts"],
                          values=True)
        return {"k": k, "v": v, "pool": state["pool"]}
    if kind == "attend":
        return kv4.attention(state["q"], state["pool"], state["pages"], state["lengths"], state["scale"],
                             starts=state["starts"])
    if kind == "sparse":
        chosen = kv4.select_pages(state["q"], state["pool"], state["pages"], state["lengths"], state["case"]["count"])
        out = kv4.attention(state["q"], state["pool"], state["pages"], state["lengths"], state["scale"], selected=chosen)
        return {"pages": chosen, "out": out}
    kv4.copy_pages(state["pool"], state["src"], state["dst"])
    return state["pool"]


def work(case):
    d, groups = case["dim"], case["dim"] // case["group"]
    row = d + 8 * groups  # bytes of a cached row of one head, key and value
    if case["kind"] == "copy":
        return {"bytes": 2 * case["moved"] * case["layers"] * case["kv_heads"] * _record(case) + 8 * case["moved"],
                "flops": 0}
    lens, new = _sizes(case)
    h = case["kv_heads"]
    if case["kind"] == "append":
        # rows read and written, their values written, bounds of touched pages; comparisons, differences, quotients
        touched = sum((n - 1) // PAGE - (n - t) // PAGE + 1 for n, t in zip(lens, new))
        return {"bytes": sum(new) * h * (8 * d + row) + touched * h * 4 * d, "flops": sum(new) * h * 2 * d * 6}
    if case["kind"] == "sparse":
        pages = [(n + PAGE - 1) // PAGE for n in lens]
        seen = [n if p <= case["count"] else (case["count"] - 1) * PAGE + (n - 1) % PAGE + 1 for n, p in zip(lens, pages)]
        scored = sum(p for p in pages if p > case["count"])
        return {"bytes": sum(seen) * h * row + scored * h * 4 * d + len(lens) * (case["heads"] * d * 4 + h * case["count"] * 4),
                "flops": case["heads"] * d * (4 * sum(seen) + 4 * scored)}
    pairs = sum(t * n - t * (t - 1) // 2 for n, t in zip(lens, new))
    return {"bytes": sum(lens) * h * row + sum(new) * case["heads"] * d * 4, "flops": 4 * pairs * case["heads"] * d}


# ------------------------------------------------------------------------------------------------- in 64 bits

def _places(d, g):
    """Where a record holds element e of row r: byte and shift of its codes, byte of its scale (its minimum is 8 behind)."""
    kb, ks, vb, vs, ksm, vsm = ([[0] * d for _ in range(PAGE)] for _ in range(6))
    for r in range(PAGE):
        for w in range(d // 8):
            for n in range(8):
                c, i = w // (d // 32), w % (d // 32)
                e = 64 * (i // 2) + 32 * (n % 2) + 8 * c + 4 * (n // 2 % 2) + 2 * (i % 2) + n // 4
                kb[r][e], ks[r][e] = r * (d // 2) + 4 * w + n // 2, 4 * (n % 2)
                e = 16 * n + w if d == 128 else 16 * (n % 4) + 8 * (n // 4) + w
                vb[r][e] = 32 * d + ((r // 4) * (d // 8) + w) * 16 + (r % 4) * 4 + n // 2
                vs[r][e] = 4 * (n % 2)
        for e in range(d):
            ksm[r][e] = 64 * d + (e // g) * 256 + (r // 4) * 16 + (r % 4) * 2
            vsm[r][e] = ksm[r][e] + 256 * (d // g)
    return [torch.tensor(x, device=DEV).flatten() for x in (kb, ks, vb, vs, ksm, vsm)]


def _half_at(rec, at):
    return torch.stack([rec[..., at], rec[..., at + 1]], -1).view(torch.float16)[..., 0].double()


def _read64(rec, places, d):
    """Keys and values of records uint8 [N, record] in 64 bits, [N, 64, D] each."""
    kb, ks, vb, vs, ksm, vsm = places
    out = []
    for byte, shift, sm in ((kb, ks, ksm), (vb, vs, vsm)):
        code = ((rec[:, byte].int() >> shift) & 15).double()
        out.append((code * _half_at(rec, sm) + _half_at(rec, sm + 8)).view(-1, PAGE, d))
    return out


def exact(case, seed):
    st = prepare(case, seed)
    d, g = case["dim"], case["group"]
    if case["kind"] == "copy":
        pool = st["pool"].clone()
        for a, b in zip(st["src"].tolist(), st["dst"].tolist()):
            pool[:, b] = st["pool"][:, a]
        return pool
    h = case["kv_heads"]
    if case["kind"] == "append":
        out = {"pool": None}
        for name in ("k", "v"):
            x = st[name].double().reshape(-1, g)
            low, high = x.min(1).values, x.max(1).values
            s = ((high - low).float().double() / 15).float().half().double()
            # the quotient is one of fp32 numbers, rounded to fp32 and then to the nearest whole number
            quotient = ((x - low[:, None]).float().double() / torch.where(s > 0, s, torch.ones_like(s))[:, None]).float()
            code = torch.clamp(torch.round(quotient.double()), 0, 15) * (s > 0)[:, None]
            out[name] = (code * s[:, None] + low[:, None]).view(st[name].shape)
        return out
    places = _places(d, g)
    share = case["heads"] // h
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    chosen = torch.full((case["batch"], h, case.get("count", 0)), -1, dtype=torch.int32, device=DEV)
    for b, (n, new) in enumerate(zip(st["host_lengths"], st["host_new"])):
        total = (n + PAGE - 1) // PAGE
        at = st["host_starts"][b]
        for j in range(h):
            named = list(range(total))
            q = st["q"][at:at + new, j * share:(j + 1) * share].double()  # [new, share, d]
            if case["kind"] == "sparse" and total > case["count"]:
                tail = st["pool"][st["pages"][b, :total].long(), j, 64 * d + 512 * (d // g):].contiguous()
                hi, lo = tail.view(torch.float16).double().split(d, 1)
                up, down = q[0].clamp(min=0), q[0].clamp(max=0)
                score = (up @ hi.t() + down @ lo.t()).max(0).values.tolist()
                score[0] = score[-1] = math.inf
                named = sorted(sorted(named, key=lambda p: (-score[p], p))[:case["count"]])
            if case["kind"] == "sparse":
                chosen[b, j, :len(named)] = torch.tensor(named, dtype=torch.int32)
            index = torch.tensor(named, device=DEV)
            k, v = _read64(st["pool"][st["pages"][b].long()[index], j], places, d)
            where = (index[:, None] * PAGE + torch.arange(PAGE, device=DEV)).flatten()
            pos = torch.arange(n - new, n, device=DEV)
            s = (q.reshape(-1, d) @ k.view(-1, d).t()) * st["scale"]
            s.view(new, share, -1).masked_fill_((where[None] > pos[:, None])[:, None], -math.inf)
            p = torch.softmax(s, -1)
            out[at:at + new, j * share:(j + 1) * share] = (p @ v.view(-1, d)).view(new, share, d)
    return {"pages": chosen, "out": out} if case["kind"] == "sparse" else out
