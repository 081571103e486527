"""What a decoder over fp16 caches is served with beside its linears, as cases that can be timed one by one:

    prefix   causal attention of each sequence's last tokens over a prefix that all sequences share and over rows of their own:
             q [tokens, heads, D], prefix [kv_heads, P, D], own rows [batch, kv_heads, room, D]; the tokens' own rows are
             stored first
    step     one token of each sequence over a cache of `room` rows a head that evicts by accumulated attention weight: where
             the cache is full the row of the lowest weight, neither among the first `first` nor the last `last` tokens,
             makes way for the new one; the weights that the token gives are added up
    weigh    the attention weight that a prompt's queries (all, or the last `window`) give each of its keys, summed
    keep     of a prompt's rows the `room` of the highest weight, with the first `first` and the last `last` among them,
             gathered into such a cache
    rules    penalties for repeated tokens, biases by token and a grammar's mask on logits, and the best token

Caches, queries and keys are fp16, weights fp32; the query heads h s .. h s + s - 1 read key/value head h, s = heads / kv_heads.

listed() holds the cases themselves, draw() makes more over the same ranges.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"


def _package():
    package = os.path.join(os.getcwd(), "sparse-quant_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from sqamd import evict, logits, prefix
    return prefix, evict, logits


def listed():
    return [
        # the decode step of an OPT-6.7B layer: 8 sequences behind one prompt of 512 rows
        {"name": "prefix_step_8x512", "kind": "prefix", "batch": 8, "heads": 32, "kv_heads": 32, "dim": 128, "prefix": 512,
         "rows": 128, "tokens": 1, "ragged": False},
        # serving: 64 sequences of different lengths behind one long document, shared heads
        {"name": "prefix_step_64x8192", "kind": "prefix", "batch": 64, "heads": 32, "kv_heads": 8, "dim": 128, "prefix": 8192,
         "rows": 1000, "tokens": 1, "ragged": True},
        # questions of different lengths about the same document
        {"name": "prefix_prompts_16x4096", "kind": "prefix", "batch": 16, "heads": 32, "kv_heads": 8, "dim": 128,
         "prefix": 4096, "rows": 700, "tokens": 512, "ragged": True},
        # the decode step of an OPT-6.7B layer at batch 8 over caches of 512 rows
        {"name": "step_8x512", "kind": "step", "batch": 8, "heads": 32, "kv_heads": 32, "dim": 128, "room": 512, "seen": 700,
         "first": 4, "last": 128},
        # serving: 32 long sequences held to 4000 rows, some of them not full yet
        {"name": "step_32x4000", "kind": "step", "batch": 32, "heads": 32, "kv_heads": 8, "dim": 128, "room": 4000,
         "seen": 9000, "first": 16, "last": 1000},
        # the longest prompts that an OPT-6.7B layer takes, at batch 8: every query counts
        {"name": "weigh_8x2048", "kind": "weigh", "batch": 8, "heads": 32, "kv_heads": 32, "dim": 128, "rows": 2048,
         "window": 0, "ragged": False},
        # long prompts of different lengths, weighed by their last queries
        {"name": "weigh_4x8191_last64", "kind": "weigh", "batch": 4, "heads": 32, "kv_heads": 8, "dim": 128, "rows": 8191,
         "window": 64, "ragged": True},
        # the prompt of an OPT-6.7B layer at batch 8, half of it kept
        {"name": "keep_8x512", "kind": "keep", "batch": 8, "kv_heads": 32, "dim": 128, "rows": 512, "room": 256, "first": 4,
         "last": 64, "ragged": False},
        # long prompts of different lengths
        {"name": "keep_16x20000", "kind": "keep", "batch": 16, "kv_heads": 8, "dim": 128, "rows": 20000, "room": 2000,
         "first": 4, "last": 500, "ragged": True},
        # a token of one sequence, a grammar alone: launch latency
        {"name": "rules_1_mask", "kind": "rules", "batch": 1, "vocab": 50272, "dtype": "fp16", "tokens": 0, "penalties": False,
         "biases": 0, "mask": True},
        # the end of the decode step of OPT-6.7B at batch 8
        {"name": "rules_8", "kind": "rules", "batch": 8, "vocab": 50272, "dtype": "fp16", "tokens": 640, "penalties": True,
         "biases": 8, "mask": True},
        # many sequences, a large vocabulary, long texts
        {"name": "rules_200", "kind": "rules", "batch": 200, "vocab": 131077, "dtype": "fp32", "tokens": 5000, "penalties": True,
         "biases": 100, "mask": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prefix", "prefix", "step", "weigh", "keep", "rules"])
    case = {"kind": kind}
    if kind == "rules":
        case["batch"] = _log_int(rng, 1, 200)
        case["vocab"] = min(_log_int(rng, 1000, 262144), 200 * 131072 // case["batch"])
        case["dtype"] = rng.choice(["fp16", "fp32"])
        case["tokens"] = rng.choice([0, _log_int(rng, 1, 5000)])
        case["penalties"] = rng.random() < 0.7
        case["biases"] = rng.choice([0, _log_int(rng, 1, 300)])
        case["mask"] = rng.random() < 0.6
        return case
    case["dim"] = rng.choice([64, 128, 128])
    case["kv_heads"] = rng.choice([1, 2, 3, 4, 8, 8, 32])
    if kind == "keep":
        case["rows"] = _log_int(rng, 16, 20000)
        case["room"] = max(8, min(_log_int(rng, 8, 4000), case["rows"] * 2))
        case["batch"] = max(1, min(_log_int(rng, 1, 64), 16 * 20000 * 8 // (case["rows"] * case["kv_heads"]),
                                   16 * 2000 * 8 // (case["room"] * case["kv_heads"])))
        case["first"] = rng.randint(0, min(4, case["room"] // 4))
        case["last"] = rng.randint(1, case["room"] // 2)
        case["ragged"] = rng.random() < 0.5
        return case
    case["heads"] = case["kv_heads"] * rng.choice([1, 2, 4, 4, 5, 8] if case["kv_heads"] <= 8 else [1, 2])
    if kind == "step":
        case["room"] = _log_int(rng, 8, 8000)
        case["batch"] = max(1, min(_log_int(rng, 1, 128), 32 * 4000 * 8 // (case["room"] * case["kv_heads"])))
        case["seen"] = _log_int(rng, 1, 3 * case["room"])
        case["first"] = rng.randint(0, min(16, case["room"] // 4))
        case["last"] = rng.randint(1, case["room"] // 2)
        return case
    if kind == "weigh":
        case["window"] = rng.choice([0, _log_int(rng, 1, 128)])
        case["rows"] = _log_int(rng, 16, 8191 if case["window"] else 4096)
        room = 4 * 8191 * 8 // (case["rows"] * case["kv_heads"]) if case["window"] else \
            8 * 32 * 2048 * 2048 // (case["rows"] ** 2 * case["heads"])
        case["batch"] = max(1, min(_log_int(rng, 1, 32), room))
        case["ragged"] = rng.random() < 0.5
        return case
    case["ragged"] = rng.random() < 0.5
    case["tokens"] = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 8, 512)])
    case["prefix"] = _log_int(rng, 1, 16384)
    case["rows"] = case["tokens"] + _log_int(rng, 1, 2048) - 1
    room = min(64 * 1000 * 8 // (case["rows"] * case["kv_heads"]),
               16 * 128 * 4096 * 32 // (case["tokens"] * (case["prefix"] + case["rows"]) * case["heads"]))
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


def _seen(case):
    """Tokens of every sequence, the present one among them: by the case alone."""
    rng = random.Random("%d %d %d" % (case["batch"], case["room"], case["seen"]))
    return [case["seen"] if i == 0 else rng.randint(max(1, case["seen"] // 4), case["seen"]) for i in range(case["batch"])]


def _normal(gen, *shape):
    return torch.randn(shape, device=DEV, generator=gen).half()


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    st = {"case": case}
    if case["kind"] == "rules":
        return _prepare_rules(case, st, gen)
    d, h, b = case["dim"], case["kv_heads"], case["batch"]
    st["scale"] = 1.0 / math.sqrt(d)
    if case["kind"] == "prefix":
        lens, new = _sizes(case)
        st["host_lengths"], st["host_new"], st["host_starts"] = lens, new, [0]
        for n in new:
            st["host_starts"].append(st["host_starts"][-1] + n)
        t = st["host_starts"][-1]
        st["starts"] = None if min(new) == max(new) else torch.tensor(st["host_starts"], dtype=torch.int32, device=DEV)
        st["lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        st["k_prefix"], st["v_prefix"] = _normal(gen, h, case["prefix"], d), _normal(gen, h, case["prefix"], d)
        room = max(lens) + 16
        st["k_cache"], st["v_cache"] = _normal(gen, b, h, room, d), _normal(gen, b, h, room, d)
        # queries, keys and values as a fused projection leaves them
        qkv = _normal(gen, t, case["heads"] + 2 * h, d)
        st["q"], st["k"], st["v"] = qkv.split([case["heads"], h, h], 1)
        return st
    if case["kind"] == "step":
        room, seen = case["room"], _seen(case)
        st["seen"] = torch.tensor(seen, dtype=torch.int32, device=DEV)
        st["k_cache"], st["v_cache"] = _normal(gen, b, h, room, d), _normal(gen, b, h, room, d)
        qkv = _normal(gen, b, case["heads"] + 2 * h, d)
        st["q"], st["k"], st["v"] = qkv.split([case["heads"], h, h], 1)
        # weights as long texts leave them: a few rows with most of it
        weight = torch.exp(1.5 * torch.randn((b, h, room), device=DEV, generator=gen))
        st["weight"] = weight * (case["heads"] // h)
        # a full cache holds the first and the last tokens and others between them, in no order
        position = torch.empty((b, h, room), dtype=torch.int32, device=DEV)
        for i, n in enumerate(seen):
            order = torch.rand((h, max(n - 1, room)), device=DEV, generator=gen)
            if n - 1 > room:
                order[:, :case["first"]] = -1.0
                order[:, n - case["last"]:n - 1] = -1.0
                order[:, n - 1:] = 2.0
                position[i] = order.argsort(-1)[:, :room].int()
            else:
                position[i] = torch.arange(room, device=DEV, dtype=torch.int32)
        st["position"] = position
        return st
    lens, _ = _sizes(case)
    st["host_lengths"] = lens
    st["lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEV) if case["ragged"] else None
    s = max(lens)
    if case["kind"] == "weigh":
        qkv = _normal(gen, b, s, case["heads"] + 2 * h, d).transpose(1, 2)
        st["q"], st["k"] = qkv[:, :case["heads"]], qkv[:, case["heads"]:case["heads"] + h]
        return st
    qkv = _normal(gen, b, s, 3 * h, d).transpose(1, 2)
    st["k"], st["v"] = qkv[:, h:2 * h], qkv[:, 2 * h:]
    st["weight"] = torch.exp(1.5 * torch.randn((b, h, s), device=DEV, generator=gen))
    room = case["room"]
    st["k_cache"] = torch.zeros((b, h, room, d), dtype=torch.float16, device=DEV)
    st["v_cache"] = torch.zeros_like(st["k_cache"])
    st["cache_weight"] = torch.zeros((b, h, room), device=DEV)
    st["position"] = torch.zeros((b, h, room), dtype=torch.int32, device=DEV)
    return st


def _prepare_rules(case, st, gen):
    m, n, length = case["batch"], case["vocab"], case["tokens"]
    dtype = torch.float16 if case["dtype"] == "fp16" else torch.float32
    st["logits"] = (3.0 * torch.randn((m, n), device=DEV, generator=gen)).to(dtype)
    for name in ("ids", "lengths", "generated_from", "repetition", "presence", "frequency", "bias_ids", "bias", "mask"):
        st[name] = None
    if length:
        # texts repeat themselves: few tokens often, many seldom
        u = torch.rand((m, length), device=DEV, generator=gen)
        st["ids"] = (n ** u).long().clamp_(max=n - 1) * 7919 % n
        rng = random.Random("%d %d" % (m, length))
        lens = [length if i == 0 else rng.randint(0, length) for i in range(m)]
        st["lengths"] = torch.tensor(lens, device=DEV)
        st["generated_from"] = torch.tensor([rng.randint(0, k) for k in lens], device=DEV)
        if case["penalties"]:
            st["repetition"] = 1.0 + 0.3 * torch.rand(m, device=DEV, generator=gen)
            st["presence"] = 0.5 * torch.rand(m, device=DEV, generator=gen)
            st["frequency"] = 0.2 * torch.rand(m, device=DEV, generator=gen)
    if case["biases"]:
        st["bias_ids"] = torch.randint(-1, n, (m, case["biases"]), dtype=torch.int32, device=DEV, generator=gen)
        st["bias"] = 4.0 * torch.randn((m, case["biases"]), device=DEV, generator=gen)
    if case["mask"]:
        words = (n + 31) // 32
        st["mask"] = torch.randint(-2 ** 31, 2 ** 31, (m, words), device=DEV, generator=gen).int()
    return st


# ---------------------------------------------------------------------------------------------- the plain forms

def _softmax(s):
    """Rows of scores fp32; a row of -inf gives 0."""
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    l = p.sum(-1, keepdim=True)
    return p / torch.where(l == 0, torch.ones_like(l), l)


def _prefix_plain(st):
    case, q = st["case"], st["q"]
    h, d, p = case["kv_heads"], case["dim"], case["prefix"]
    share = case["heads"] // h
    kp, vp = st["k_prefix"].float(), st["v_prefix"].float()
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    for b, (n, new) in enumerate(zip(st["host_lengths"], st["host_new"])):
        at = st["host_starts"][b]
        st["k_cache"][b, :, n - new:n] = st["k"][at:at + new].transpose(0, 1)
        st["v_cache"][b, :, n - new:n] = st["v"][at:at + new].transpose(0, 1)
        k = torch.cat([kp, st["k_cache"][b, :, :n].float()], 1)
        v = torch.cat([vp, st["v_cache"][b, :, :n].float()], 1)
        rows = q[at:at + new].float().view(new, h, share, d).permute(1, 0, 2, 3).reshape(h, new * share, d)
        s = torch.matmul(rows, k.transpose(1, 2)) * st["scale"]
        if new > 1:
            pos = torch.arange(p + n - new, p + n, device=q.device).repeat_interleave(share)
            s = s.masked_fill(torch.arange(p + n, device=q.device)[None] > pos[:, None], -math.inf)
        o = torch.matmul(_softmax(s), v)
        out[at:at + new] = o.view(h, new, share, d).permute(1, 0, 2, 3).reshape(new, -1, d).half()
    return {"out": out, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _step_plain(st):
    case = st["case"]
    b, h, d, room = case["batch"], case["kv_heads"], case["dim"], case["room"]
    share = case["heads"] // h
    seen = st["seen"].view(b, 1, 1)
    free = (st["position"] >= case["first"]) & (st["position"] < seen - case["last"])
    cost = torch.where(free, st["weight"], torch.full_like(st["weight"], math.inf))
    slot = torch.where(seen <= room, seen.long() - 1, cost.argmin(-1, keepdim=True))  # [b, h, 1]
    st["weight"].scatter_(2, slot, 0.0)
    st["position"].scatter_(2, slot, (seen - 1).expand(b, h, 1).contiguous())
    for cache, new in ((st["k_cache"], st["k"]), (st["v_cache"], st["v"])):
        cache.scatter_(2, slot[..., None].expand(b, h, 1, d), new[:, :, None])
    s = torch.matmul(st["q"].float().view(b, h, share, d), st["k_cache"].float().transpose(2, 3)) * st["scale"]
    valid = torch.arange(room, device=s.device) < seen[..., None]
    p = _softmax(s.masked_fill(~valid, -math.inf))
    st["weight"] += p.sum(2)
    out = torch.matmul(p, st["v_cache"].float().masked_fill(~valid.transpose(2, 3), 0.0)).half()
    return {"out": out.view(b, -1, d), "slot": slot[..., 0].int(), "weight": st["weight"], "position": st["position"],
            "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _weigh_plain(st):
    case = st["case"]
    b, h, d = case["batch"], case["kv_heads"], case["dim"]
    share, s = case["heads"] // h, st["q"].shape[2]
    out = torch.zeros((b, h, s), device=st["q"].device)
    for i, n in enumerate(st["host_lengths"]):
        first = max(0, n - case["window"]) if case["window"] else 0
        for at in range(first, n, 1024):
            end = min(at + 1024, n)
            q = st["q"][i, :, at:end].float().view(h, share, end - at, d)
            score = torch.matmul(q, st["k"][i, :, None, :n].float().transpose(2, 3)) * st["scale"]
            pos = torch.arange(at, end, device=q.device)
            score = score.masked_fill(torch.arange(n, device=q.device)[None] > pos[:, None], -math.inf)
            out[i, :, :n] += _softmax(score).sum((1, 2))
    return out


def _keep_plain(st):
    case = st["case"]
    b, h, d, room = case["batch"], case["kv_heads"], case["dim"], case["room"]
    dev = st["k"].device
    rows = torch.full((b, h, room), -1, dtype=torch.int32, device=dev)
    for i, n in enumerate(st["host_lengths"]):
        score = st["weight"][i, :, :n].clone()
        score[:, :case["first"]] = math.inf
        score[:, max(0, n - case["last"]):] = math.inf
        best = torch.sort(score, dim=-1, descending=True, stable=True).indices[:, :room].sort(-1).values
        m = best.shape[1]
        rows[i, :, :m] = best.int()
        index = best[..., None].expand(h, m, d)
        st["k_cache"][i, :, :m] = st["k"][i].gather(1, index)
        st["v_cache"][i, :, :m] = st["v"][i].gather(1, index)
        st["cache_weight"][i, :, :m] = st["weight"][i].gather(1, best)
        st["position"][i, :, :m] = best.int()
    return {"rows": rows, "k_cache": st["k_cache"], "v_cache": st["v_cache"], "weight": st["cache_weight"],
            "position": st["position"]}


def _counts(st):
    """How often each token stands in a row's text, and in the generated part of it: int64 [batch, vocab] each."""
    ids, case = st["ids"], st["case"]
    m, n = case["batch"], case["vocab"]
    place = torch.arange(ids.shape[1], device=ids.device)[None]
    inside = place < st["lengths"][:, None]
    out = []
    for counted in (inside, inside & (place >= st["generated_from"][:, None])):
        c = torch.zeros((m, n), dtype=torch.int64, device=ids.device)
        out.append(c.scatter_add_(1, ids, counted.long()))
    return out


def _last_bias(st, dtype):
    """Biases by token: [batch, vocab]; of a token that stands twice the last entry counts, one outside is none."""
    case = st["case"]
    m, n, count = case["batch"], case["vocab"], case["biases"]
    entry = torch.zeros((m, n + 1), dtype=torch.int64, device=DEV)
    where = torch.where(st["bias_ids"] < 0, torch.full_like(st["bias_ids"], n), st["bias_ids"]).long()
    order = torch.arange(1, count + 1, device=DEV).expand(m, count)
    entry = entry.scatter_reduce(1, where, order, "amax")[:, :n]
    padded = torch.cat([torch.zeros((m, 1), device=DEV), st["bias"]], 1).to(dtype)
    return padded.gather(1, entry)


def _allowed(st):
    bit = torch.arange(32, dtype=torch.int32, device=DEV)
    return (((st["mask"][..., None] >> bit) & 1) != 0).flatten(1)[:, :st["case"]["vocab"]]


def _rules_plain(st):
    x = st["logits"].float()
    if st["repetition"] is not None:
        count, generated = _counts(st)
        r = st["repetition"][:, None]
        x = torch.where(count > 0, torch.where(x > 0, x / r, x * r), x)
        x = torch.where(generated > 0, x - st["frequency"][:, None] * generated.float(), x)
        x = torch.where(generated > 0, x - st["presence"][:, None], x)
    if st["bias_ids"] is not None:
        x = x + _last_bias(st, torch.float32)
    if st["mask"] is not None:
        x = x.masked_fill(~_allowed(st), -math.inf)
    x = x.to(st["logits"].dtype)
    best = x.amax(1, keepdim=True)
    index = torch.arange(x.shape[1], device=DEV).expand(x.shape)
    token = torch.where(x == best, index, torch.full_like(index, x.shape[1])).amin(1)
    return {"logits": x, "token": torch.where(best[:, 0] == -math.inf, torch.zeros_like(token), token)}


def run(state):
    st, case = state, state["case"]
    kind = case["kind"]
    if not own:
        return {"prefix": _prefix_plain, "step": _step_plain, "weigh": _weigh_plain, "keep": _keep_plain,
                "rules": _rules_plain}[kind](st)
    prefix, evict, logits = _package()
    if kind == "prefix":
        out = prefix.attention(st["q"], st["k_prefix"], st["v_prefix"], st["k_cache"], st["v_cache"], st["lengths"],
                               st["scale"], starts=st["starts"], k_new=st["k"], v_new=st["v"])
        return {"out": out, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    if kind == "step":
        out, slot = evict.attention(st["q"], st["k"], st["v"], st["k_cache"], st["v_cache"], st["weight"], st["position"],
                                    st["seen"], st["scale"], case["first"], case["last"])
        return {"out": out, "slot": slot, "weight": st["weight"], "position": st["position"], "k_cache": st["k_cache"],
                "v_cache": st["v_cache"]}
    if kind == "weigh":
        return evict.attention_weights(st["q"], st["k"], st["scale"], window=case["window"] or None, lengths=st["lengths"])
    if kind == "keep":
        rows = evict.keep(st["k"], st["v"], st["weight"], st["k_cache"], st["v_cache"], st["cache_weight"], st["position"],
                          case["first"], case["last"], lengths=st["lengths"])
        return {"rows": rows, "k_cache": st["k_cache"], "v_cache": st["v_cache"], "weight": st["cache_weight"],
                "position": st["position"]}
    out, token = logits.apply_rules(st["logits"], st["ids"], st["lengths"], st["generated_from"], st["repetition"],
                                    st["presence"], st["frequency"], st["bias_ids"], st["bias"], st["mask"])
    return {"logits": out, "token": token}


def work(case):
    kind, b = case["kind"], case["batch"]
    if kind == "rules":
        n, size = case["vocab"], 2 if case["dtype"] == "fp16" else 4
        text = sum(_prepared_lengths(case)) * 8
        per_row = 2 * n * size + case["biases"] * 8 + (4 * ((n + 31) // 32) if case["mask"] else 0) + 8
        return {"bytes": b * per_row + (text if case["penalties"] else 0), "flops": 8 * b * n}
    d, h = case["dim"], case["kv_heads"]
    if kind == "step":
        rows = [min(n, case["room"]) for n in _seen(case)]
        return {"bytes": sum(rows) * h * (4 * d + 12) + b * (4 * d * case["heads"] + h * (8 * d + 12)),
                "flops": 4 * d * case["heads"] * sum(rows)}
    lens, new = _sizes(case)
    if kind == "keep":
        kept = sum(min(n, case["room"]) for n in lens)
        return {"bytes": h * (kept * (8 * d + 16) + 4 * sum(lens)), "flops": 0}
    if kind == "weigh":
        w = [min(n, case["window"]) if case["window"] else n for n in lens]
        pairs = sum(m * n - m * (m - 1) // 2 for n, m in zip(lens, w))
        return {"bytes": sum(lens) * h * (2 * d + 4) + sum(w) * case["heads"] * 2 * d, "flops": 2 * d * case["heads"] * pairs}
    pairs = sum(t * (case["prefix"] + n) - t * (t - 1) // 2 for n, t in zip(lens, new))
    return {"bytes": (case["prefix"] + sum(lens)) * h * 4 * d + sum(new) * (case["heads"] + h) * 4 * d,
            "flops": 4 * d * case["heads"] * pairs}


def _prepared_lengths(case):
    rng = random.Random("%d %d" % (case["batch"], case["tokens"]))
    return [case["tokens"] if i == 0 else rng.randint(0, case["tokens"]) for i in range(case["batch"])]


# ------------------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    return {"prefix": _prefix_exact, "step": _step_exact, "weigh": _weigh_exact, "keep": _keep_exact,
            "rules": _rules_exact}[case["kind"]](case, st)


def _probabilities(q, k, scale, hidden=None):
    s = (q @ k.t()) * scale
    return torch.softmax(s if hidden is None else s.masked_fill(hidden, -math.inf), -1)


def _prefix_exact(case, st):
    share = case["heads"] // case["kv_heads"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    p = case["prefix"]
    for b, (n, new) in enumerate(zip(st["host_lengths"], st["host_new"])):
        at = st["host_starts"][b]
        for t in range(new):
            st["k_cache"][b, :, n - new + t] = st["k"][at + t]
            st["v_cache"][b, :, n - new + t] = st["v"][at + t]
        col = torch.arange(p + n, device=DEV)
        hidden = (col[None] > (p + n - new + torch.arange(new, device=DEV))[:, None])[:, None].expand(new, share, p + n)
        for j in range(case["kv_heads"]):
            k = torch.cat([st["k_prefix"][j], st["k_cache"][b, j, :n]]).double()
            v = torch.cat([st["v_prefix"][j], st["v_cache"][b, j, :n]]).double()
            q = st["q"][at:at + new, j * share:(j + 1) * share].double().reshape(new * share, -1)
            o = _probabilities(q, k, st["scale"], hidden.reshape(new * share, -1)) @ v
            out[at:at + new, j * share:(j + 1) * share] = o.view(new, share, -1)
    return {"out": out, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _step_exact(case, st):
    share, room = case["heads"] // case["kv_heads"], case["room"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    weight = st["weight"].double()
    slots = torch.zeros(weight.shape[:2], dtype=torch.int32, device=DEV)
    for b, n in enumerate(_seen(case)):
        for j in range(case["kv_heads"]):
            at = n - 1
            if n > room:
                pos, w = st["position"][b, j].tolist(), weight[b, j].tolist()
                at = min((w[r], r) for r in range(room) if case["first"] <= pos[r] < n - case["last"])[1]
            slots[b, j] = at
            st["k_cache"][b, j, at], st["v_cache"][b, j, at] = st["k"][b, j], st["v"][b, j]
            weight[b, j, at], st["position"][b, j, at] = 0.0, n - 1
            used = min(n, room)
            q = st["q"][b, j * share:(j + 1) * share].double()
            p = _probabilities(q, st["k_cache"][b, j, :used].double(), st["scale"])
            weight[b, j, :used] += p.sum(0)
            out[b, j * share:(j + 1) * share] = p @ st["v_cache"][b, j, :used].double()
    return {"out": out, "slot": slots, "weight": weight, "position": st["position"], "k_cache": st["k_cache"],
            "v_cache": st["v_cache"]}


def _weigh_exact(case, st):
    share = case["heads"] // case["kv_heads"]
    b, _, s, _ = st["k"].shape
    out = torch.zeros((b, case["kv_heads"], s), dtype=torch.float64, device=DEV)
    for i, n in enumerate(st["host_lengths"]):
        first = max(0, n - case["window"]) if case["window"] else 0
        hidden = torch.arange(n, device=DEV)[None] > torch.arange(first, n, device=DEV)[:, None]
        for g in range(case["heads"]):
            q, k = st["q"][i, g, first:n].double(), st["k"][i, g // share, :n].double()
            out[i, g // share, :n] += _probabilities(q, k, st["scale"], hidden).sum(0)
    return out


def _keep_exact(case, st):
    room = case["room"]
    b, h, _, _ = st["k"].shape
    rows = torch.full((b, h, room), -1, dtype=torch.int32)
    for i, n in enumerate(st["host_lengths"]):
        for j in range(h):
            w = st["weight"][i, j, :n].tolist()
            forced = [r for r in range(n) if r < case["first"] or r >= n - case["last"]]
            others = sorted((r for r in range(case["first"], n - case["last"])), key=lambda r: (-w[r], r))
            kept = sorted((forced + others)[:room])
            rows[i, j, :len(kept)] = torch.tensor(kept, dtype=torch.int32)
            index = torch.tensor(kept, device=DEV)
            st["k_cache"][i, j, :len(kept)], st["v_cache"][i, j, :len(kept)] = st["k"][i, j, index], st["v"][i, j, index]
            st["cache_weight"][i, j, :len(kept)], st["position"][i, j, :len(kept)] = st["weight"][i, j, index], index.int()
    return {"rows": rows.to(DEV), "k_cache": st["k_cache"], "v_cache": st["v_cache"], "weight": st["cache_weight"],
            "position": st["position"]}


def _rules_exact(case, st):
    x = st["logits"].double()
    n = case["vocab"]
    for i in range(case["batch"]):
        row = x[i]
        if st["repetition"] is not None:
            text = st["ids"][i, :int(st["lengths"][i])]
            made = text[int(st["generated_from"][i]):]
            r, f, p = (float(st[name][i]) for name in ("repetition", "frequency", "presence"))
            at = text.unique()
            row[at] = torch.where(row[at] > 0, row[at] / r, row[at] * r)
            at, count = made.unique(return_counts=True)
            row[at] = row[at] - f * count.double() - p
        if st["bias_ids"] is not None:
            named = dict(zip(st["bias_ids"][i].tolist(), st["bias"][i].tolist()))
            named.pop(-1, None)
            at = torch.tensor(list(named), dtype=torch.int64, device=DEV)
            row[at] += torch.tensor(list(named.values()), dtype=torch.float64, device=DEV)
        if st["mask"] is not None:
            word = torch.arange(n, device=DEV)
            row[((st["mask"][i].long()[word // 32] >> (word % 32)) & 1) == 0] = -math.inf
    return {"logits": x, "token": None}  # the token is the best of the rounded logits
