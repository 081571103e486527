"""The cache that evicts by accumulated attention weight, on the device against the oracle (64 bits).

Outputs: as for attention behind a prefix, 2^-11 (2 sum P |v| + |out|).  Weights are fp32: a score is a sum of D products, in
error by at most D 2^-24 sum |q k| scale, and its scaling, reference and exponential (2^-23) by a few 2^-24 of the score; the sums of
N exponentials by N 2^-24 at most.  With |q|, |k| as drawn here sum |q k| scale < 2 sqrt(D): (2 D sqrt(D) + 8 |s| + N + 64) 2^-24
of a probability, |s| < 64."""
import numpy as np
import pytest
import torch

import serving_oracle as so

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOL = 3 * 2.0 ** -11 * 1.02


@pytest.fixture(scope="module")
def evict(built_lib):
    from sqamd import evict as m
    return m


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def normal(rng, *shape, scale=1.0):
    return (rng.normal(0, scale, shape)).astype(np.float16)


def weight_tol(d, n):
    return (2 * d * np.sqrt(d) + 8 * 64 + n + 64) * 2.0 ** -24


def state(rng, b, h, room, d, seen, first, last):
    """A cache after seen - 1 tokens: the first and the last, and others of them between in no order."""
    position = np.zeros((b, h, room), np.int32)
    for i, n in enumerate(seen):
        for j in range(h):
            if n - 1 <= room:
                position[i, j] = np.arange(room)
            else:
                forced = np.r_[:first, n - last:n - 1]
                others = rng.permutation(np.arange(first, n - last))[:room - len(forced)]
                position[i, j] = rng.permutation(np.r_[forced, others])
    weight = np.exp(rng.normal(0, 1, (b, h, room))).astype(np.float32)
    return normal(rng, b, h, room, d), normal(rng, b, h, room, d), weight, position


def check_step(got, want, d, room):
    (out, slot), (kc, vc, weight, position) = got
    ref, size, rslot, rk, rv, rw, rp = want
    assert np.array_equal(slot.cpu().numpy(), rslot)
    assert np.array_equal(kc.cpu().numpy(), rk, equal_nan=True) and np.array_equal(vc.cpu().numpy(), rv, equal_nan=True)
    assert np.array_equal(position.cpu().numpy(), rp)
    out = out.float().cpu().numpy()
    assert (np.abs(out - ref) <= TOL * size + 1e-6).all(), np.abs(out - ref).max()
    w = weight.cpu().numpy()
    assert (np.abs(w - rw) <= weight_tol(d, room) * np.abs(rw) + 1e-9).all(), (np.abs(w - rw) / np.abs(rw)).max()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,h", [(4, 4), (8, 2), (5, 1), (70, 1)])
@pytest.mark.parametrize("room,first,last", [(1, 0, 1), (8, 2, 3), (64, 4, 16), (65, 0, 1), (300, 4, 100), (2100, 16, 500)])
def test_steps(evict, d, heads, h, room, first, last):
    rng = np.random.default_rng(room + d + heads)
    b = 4
    seen = np.array([1, room, room + 1, 3 * room + 5], np.int32)
    kc, vc, weight, position = state(rng, b, h, room, d, seen, first, last)
    kc[0, :, 0:], vc[0, :, 0:] = np.nan, np.nan  # (rows that hold nothing yet)
    cache = [dev(x) for x in (kc, vc, weight, position)]
    for i in range(3):
        q, kn, vn = normal(rng, b, heads, d), normal(rng, b, h, d), normal(rng, b, h, d)
        want = so.evict_step(q, kn, vn, kc, vc, weight, position, seen, 1 / np.sqrt(d), first, last)
        got = evict.attention(dev(q), dev(kn), dev(vn), *cache, dev(seen), 1 / np.sqrt(d), first, last)
        # (weights of rows that hold nothing do not change)
        check_step((got, cache), want, d, room)
        kc, vc, position = want[3], want[4], want[6]
        weight = cache[2].cpu().numpy()
        seen = seen + 1


def test_weights_of_any_kind(evict):
    # ties go to the lowest row, NaN is the lowest weight, infinities have their place, no row may go: row 0
    rng = np.random.default_rng(1)
    b, h, room, d = 6, 2, 40, 64
    seen = np.full(b, 100, np.int32)
    kc, vc, weight, position = state(rng, b, h, room, d, seen, 2, 5)
    weight[0] = 1.0
    weight[1, :, 17] = np.nan
    weight[2] = np.inf
    weight[3, :, 20:] = -np.inf
    weight[4] = -rng.random((h, room))
    position[5] = np.arange(100 - room, 100)
    position[5][position[5] < 95] = 1
    q, kn, vn = normal(rng, b, h, d), normal(rng, b, h, d), normal(rng, b, h, d)
    with np.errstate(invalid="ignore"):
        want = so.evict_step(q, kn, vn, kc, vc, weight, position, seen, 0.125, 2, 5)
    cache = [dev(x) for x in (kc, vc, weight, position)]
    _, slot = evict.attention(dev(q), dev(kn), dev(vn), *cache, dev(seen), 0.125, 2, 5)
    assert np.array_equal(slot.cpu().numpy(), want[2])
    assert np.array_equal(np.isnan(cache[2].cpu().numpy()), np.isnan(want[5]))
    assert np.array_equal(cache[3].cpu().numpy(), want[6])


def test_nothing_seen_and_large_scores(evict):
    rng = np.random.default_rng(2)
    b, h, room, d = 3, 2, 130, 128
    seen = np.array([0, -4, 400], np.int32)
    kc, vc, weight, position = state(rng, b, h, room, d, np.array([1, 1, 400]), 4, 30)
    q, kn, vn = normal(rng, b, 4, d, scale=8.0), normal(rng, b, h, d), normal(rng, b, h, d)
    want = so.evict_step(q, kn, vn, kc, vc, weight, position, seen, 1 / np.sqrt(d), 4, 30)
    cache = [dev(x) for x in (kc, vc, weight, position)]
    out = torch.full((b, 4, d), 5.0, dtype=torch.float16, device=DEV)
    got, slot = evict.attention(dev(q), dev(kn), dev(vn), *cache, dev(seen), 1 / np.sqrt(d), 4, 30, out=out)
    assert got is out and (slot[:2] == -1).all() and (out[:2] == 0).all()
    assert np.array_equal(slot.cpu().numpy(), want[2]) and np.array_equal(cache[0].cpu().numpy(), want[3])
    assert (np.abs(out.float().cpu().numpy() - want[0]) <= TOL * want[1] + 1e-6).all()


@pytest.mark.parametrize("b,heads,room", [(2, 4, 700), (80, 8, 100), (2, 80, 100)])
def test_the_result_in_the_place_of_the_queries(evict, b, heads, room):
    rng = np.random.default_rng(b + heads)
    h, d = heads // 4 if heads < 80 else 2, 64
    seen = np.full(b, 2 * room, np.int32)
    cache = [dev(x) for x in state(rng, b, h, room, d, seen, 2, 5)]
    twin = [x.clone() for x in cache]
    q, kn, vn = dev(normal(rng, b, heads, d)), dev(normal(rng, b, h, d)), dev(normal(rng, b, h, d))
    want, _ = evict.attention(q, kn, vn, *cache, dev(seen), 0.125, 2, 5)
    got, _ = evict.attention(q, kn, vn, *twin, dev(seen), 0.125, 2, 5, out=q)
    assert got is q and torch.equal(q, want) and all(torch.equal(a, c) for a, c in zip(cache, twin))


def test_strided_rows_and_caches(evict):
    rng = np.random.default_rng(3)
    b, heads, h, room, d = 2, 4, 2, 70, 64
    seen = np.array([71, 200], np.int32)
    kc, vc, weight, position = state(rng, b, h, room, d, seen, 1, 8)
    qkv = normal(rng, b, heads + 2 * h, d)
    want = so.evict_step(qkv[:, :heads], qkv[:, heads:heads + h], qkv[:, heads + h:], kc, vc, weight, position, seen, 0.125, 1, 8)
    both = torch.zeros((b, room + 2, 2, h, d), dtype=torch.float16, device=DEV)
    views = [both[:, :room, i].transpose(1, 2) for i in range(2)]
    views[0].copy_(dev(kc))
    views[1].copy_(dev(vc))
    x = dev(qkv)
    rest = [dev(weight), dev(position)]
    got = evict.attention(x[:, :heads], x[:, heads:heads + h], x[:, heads + h:], *views, *rest, dev(seen), 0.125, 1, 8)
    check_step((got, views + rest), want, d, room)
    assert (both[:, room:] == 0).all()


def test_captured_steps(evict):
    rng = np.random.default_rng(4)
    b, heads, h, room, d = 2, 4, 2, 48, 128
    seen = torch.tensor([44, 100], dtype=torch.int32, device=DEV)
    cache = [dev(x) for x in state(rng, b, h, room, d, [44, 100], 2, 8)]
    qkv = dev(normal(rng, b, heads + 2 * h, d))

    def step(c):
        return evict.attention(qkv[:, :heads], qkv[:, heads:heads + h], qkv[:, heads + h:], *c, seen, 0.09, 2, 8)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([c.clone() for c in cache])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, slot = step(cache)
    twin = [c.clone() for c in cache]
    for i in range(8):
        qkv.copy_(dev(normal(rng, b, heads + 2 * h, d)))
        want = [x.clone() for x in step(twin)]
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(out, want[0]) and torch.equal(slot, want[1]), i
        assert all(torch.equal(a, c) for a, c in zip(cache, twin)), i
        seen += 1


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,h", [(2, 2), (6, 2), (5, 1)])
@pytest.mark.parametrize("s,window", [(1, None), (33, None), (64, 3), (129, None), (129, 64), (300, 1), (300, 1000), (700, 40)])
def test_weights(evict, d, heads, h, s, window):
    rng = np.random.default_rng(s + heads)
    b = 3
    lens = np.array([s, max(1, s // 2), 0], np.int32)
    qk = normal(rng, b, s, heads + h, d)  # as a fused projection leaves them
    x = dev(qk).transpose(1, 2)
    want = so.attention_weights(qk.transpose(0, 2, 1, 3)[:, :heads], qk.transpose(0, 2, 1, 3)[:, heads:], lens, 1 / np.sqrt(d), window)
    got = evict.attention_weights(x[:, :heads], x[:, heads:], 1 / np.sqrt(d), window, dev(lens)).cpu().numpy()
    assert (np.abs(got - want) <= weight_tol(d, 2 * s) * want + 1e-9).all(), np.abs(got - want).max()
    full = evict.attention_weights(x[:1, :heads], x[:1, heads:], 1 / np.sqrt(d), window).cpu().numpy()
    assert np.array_equal(full, got[:1]) or (np.abs(full - want[:1]) <= weight_tol(d, 2 * s) * want[:1] + 1e-9).all()


def test_weights_of_many_heads(evict):
    # enough workgroups for the form of wide key tiles
    rng = np.random.default_rng(5)
    b, heads, h, s, d = 20, 32, 16, 260, 64
    qk = normal(rng, b, heads + h, s, d)
    lens = np.array([s - 7 * i for i in range(b)], np.int32)
    want = so.attention_weights(qk[:, :heads], qk[:, heads:], lens, 0.125)
    got = evict.attention_weights(dev(qk[:, :heads]), dev(qk[:, heads:]), 0.125, lengths=dev(lens)).cpu().numpy()
    assert (np.abs(got - want) <= weight_tol(d, 2 * s) * want + 1e-9).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("s,room,first,last", [(1, 1, 0, 0), (10, 16, 2, 3), (17, 16, 2, 3), (100, 16, 16, 0), (1500, 64, 4, 60),
                                               (5000, 1000, 4, 100), (3000, 2999, 0, 0),
                                               (20, 6, 2, 4), (5000, 4500, 0, 1), (32768, 300, 0, 7), (33000, 500, 4, 100)])
@pytest.mark.parametrize("kind", ["spread", "few", "odd"])
def test_keep(evict, d, s, room, first, last, kind):
    rng = np.random.default_rng(s + room)
    b, h = 3, 2
    lens = np.array([s, max(0, s - 5), s // 2], np.int32)
    kv = normal(rng, b, s, 2, h, d)
    weight = np.exp(rng.normal(0, 2, (b, h, s))).astype(np.float32)
    if kind == "few":   # many equals
        weight = rng.integers(0, 3, (b, h, s)).astype(np.float32)
    if kind == "odd":
        weight[:, :, ::3] = np.nan
        weight[:, :, 1::7] = np.inf
        weight[:, :, 2::5] *= -1
    kc, vc = normal(rng, b, h, room, d), normal(rng, b, h, room, d)
    cw, cp = rng.random((b, h, room)).astype(np.float32), np.full((b, h, room), -9, np.int32)
    x = dev(kv)
    out = [dev(a) for a in (kc, vc, cw, cp)]
    rows = evict.keep(x[:, :, 0].transpose(1, 2), x[:, :, 1].transpose(1, 2), dev(weight), *out, first, last, lengths=dev(lens))
    rows = rows.cpu().numpy()
    for i in range(b):
        for j in range(h):
            kept = so.keep_rows(weight[i, j], int(lens[i]), room, first, last)
            m = len(kept)
            assert rows[i, j, :m].tolist() == kept and (rows[i, j, m:] == -1).all()
            kc[i, j, :m], vc[i, j, :m] = kv[i, kept, 0, j], kv[i, kept, 1, j]
            cw[i, j, :m], cp[i, j, :m] = weight[i, j, kept], kept
    for got, want in zip(out, (kc, vc, cw, cp)):
        assert np.array_equal(got.cpu().numpy(), want, equal_nan=True)


def test_refusals(evict):
    f = dict(dtype=torch.float16, device=DEV)
    q, kn, kc = torch.zeros((2, 4, 64), **f), torch.zeros((2, 2, 64), **f), torch.zeros((2, 2, 16, 64), **f)
    w, p = torch.zeros((2, 2, 16), device=DEV), torch.zeros((2, 2, 16), dtype=torch.int32, device=DEV)
    n = torch.ones(2, dtype=torch.int32, device=DEV)
    good = [q, kn, kn, kc, kc.clone(), w, p, n, 1.0, 2, 4]
    evict.attention(*good)
    for i, x in ((0, q.float()), (0, q[:, :3]), (1, kn[:1]), (2, kn.float()), (3, kc[:, :, :8]), (4, kc.cpu()), (5, w.double()),
                 (5, w[:, :1]), (6, p.long()), (7, n.long()), (7, n[:1]), (9, -1), (10, 0), (10, 15), (3, kc[:1].expand(2, -1, -1, -1))):
        with pytest.raises(ValueError):
            evict.attention(*(good[:i] + [x] + good[i + 1:]))
    with pytest.raises(ValueError):
        evict.attention(*good, out=q[:, :2])
    x, k = torch.zeros((2, 4, 30, 64), **f), torch.zeros((2, 2, 30, 64), **f)
    for args in ((x.float(), k, 1.0), (x[:, :3], k, 1.0), (x, k[:, :, :5], 1.0), (x, k, 1.0, 0), (x, k, 1.0, None, n.long()),
                 (x[..., :32], k[..., :32], 1.0)):
        with pytest.raises(ValueError):
            evict.attention_weights(*args)
    wk = torch.zeros((2, 2, 30), device=DEV)
    good = [k, k, wk, kc, kc.clone(), w, p, 2, 4]
    evict.keep(*good)
    for i, y in ((0, k[:1]), (1, k[:, :, :4]), (2, wk.half()), (2, wk[..., :3]), (3, kc.float()), (5, w[:1]), (6, p.float()), (7, -1),
                 (8, 15), (3, k[:, :, :16])):
        with pytest.raises(ValueError):
            evict.keep(*(good[:i] + [y] + good[i + 1:]))
    with pytest.raises(ValueError):
        evict.keep(*good, lengths=n.long())


def large_tol(q, k, scale, n):
    """A score is off by D 2^-24 sum |q k| scale and a few 2^-24 of itself; it and the logarithm of its row's sum bear on a weight,
    and sums of up to n exponentials (2^-23 each) by n 2^-24."""
    share = q.shape[1] // k.shape[1]
    size = max((np.abs(q[:, g].astype(np.float64)) @ np.abs(k[:, g // share].astype(np.float64)).transpose(0, 2, 1)).max()
               for g in range(q.shape[1])) * scale
    return (2 * (q.shape[-1] + 8) * size + n + 64) * 2.0 ** -24


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("s,window", [(1, None), (5, None), (40, 3), (200, None), (300, 70)])
@pytest.mark.parametrize("kind", ["opposed", "low", "large", "first"])
def test_weights_of_large_scores(evict, d, s, window, kind):
    # a lane's first score far below 0 (less than -128 in units of log2), all scores there, scores of any kind up to hundreds
    rng = np.random.default_rng(s + d)
    b, heads, h = 2, 4, 2
    q, k = normal(rng, b, heads, s, d), normal(rng, b, h, s, d)
    if kind == "opposed":  # a row's own key is what it likes least
        q = (-24 * k.repeat(heads // h, 1).astype(np.float32) + q).astype(np.float16)
    if kind == "low":
        q, k = (q / 8 - 5).astype(np.float16), (k / 8 + 5).astype(np.float16)
    if kind == "large":
        q *= 16
    if kind == "first":  # the first keys alone
        q, k[:, :, :3] = (q - 3).astype(np.float16), 8.0
    lens = np.array([s, max(1, s - 2)], np.int32)
    scale = 1 / np.sqrt(d)
    want = so.attention_weights(q, k, lens, scale, window)
    got = evict.attention_weights(dev(q), dev(k), scale, window, dev(lens)).cpu().numpy()
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= large_tol(q, k, scale, 2 * s) * want + 1e-9).all(), (np.abs(got - want) / (want + 1e-9)).max()


def test_weights_under_keys_that_are_no_numbers(evict):
    # whole steps of them in front of others: every row sees them, and no sum begins anew behind them
    rng = np.random.default_rng(7)
    q, k = normal(rng, 1, 2, 200, 64), normal(rng, 1, 2, 200, 64)
    k[:, 1, :70] = np.nan
    got = evict.attention_weights(dev(q), dev(k), 0.125).cpu().numpy()
    assert np.isfinite(got[0, 0]).all() and np.isnan(got[0, 1]).all()


def test_zeros_of_both_signs_are_equal(evict):
    # among equals the lowest row goes, and the lower one stays
    rng = np.random.default_rng(6)
    b, h, room, d = 3, 2, 90, 64
    seen = np.full(b, 300, np.int32)
    kc, vc, weight, position = state(rng, b, h, room, d, seen, 2, 5)
    weight[:] = np.where(rng.random(weight.shape) < 0.5, 0.0, -0.0)
    q, kn, vn = normal(rng, b, h, d), normal(rng, b, h, d), normal(rng, b, h, d)
    want = so.evict_step(q, kn, vn, kc, vc, weight, position, seen, 0.125, 2, 5)
    cache = [dev(x) for x in (kc, vc, weight, position)]
    _, slot = evict.attention(dev(q), dev(kn), dev(vn), *cache, dev(seen), 0.125, 2, 5)
    assert np.array_equal(slot.cpu().numpy(), want[2]) and np.array_equal(cache[3].cpu().numpy(), want[6])
    for s in (200, 33000):  # either way that rows are kept
        k, w = dev(normal(rng, b, h, s, d)), np.where(rng.random((b, h, s)) < 0.5, 0.0, -0.0).astype(np.float32)
        w[:, :, 7::50], w[:, :, 9::50] = 1.0, -1.0
        rows = evict.keep(k, k.clone(), dev(w), *cache, 3, 4).cpu().numpy()
        for i in range(b):
            for j in range(h):
                assert rows[i, j].tolist() == so.keep_rows(w[i, j], s, room, 3, 4), (s, i, j)


def test_what_many_rows_add_up_to_beside_one_large_score(evict):
    # as in test_gpu_prefix.py: a million rows of 2^-26 of the largest probability, which is given to a value of 0
    d, room = 64, 1 << 20
    kc = torch.zeros((1, 1, room, d), dtype=torch.float16, device=DEV)
    vc = torch.ones_like(kc)
    kc[:, :, 7, 0], vc[:, :, 7] = 26.0, 0.0
    weight, position = torch.zeros((1, 1, room), device=DEV), torch.arange(room, dtype=torch.int32, device=DEV).view(1, 1, room)
    q, kn, vn = (torch.zeros((1, n, d), dtype=torch.float16, device=DEV) for n in (2, 1, 1))
    q[:, :, 0], vn[:] = 1.0, 1.0
    out, _ = evict.attention(q, kn, vn, kc, vc, weight, position, torch.tensor([room], dtype=torch.int32, device=DEV), np.log(2.0), 8, 8)
    want = (room - 1) * 2.0 ** -26 / (1 + (room - 1) * 2.0 ** -26)
    assert ((out.double() - want).abs() <= TOL * want).all(), (out.min().item(), out.max().item(), want)
