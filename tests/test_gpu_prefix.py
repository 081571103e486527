"""Attention behind a shared prefix on the device against the oracle (64 bits).

Tolerance of an output: the probabilities are rounded to fp16 where they meet the values, and so is their sum's share, each by
at most 2^-11 of itself, and the result once more: 2^-11 (2 sum P |v| + |out|) <= 3 * 2^-11 sum P |v|.  Probabilities below fp16's
smallest normal number are off by at most 2^-25 of the reference's, which is at least 1 (2^-8 where it moves lazily), each:
2^-17 of |v| per 2^8 rows is below 2^-11 of the sum for the sizes here.  Scores in fp32 add below 1e-5 of the result."""
import numpy as np
import pytest
import torch

import serving_oracle as so

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOL = 3 * 2.0 ** -11 * 1.02


@pytest.fixture(scope="module")
def prefix(built_lib):
    from sqamd import prefix as m
    return m


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def normal(rng, *shape, scale=1.0):
    return (rng.normal(0, scale, shape)).astype(np.float16)


def starts_of(new):
    return torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=DEV)


def check(out, ref, size, what=""):
    out = out.float().cpu().numpy().astype(np.float64)
    bad = np.abs(out - ref) > TOL * size + 1e-6
    bad |= np.isnan(out) != np.isnan(ref)
    assert not bad.any(), "%s: %d values off, worst %.3e of %.3e" % (what, bad.sum(), np.nanmax(np.abs(out - ref) - TOL * size),
                                                                    np.nanmax(size))


def run(prefix, rng, b, heads, h, d, p, lens, new, room, ragged=True, given=True, q_scale=1.0, scale=None):
    t = sum(new)
    scale = 1 / np.sqrt(d) if scale is None else scale
    q, kn, vn = normal(rng, t, heads, d, scale=q_scale), normal(rng, t, h, d), normal(rng, t, h, d)
    kp, vp = normal(rng, h, p, d), normal(rng, h, p, d)
    kc, vc = normal(rng, b, h, room, d), normal(rng, b, h, room, d)
    ref, size, kr, vr = so.prefix_attention(q, kp, vp, kc, vc, lens, new, scale, kn if given else None, vn if given else None)
    kd, vd = dev(kc), dev(vc)
    new_rows = {"k_new": dev(kn), "v_new": dev(vn)} if given else {}
    out = prefix.attention(dev(q), dev(kp), dev(vp), kd, vd, torch.tensor(lens, dtype=torch.int32, device=DEV), scale,
                           starts=starts_of(new) if ragged else None, **new_rows)
    check(out, ref, size, (b, heads, h, d, p, lens, new))
    assert np.array_equal(kd.cpu().numpy(), kr) and np.array_equal(vd.cpu().numpy(), vr)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,h", [(4, 4), (8, 2), (5, 1), (40, 1)])
@pytest.mark.parametrize("p", [0, 1, 63, 64, 65, 700])
def test_one_token_of_each_sequence(prefix, d, heads, h, p):
    rng = np.random.default_rng(p + d + heads)
    run(prefix, rng, 3, heads, h, d, p, [1, 65, 130], [1, 1, 1], 140, ragged=False)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [[1], [5], [33], [70], [150], [1, 7, 0, 40], [3, 3, 3], [64, 1, 200], [0, 0, 1], [17] * 20])
@pytest.mark.parametrize("p", [0, 100, 257])
def test_several_tokens(prefix, d, new, p):
    rng = np.random.default_rng(sum(new) + p)
    extra = [int(rng.integers(0, 90)) for _ in new]
    lens = [n + e for n, e in zip(new, extra)]
    run(prefix, rng, len(new), 4, 2, d, p, lens, new, max(lens) + 3, ragged=True)
    if len(set(new)) == 1:
        run(prefix, rng, len(new), 4, 2, d, p, lens, new, max(lens) + 3, ragged=False, given=False)


def test_many_sequences_packed_into_tiles(prefix):
    rng = np.random.default_rng(1)
    lens = [int(x) for x in rng.integers(1, 30, 150)]
    run(prefix, rng, 150, 2, 1, 64, 513, lens, [1] * 150, 31, ragged=False)
    run(prefix, rng, 100, 3, 1, 128, 130, lens[:100], [1] * 100, 31, ragged=True)


@pytest.mark.parametrize("b,heads,h,new,p", [(70, 8, 8, 1, 500), (70, 8, 8, 1, 700), (520, 4, 1, 2, 900), (20, 8, 1, 4, 2100), (9, 4, 2, 16, 129),
                                             (2, 8, 2, 32, 300), (5, 16, 8, 60, 100)])
def test_either_side_of_each_way(prefix, b, heads, h, new, p):
    # packed or not (many sequences, short prefixes), many pieces of a long prefix, tiles of 64 and 128 rows
    rng = np.random.default_rng(b + p)
    lens = [int(x) for x in rng.integers(new, new + 70, b)]
    run(prefix, rng, b, heads, h, 64, p, lens, [new] * b, new + 70, ragged=bool(b % 2))


def test_lengths_that_fit_nothing(prefix):
    # no rows, negative lengths, more tokens than rows, more rows than room
    rng = np.random.default_rng(2)
    run(prefix, rng, 5, 2, 2, 64, 40, [0, -3, 1, 20, 33], [1, 1, 3, 2, 4], 16)
    run(prefix, rng, 5, 2, 2, 64, 0, [0, -3, 1, 20, 33], [1, 1, 3, 2, 4], 16)
    run(prefix, rng, 2, 2, 2, 128, 0, [0, 0], [70, 1], 16)


def test_large_scores(prefix):
    # the reference maximum moves often, and most probabilities vanish
    rng = np.random.default_rng(3)
    run(prefix, rng, 2, 4, 4, 64, 900, [300, 40], [2, 1], 310, q_scale=8.0)
    run(prefix, rng, 1, 4, 2, 128, 1500, [200], [130], 210, q_scale=8.0)


def test_tokens_behind_the_last_sequence_are_left(prefix):
    rng = np.random.default_rng(4)
    for new, t in (([2, 1], 9), ([90, 60], 170)):
        q, kn = dev(normal(rng, t, 2, 64)), dev(normal(rng, t, 2, 64))
        kp = dev(normal(rng, 2, 50, 64))
        kc = dev(normal(rng, 2, 2, 100, 64))
        out = torch.full((t, 2, 64), 7.0, dtype=torch.float16, device=DEV)
        got = prefix.attention(q, kp, kp, kc, kc.clone(), torch.tensor(new, dtype=torch.int32, device=DEV), 0.1,
                               starts=starts_of(new), out=out, k_new=kn, v_new=kn)
        assert got is out and (out[sum(new):] == 7).all() and not (out[:sum(new)] == 7).all(-1).any()


def test_starts_and_lengths_of_any_content(prefix):
    # whatever they hold, nothing outside the tensors is touched: rows in front of, between and behind the caches stay
    rng = np.random.default_rng(5)
    big = torch.full((4, 3, 2, 24, 64), 3.0, dtype=torch.float16, device=DEV)
    kc, vc = big[1, :, :, :16], big[2, :, :, :16]
    q, kn, kp = dev(normal(rng, 12, 4, 64)), dev(normal(rng, 12, 2, 64)), dev(normal(rng, 2, 70, 64))
    for starts in ([0, 12, 4, 2], [5, 5, 5, 5], [-7, 99, 3, 12], [12, 0, 12, 0], [2 ** 31 - 1, -2 ** 31, 6, 7]):
        for lens in ([2 ** 31 - 1, -2 ** 31, 16], [16, 17, 40], [-1, 0, 3]):
            prefix.attention(q, kp, kp, kc, vc, torch.tensor(lens, dtype=torch.int32, device=DEV), 0.1,
                             starts=torch.tensor(starts, dtype=torch.int32, device=DEV), k_new=kn, v_new=kn)
    torch.cuda.synchronize()
    assert (big[0] == 3).all() and (big[3] == 3).all() and (big[:, :, :, 16:] == 3).all()


@pytest.mark.parametrize("new", [[1, 1], [90, 70]])
def test_strides(prefix, new):
    rng = np.random.default_rng(6)
    t, heads, h, d, p, room = sum(new), 4, 2, 128, 130, 200
    lens = [n + 20 for n in new]
    qkv = normal(rng, t, heads + 2 * h, d)
    rows = normal(rng, p, 2, h, d)            # a prefix as a fused projection left it
    caches = normal(rng, 2, room, 2, h, d)    # [sequence, row, k or v, head]
    x, r, c = dev(qkv), dev(rows), dev(caches)
    ref, size, kr, vr = so.prefix_attention(qkv[:, :heads], rows[:, 0].transpose(1, 0, 2), rows[:, 1].transpose(1, 0, 2),
                                            caches[:, :, 0].transpose(0, 2, 1, 3), caches[:, :, 1].transpose(0, 2, 1, 3), lens, new,
                                            0.08, qkv[:, heads:heads + h], qkv[:, heads + h:])
    kc, vc = c[:, :, 0].transpose(1, 2), c[:, :, 1].transpose(1, 2)
    out = prefix.attention(x[:, :heads], r[:, 0].transpose(0, 1), r[:, 1].transpose(0, 1), kc, vc,
                           torch.tensor(lens, dtype=torch.int32, device=DEV), 0.08, starts=starts_of(new),
                           k_new=x[:, heads:heads + h], v_new=x[:, heads + h:])
    check(out, ref, size)
    assert np.array_equal(kc.cpu().numpy(), kr) and np.array_equal(vc.cpu().numpy(), vr)
    # what cannot be read as it lies is copied: queries, new rows and prefix at odd addresses, values strided otherwise
    odd = torch.empty(x.numel() + 1, dtype=torch.float16, device=DEV)[1:].view_as(x).copy_(x)
    again = prefix.attention(odd[:, :heads], r[:, 0].transpose(0, 1), r[:, 1].transpose(0, 1).contiguous(), kc, vc,
                             torch.tensor(lens, dtype=torch.int32, device=DEV), 0.08, starts=starts_of(new),
                             k_new=odd[:, heads:heads + h], v_new=odd[:, heads + h:].contiguous())
    assert torch.equal(again, out)


@pytest.mark.parametrize("new", [[40], [100, 20]])
def test_infinities_and_nan_reach_those_that_see_them_alone(prefix, new):
    rng = np.random.default_rng(7)
    t, h, d, p = sum(new), 2, 64, 70
    q, kn, vn = normal(rng, t, h, d), normal(rng, t, h, d), normal(rng, t, h, d)
    kp, vp = normal(rng, h, p, d), normal(rng, h, p, d)
    kc, vc = normal(rng, len(new), h, 120, d), normal(rng, len(new), h, 120, d)
    vn[30, 0, 5], vn[35, 1, 63], kn[33, 1, 0], vn[new[0] - 1, 0, 9] = np.inf, np.nan, np.nan, -np.inf
    kc[:, :, new[0]:], vc[:, :, new[0]:] = np.nan, np.nan  # rows behind the last
    with np.errstate(invalid="ignore"):
        ref, size, _, _ = so.prefix_attention(q, kp, vp, kc, vc, new, new, 0.125, kn, vn)
        out = prefix.attention(dev(q), dev(kp), dev(vp), dev(kc), dev(vc), torch.tensor(new, dtype=torch.int32, device=DEV), 0.125,
                               starts=starts_of(new), k_new=dev(kn), v_new=dev(vn)).float().cpu().numpy()
    assert np.array_equal(np.isfinite(out), np.isfinite(ref))
    assert np.array_equal(out == np.inf, ref == np.inf) and np.array_equal(out == -np.inf, ref == -np.inf)
    fine = np.isfinite(ref)
    assert (np.abs(out[fine] - ref[fine]) <= TOL * size[fine] + 1e-6).all()


def test_captured_steps_follow_the_device(prefix):
    rng = np.random.default_rng(8)
    b, heads, h, d, p, room = 3, 4, 2, 128, 300, 90
    kp, vp = dev(normal(rng, h, p, d)), dev(normal(rng, h, p, d))
    caches = [dev(normal(rng, b, h, room, d)) for _ in range(2)]
    lengths = torch.tensor([1, 30, 60], dtype=torch.int32, device=DEV)
    qkv = dev(normal(rng, b, heads + 2 * h, d))

    def step(kc, vc):
        return prefix.attention(qkv[:, :heads], kp, vp, kc, vc, lengths, 0.09, k_new=qkv[:, heads:heads + h], v_new=qkv[:, heads + h:])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*(c.clone() for c in caches))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(*caches)
    twin = [c.clone() for c in caches]
    for i in range(5):
        qkv.copy_(dev(normal(rng, b, heads + 2 * h, d)))
        want = step(*twin).clone()
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(out, want) and all(torch.equal(a, c) for a, c in zip(caches, twin)), i
        lengths += 1


def test_two_streams_at_once(prefix):
    rng = np.random.default_rng(9)
    args = []
    for i in range(2):
        args.append((dev(normal(rng, 16, 8, 128)), dev(normal(rng, 2, 2000, 128)), dev(normal(rng, 2, 2000, 128)),
                     dev(normal(rng, 16, 2, 300, 128)), dev(normal(rng, 16, 2, 300, 128)),
                     torch.full((16,), 300, dtype=torch.int32, device=DEV), 0.09))
    want = [prefix.attention(*a).clone() for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(prefix.attention(*args[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


@pytest.mark.parametrize("b,new,p", [(16, 1, 700), (1, 1, 2000), (3, 200, 300)])
def test_the_result_in_the_place_of_the_queries(prefix, b, new, p):
    rng = np.random.default_rng(b)
    q, rows = dev(normal(rng, b * new, 8, 64)), [dev(normal(rng, 2, p, 64)) for _ in range(2)]
    caches = [dev(normal(rng, b, 2, 320, 64)) for _ in range(2)]
    lengths = torch.full((b,), 300, dtype=torch.int32, device=DEV)
    want = prefix.attention(q, *rows, *caches, lengths, 0.125)
    assert prefix.attention(q, *rows, *caches, lengths, 0.125, out=q) is q and torch.equal(q, want)


def test_refusals(prefix):
    q = torch.zeros((4, 4, 64), dtype=torch.float16, device=DEV)
    kp = torch.zeros((2, 10, 64), dtype=torch.float16, device=DEV)
    kc = torch.zeros((4, 2, 8, 64), dtype=torch.float16, device=DEV)
    kn = torch.zeros((4, 2, 64), dtype=torch.float16, device=DEV)
    n = torch.ones(4, dtype=torch.int32, device=DEV)
    bad = [((q.float(), kp, kp, kc, kc, n, 1.0), {}), ((q, kp.cpu(), kp, kc, kc, n, 1.0), {}), ((q, kp, kp[:, :5], kc, kc, n, 1.0), {}),
           ((q, kp[:1], kp[:1], kc, kc, n, 1.0), {}), ((q, kp, kp, kc, kc[:, :, :4], n, 1.0), {}), ((q, kp, kp, kc, kc, n.long(), 1.0), {}),
           ((q, kp, kp, kc, kc, n[:3], 1.0), {}), ((q[:3], kp, kp, kc, kc, n, 1.0), {}), ((q, kp, kp, kc, kc, n, 1.0), {"k_new": kn}),
           ((q, kp, kp, kc, kc, n, 1.0), {"starts": n}), ((q, kp, kp, kc, kc, n, 1.0), {"k_new": kn, "v_new": kn[:3]}),
           ((q[:, :3], kp, kp, kc, kc, n, 1.0), {}), ((q[..., :32], kp[..., :32], kp[..., :32], kc[..., :32], kc[..., :32], n, 1.0), {}),
           ((q, kp, kp, kc, kc, n, 1.0), {"out": q[:, :2]}), ((q, kp, kp, kc, kc, n, 1.0), {"out": q.float()}),
           ((q, kp, kp, kc[:1].expand(4, -1, -1, -1), kc, n, 1.0), {"k_new": kn, "v_new": kn}),
           ((q, kp, kp, kc.transpose(2, 3)[..., :8, :], kc.transpose(2, 3), n, 1.0), {})]
    for args, kw in bad:
        with pytest.raises(ValueError):
            prefix.attention(*args, **kw)
    empty = prefix.attention(q[:0], kp, kp, kc[:0], kc[:0], n[:0], 1.0)
    assert empty.shape == (0, 4, 64)


@pytest.mark.parametrize("heads,h,new,before,p", [
    (2, 2, [65], 0, 70), (2, 2, [65], 30, 0), (70, 1, [1], 40, 70), (64, 8, [129], 20, 65), (2, 2, [70, 129], 5, 10), (2, 2, [100], 90, 0)])
def test_infinities_and_nan_in_front_of_a_tile_of_one_token(prefix, heads, h, new, before, p):
    # the last tile's rows are one token's (or tokens that see equally many rows, those that the cache has room for): it sees
    # every row of its last step
    rng = np.random.default_rng(sum(new) + heads)
    t, d, room = sum(new), 64, 150
    q, kn, vn = normal(rng, t, heads, d), normal(rng, t, h, d), normal(rng, t, h, d)
    kp, vp = normal(rng, h, p, d), normal(rng, h, p, d)
    kc, vc = normal(rng, len(new), h, room, d), normal(rng, len(new), h, room, d)
    lens, at = [n + before for n in new], 0
    for i, n in enumerate(new):
        last = min(lens[i], room) - 1  # the last row that is seen
        for row, value in ((last, np.inf), (last // 64 * 64, np.nan), (max(last - 2, 0), -np.inf)):
            rows, j = (vn, at + row - before) if row >= before else (vc[i].transpose(1, 0, 2), row)
            rows[j, 0, 3 + row % 7] = value
        at += n
    with np.errstate(invalid="ignore"):
        ref, size, _, _ = so.prefix_attention(q, kp, vp, kc, vc, lens, new, 0.125, kn, vn)
        out = prefix.attention(dev(q), dev(kp), dev(vp), dev(kc), dev(vc), torch.tensor(lens, dtype=torch.int32, device=DEV), 0.125,
                               starts=starts_of(new), k_new=dev(kn), v_new=dev(vn)).float().cpu().numpy()
    assert not np.isfinite(ref).all()
    assert np.array_equal(np.isfinite(out), np.isfinite(ref))
    assert np.array_equal(out == np.inf, ref == np.inf) and np.array_equal(out == -np.inf, ref == -np.inf)
    fine = np.isfinite(ref)
    assert (np.abs(out[fine] - ref[fine]) <= TOL * size[fine] + 1e-6).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,heads,h,new,p,ragged,given", [
    (9, 16, 8, 130, 0, False, True), (9, 16, 8, 130, 100, True, True), (9, 16, 8, 130, 257, False, False), (5, 40, 8, 70, 300, True, False),
    (36, 8, 8, 130, 300, False, True), (36, 8, 8, 130, 300, True, True)])
def test_prompts_in_tiles_of_128_rows(prefix, d, b, heads, h, new, p, ragged, given):
    # more than 64 rows of a sequence and more than 64 such tiles of all heads; with 36 sequences more than 512, of which the last
    # are cut into parts (576 of equally many tokens, fewer of ragged ones)
    rng = np.random.default_rng(b + p + d)
    tokens = [new] * b if not ragged else [new if i % 3 else int(rng.integers(1, 2 * new)) for i in range(b)]
    lens = [n + int(rng.integers(0, 90)) for n in tokens]
    run(prefix, rng, b, heads, h, d, p, lens, tokens, max(lens) + 5, ragged=ragged, given=given)


def test_prompts_in_tiles_of_128_rows_with_large_scores(prefix):
    rng = np.random.default_rng(11)
    run(prefix, rng, 9, 16, 8, 64, 200, [150 + i for i in range(9)], [130] * 9, 170, q_scale=8.0)


def test_infinities_and_nan_under_tiles_of_128_rows(prefix):
    rng = np.random.default_rng(12)
    b, heads, h, new, p, d = 9, 16, 8, 130, 70, 64
    t = b * new
    q, kn, vn = normal(rng, t, heads, d), normal(rng, t, h, d), normal(rng, t, h, d)
    kp, vp = normal(rng, h, p, d), normal(rng, h, p, d)
    kc, vc = np.full((2, b, h, 140, d), np.nan, np.float16)
    vn[30, 0, 5], vn[new + 70, 1, 63], kn[33, 2, 0], vn[2 * new - 1, 0, 9] = np.inf, np.nan, np.nan, -np.inf
    with np.errstate(invalid="ignore"):
        ref, size, _, _ = so.prefix_attention(q, kp, vp, kc, vc, [new] * b, [new] * b, 0.125, kn, vn)
        out = prefix.attention(dev(q), dev(kp), dev(vp), dev(kc), dev(vc), torch.full((b,), new, dtype=torch.int32, device=DEV), 0.125,
                               k_new=dev(kn), v_new=dev(vn)).float().cpu().numpy()
    assert np.array_equal(np.isfinite(out), np.isfinite(ref)) and np.array_equal(out == np.inf, ref == np.inf)
    fine = np.isfinite(ref)
    assert (np.abs(out[fine] - ref[fine]) <= TOL * size[fine] + 1e-6).all()


def test_what_many_rows_add_up_to_beside_one_large_score(prefix):
    # one row of the largest score, and so many others of 2^-26 of its probability that they make a hundredth of the sum
    d, h, p = 64, 1, 1 << 20
    kp = torch.zeros((h, p, d), dtype=torch.float16, device=DEV)
    vp = torch.ones((h, p, d), dtype=torch.float16, device=DEV)
    kp[:, 7, 0], vp[:, 7] = 26.0, 0.0
    kc = torch.zeros((1, h, 40, d), dtype=torch.float16, device=DEV)
    for t, heads in ((1, 1), (33, 2), (40, 4)):
        q = torch.zeros((t, heads, d), dtype=torch.float16, device=DEV)
        q[:, :, 0] = 1.0
        got = prefix.attention(q, kp, vp, kc, kc, torch.zeros(1, dtype=torch.int32, device=DEV), np.log(2.0)).double()
        want = (p - 1) * 2.0 ** -26 / (1 + (p - 1) * 2.0 ** -26)
        assert ((got - want).abs() <= TOL * want).all(), (t, heads, got.min().item(), got.max().item(), want)
