"""The 4-bit key/value cache on the device against the oracle (64 bits; codes and scales bit for bit)."""
import numpy as np
import pytest
import torch

import kv4_oracle as ko

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SIZES = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)]


@pytest.fixture(scope="module")
def kv4(built_lib):
    from sqamd import kv4 as m
    return m


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def random_pool(rng, pages, h, d, g, magnitude=1.0):
    """Records as of rows of normal numbers: any codes, scales in (0.2, 0.4), minima about -7.5 scales."""
    rec = rng.integers(0, 256, (pages, h, ko.record_bytes(d, g)), dtype=np.uint8)
    n = 2 * (d // g) * 16
    s = rng.uniform(0.2, 0.4, (pages, h, n, 1, 4)) * magnitude
    m = rng.normal(0, 0.3, (pages, h, n, 1, 4)) * magnitude - 7.5 * s
    rec[..., 64 * d:64 * d + 16 * n] = np.concatenate([s, m], -2).astype(np.float16).reshape(pages, h, -1).view(np.uint8)
    b = np.sort(rng.normal(0, 2, (pages, h, 2, d)), 2)[:, :, ::-1]
    rec[..., -4 * d:] = np.ascontiguousarray(b.astype(np.float16)).reshape(pages, h, -1).view(np.uint8)
    return rec


def tables(rng, lens, spare=2, width=None):
    counts = [(max(n, 0) + 63) // 64 for n in lens]
    order = rng.permutation(sum(counts) + spare).astype(np.int32)
    pages = np.full((len(lens), width if width is not None else max(counts + [1])), -1, dtype=np.int32)
    at = 0
    for i, c in enumerate(counts):
        pages[i, :c] = order[at:at + c]
        at += c
    return pages, sum(counts) + spare


def starts_of(new):
    return np.concatenate([[0], np.cumsum(new)]).astype(np.int32)


# ----------------------------------------------------------------------------------------------------------- append

def expect_append(pool, k, v, pages, lens, new, d, g):
    """The oracle's records after the call, by fields, and which (page, row) were written."""
    fields = ko.read(pool, d, g)
    written = np.zeros((pool.shape[0], 64), dtype=bool)
    t = 0
    for b, (n, c) in enumerate(zip(lens, new)):
        for pos in range(n - c, n):
            kt, vt = k[t], v[t]
            t += 1
            if pos < 0 or pos >= 64 * pages.shape[1] or not 0 <= pages[b, pos // 64] < pool.shape[0]:
                continue
            page, r = pages[b, pos // 64], pos % 64
            written[page, r] = True
            for x, names in ((kt, ("kc", "ks", "km")), (vt, ("vc", "vs", "vm"))):
                for name, val in zip(names, ko.quantise(x, g)):
                    fields[name][page, :, r] = val
            hi, lo = fields["bounds"][page, :, 0], fields["bounds"][page, :, 1]
            fields["bounds"][page, :, 0] = kt if r == 0 else np.fmax(hi, kt)
            fields["bounds"][page, :, 1] = kt if r == 0 else np.fmin(lo, kt)
    return fields, written


@pytest.mark.parametrize("d,g", SIZES)
@pytest.mark.parametrize("h,lens,new,equal", [
    (1, [1], [1], True),
    (3, [64, 65, 1, 200], [1, 1, 1, 1], True),
    (2, [5, 70], [5, 5], True),
    (8, [130, 64, 63, 300], [130, 64, 63, 70], False),
    (2, [129, 500, 7], [0, 2, 7], False),
    (32, [640] * 8, [1] * 8, True),
], ids=["one", "page-edges", "five-each", "prompts", "none-of-one", "step"])
def test_append(kv4, d, g, h, lens, new, equal):
    rng = np.random.default_rng(d + g + h + len(lens))
    pages, total = tables(rng, lens)
    pool = random_pool(rng, total, h, d, g)
    t = sum(new)
    kv = rng.normal(0, 1, (t, 2, h, d)).astype(np.float16)
    kv[:, 0, :, ::17] *= 6  # keys with large channels
    dkv, dpool = dev(kv), dev(pool)
    k_hat, v_hat = kv4.append(dkv[:, 0], dkv[:, 1], dpool, dev(pages), dev(np.array(lens, dtype=np.int32)),
                              None if equal else dev(starts_of(new)), values=True)
    want, written = expect_append(pool, kv[:, 0], kv[:, 1], pages, lens, new, d, g)
    got = dpool.cpu().numpy()
    fields = ko.read(got, d, g)
    for name in want:
        assert np.array_equal(fields[name], want[name]), name
    untouched = [p for p in range(total) if not written[p].any()]
    assert np.array_equal(got[untouched], pool[untouched])
    for i, (hat, n3) in enumerate(((k_hat, ("kc", "ks", "km")), (v_hat, ("vc", "vs", "vm")))):
        c, s, m = ko.quantise(kv[:, i], g)
        assert np.array_equal(hat.cpu().numpy(), (s.astype(np.float32) * c + m.astype(np.float32)).astype(np.float16))


def test_append_of_awkward_rows(kv4):
    # constant rows, ranges below the smallest scale, the largest numbers, infinities, NaN, denormals
    d, g, h = 64, 32, 1
    x = np.zeros((9, 1, d), dtype=np.float16)
    x[0] = 3.25
    x[1, 0, :32] = np.linspace(0, 2 ** -23, 32)
    x[2, 0, ::2], x[2, 0, 1::2] = 65504, -65504
    x[3, 0, 5] = np.inf
    x[4, 0, 40] = np.nan
    x[5, 0, :] = -np.float16(6e-8) * np.arange(d)
    x[6, 0, :] = np.arange(d) / 16
    x[7, 0, 3] = -np.inf
    x[8, 0, :] = -2.0
    pool = random_pool(np.random.default_rng(0), 1, h, d, g)
    dpool, dx = dev(pool), dev(x)
    k_hat, v_hat = kv4.append(dx, dx.clone(), dpool, dev(np.zeros((1, 1), np.int32)), dev(np.array([9], np.int32)), values=True)
    f = ko.read(dpool.cpu().numpy(), d, g)
    c, s, m = ko.quantise(x, g)
    clean = np.isfinite(x).reshape(9, 1, 2, 32).all(-1).repeat(32, -1)[:, 0]
    for kind, hat in (("k", k_hat), ("v", v_hat)):
        with np.errstate(invalid="ignore"):
            got = ko.values(f[kind + "c"], f[kind + "s"], f[kind + "m"])[0, 0, :9]
            want = ko.values(c, s, m)[:, 0]
        assert np.array_equal(got[clean], want[clean])
        assert np.all(np.isnan(got[~clean])) and np.all(np.isnan(want[~clean]))
        hat = hat.cpu().numpy()[:, 0]
        with np.errstate(over="ignore"):  # 65504 reads as a little more: infinite in fp16
            assert np.all(np.isnan(hat[~clean])) and np.array_equal(hat[clean], want[clean].astype(np.float32).astype(np.float16))


def test_append_leaves_out_what_has_no_page(kv4):
    d, g, h = 128, 64, 2
    rng = np.random.default_rng(5)
    pages = np.array([[0, 7, 2], [-1, 3, 2 ** 31 - 1], [4, 4, 4], [-2 ** 31, 5, 6]], dtype=np.int32)
    lens, new = [300, 130, 2, 70], [290, 130, 6, 70]  # beyond the table, pages outside the pool, rows before the first
    pool = random_pool(rng, 7, h, d, g)
    t = sum(new)
    k, v = (rng.normal(0, 1, (t + 3, h, d)).astype(np.float16) for _ in range(2))
    dpool = dev(pool)
    dk, dv = dev(k), dev(v)
    st = starts_of(new)
    hats = torch.full((2, t + 3, h, d), 7.0, dtype=torch.float16, device=DEV)
    import ctypes
    from sqamd import capi
    strides = (ctypes.c_long * 4)(h * d, d, h * d, d)
    p = capi._ptr
    keep = [dev(pages), dev(np.array(lens, np.int32)), dev(st)]
    assert capi.lib().sq_kv4_append(p(dk), p(dv), p(hats[0]), p(hats[1]), p(dpool), p(keep[0]), p(keep[1]), p(keep[2]), t + 3, 4,
                                    h, d, g, 7, 3, 3, strides, capi._stream()) == 0
    want, written = expect_append(pool, k, v, pages, lens, new, d, g)
    got = dpool.cpu().numpy()
    fields = ko.read(got, d, g)
    for name in want:
        assert np.array_equal(fields[name], want[name]), name
    placed = np.zeros(t + 3, dtype=bool)
    at = 0
    for b, (n, c) in enumerate(zip(lens, new)):
        for pos in range(n - c, n):
            placed[at] = 0 <= pos < 192 and 0 <= pages[b, pos // 64] < 7
            at += 1
    assert torch.all(hats[:, dev(~placed)] == 7.0) and not torch.any(torch.all(hats[:, dev(placed)].flatten(2) == 7.0, -1))


def test_append_reads_any_strides(kv4):
    d, g, h = 128, 32, 4
    rng = np.random.default_rng(6)
    base = rng.normal(0, 1, (5, 3, h, d + 4)).astype(np.float16)
    x = dev(base)
    views = [x[:, 0, :, :d], x[:, 1, :, 1:d + 1], x[:, 2, :, :d].transpose(0, 1).contiguous().transpose(0, 1), x.flip(-1)[:, 0, :, :d]]
    pages, lens = dev(np.zeros((1, 1), np.int32)), dev(np.array([5], np.int32))
    for k in views:
        a, b = kv4.new_pool(1, h, d, g), kv4.new_pool(1, h, d, g)
        a.zero_(), b.zero_()
        v = k * 2
        kv4.append(k, k, a, pages, lens)
        kv4.append(k.contiguous().clone(), k.contiguous().clone(), b, pages, lens)
        assert torch.equal(a, b)
        kv4.append(k, v, a, pages, lens)
        assert not torch.equal(a, b)


# -------------------------------------------------------------------------------------------------------- attention

def check_attention(kv4, rng, d, g, h, share, lens, new, equal, magnitude=1.0, scale=None, ws=True):
    pages, total = tables(rng, lens)
    pool = random_pool(rng, total, h, d, g, magnitude)
    t, scale = sum(new), scale if scale is not None else d ** -0.5
    q = rng.normal(0, 1, (t, h * share, d)).astype(np.float16)
    out = kv4.attention(dev(q), dev(pool), dev(pages), dev(np.array(lens, np.int32)), scale,
                        None if equal else dev(starts_of(new))).cpu().numpy().astype(np.float64)
    compare(out, q, pool, pages, lens, new, d, g, h, share, scale)


def compare(out, q, pool, pages, lens, new, d, g, h, share, scale, few=24, middles=0.0):
    """Every output of up to `few` tokens of a sequence (the first, the last and some between)."""
    at = 0
    for b, (n, c) in enumerate(zip(lens, new)):
        tokens = range(c) if c <= few else sorted({0, 1, 2, c - 1, c - 2} | set(range(0, c, c // (few - 4))))
        for head in range(h):
            rows = ko.Rows(pool, pages[b, :(max(n, 0) + 63) // 64], max(n, 0), head, d, g)
            for i in tokens:
                seen = np.arange(max(0, min(n - c + i + 1, max(n, 0))))
                for j in range(head * share, (head + 1) * share):
                    want, tol = ko.attend(rows, q[at + i, j].astype(np.float64), scale, seen, middles)
                    err = np.abs(out[at + i, j] - want)
                    assert np.all(err <= tol), "sequence %d token %d head %d: %.3g of %.3g" % (
                        b, i, j, err[np.argmax(err - tol)], tol[np.argmax(err - tol)])
        at += c


@pytest.mark.parametrize("d,g", SIZES)
@pytest.mark.parametrize("h,share,lens", [
    (1, 1, [1]), (2, 1, [31, 32, 33, 64, 65]), (2, 4, [640]), (8, 1, [100] * 4), (1, 7, [129, 5, 1000]), (3, 16, [257]),
    (1, 40, [77, 300]), (2, 8, [5000, 1, 63]),
], ids=["one-row", "edges", "640", "unshared", "seven", "sixteen", "forty", "split"])
def test_attention_of_one_token(kv4, d, g, h, share, lens):
    check_attention(kv4, np.random.default_rng(d + g + share), d, g, h, share, lens, [1] * len(lens), True)


@pytest.mark.parametrize("d,g", [(64, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("h,share,lens,new,equal", [
    (2, 4, [300, 64, 4], [4, 4, 4], True),
    (1, 1, [200], [200], True),
    (2, 5, [700, 90], [33, 90], False),
    (1, 8, [1500, 3, 128, 2], [100, 0, 128, 1], False),
    (1, 2, [2000], [500], True),
], ids=["drafts", "prompt", "ragged", "one-empty", "chunk"])
def test_attention_of_several_tokens(kv4, d, g, h, share, lens, new, equal):
    check_attention(kv4, np.random.default_rng(7 * d + g), d, g, h, share, lens, new, equal)


@pytest.mark.parametrize("magnitude,scale", [(1e-3, 0.1), (200.0, 1e-3), (1.0, 2.0), (1.0, 0.0), (1.0, -0.3)])
def test_attention_at_other_magnitudes(kv4, magnitude, scale):
    check_attention(kv4, np.random.default_rng(3), 128, 64, 2, 4, [700, 65], [1, 1], True, magnitude, scale)
    check_attention(kv4, np.random.default_rng(4), 64, 32, 1, 4, [500], [70], True, magnitude, scale)


def test_scales_of_very_different_size(kv4):
    # the power of two in P' follows the scales: rows of 1e-4 before rows of 100, and the other way round
    d, g, h = 128, 64, 1
    rng = np.random.default_rng(9)
    for order in (1, -1):
        pool = np.concatenate([random_pool(rng, 1, h, d, g, m) for m in (1e-4, 1e-2, 1.0, 100.0)][::order])
        pages, lens = np.arange(4, dtype=np.int32)[None], [256]
        for c in (1, 40):
            q = rng.normal(0, 0.01, (c, 4, d)).astype(np.float16)
            out = kv4.attention(dev(q), dev(pool), dev(pages), dev(np.array(lens, np.int32)), 0.1).cpu().numpy()
            compare(out.astype(np.float64), q, pool, pages, lens, [c], d, g, h, 4, 0.1)


@pytest.mark.parametrize("c,share,middles", [(1, 4, 0.0), (5, 4, 0.0), (70, 4, 2.0 ** -11)], ids=["one", "five", "many"])
def test_values_far_from_zero(kv4, c, share, middles):
    # minima of 40 and scales of 0.3: the middle of a group is 30 times its spread (with many rows it is held in fp16)
    d, g, h = 128, 64, 1
    rng = np.random.default_rng(31)
    lens = [700, 130]
    pages, total = tables(rng, lens)
    pool = random_pool(rng, total, h, d, g)
    sm = pool[..., 64 * d:64 * d + 512 * (d // g)].view(np.float16).reshape(total, h, 2, d // g, 16, 2, 4)
    sm[:, :, 0, :, :, 1] += np.float16(3)
    sm[:, :, 1, :, :, 1] += np.float16(40)
    pool[..., 64 * d:64 * d + 512 * (d // g)] = sm.reshape(total, h, -1).view(np.uint8)
    q = rng.normal(0, 1, (2 * c, share * h, d)).astype(np.float16)
    out = kv4.attention(dev(q), dev(pool), dev(pages), dev(np.array(lens, np.int32)), 0.1).cpu().numpy().astype(np.float64)
    compare(out, q, pool, pages, lens, [c, c], d, g, h, share, 0.1, middles=middles)


@pytest.mark.parametrize("d,g,h,share,tokens", [(64, 32, 2, 1, "one"), (128, 64, 1, 4, "one"), (64, 64, 1, 2, "few"),
                                                 (128, 128, 1, 1, "chunks"), (64, 32, 2, 6, "drafts")])
def test_many_sequences(kv4, d, g, h, share, tokens):
    # more sequences than a wave has lanes: where a workgroup's piece lies is found over several rounds of 64
    rng = np.random.default_rng(d + share)
    b = 150
    lens = rng.integers(0, 200, b).tolist()
    lens[3], lens[70], lens[149] = 0, 4000, 2500  # two of them are dealt to several workgroups
    if tokens in ("one", "drafts"):
        new = [1 if tokens == "one" else 3] * b
    elif tokens == "few":
        new = [int(x) for x in rng.integers(0, 6, b)]
    else:
        new = [int(min(x, n)) for x, n in zip(rng.integers(60, 150, b), lens)]
    pages, total = tables(rng, lens)
    pool = random_pool(rng, total, h, d, g)
    q = rng.normal(0, 1, (sum(new), h * share, d)).astype(np.float16)
    out = kv4.attention(dev(q), dev(pool), dev(pages), dev(np.array(lens, np.int32)), d ** -0.5,
                        None if tokens in ("one", "drafts") else dev(starts_of(new))).cpu().numpy().astype(np.float64)
    few = {"chunks": 8}.get(tokens, 24)
    compare(out, q, pool, pages, lens, new, d, g, h, share, d ** -0.5, few)


@pytest.mark.parametrize("d,g,h,share,singles,others", [
    (128, 64, 2, 4, 30, [(3000, 400), (70, 9), (40, 8), (5, 0), (9, 9)]), (64, 32, 1, 1, 20, [(1200, 1100), (33, 33), (32, 32), (400, 31), (0, 0)]),
    (128, 128, 1, 16, 5, [(200, 40), (90, 2), (91, 3)]), (64, 64, 1, 32, 3, [(100, 6), (2500, 1), (60, 2)]),
    (64, 64, 1, 33, 3, [(100, 6), (2500, 1), (60, 2)])], ids=["four", "one", "sixteen", "widest", "too-wide"])
def test_prompts_beside_single_tokens(kv4, d, g, h, share, singles, others):
    # few and many rows in one call: the sequences are dealt to two kernels by their rows, each once
    rng = np.random.default_rng(38)
    lens = rng.integers(1, 1500, singles).tolist() + [n for n, _ in others]
    new = [1] * singles + [c for _, c in others]
    order = rng.permutation(len(lens))
    lens, new = [int(lens[i]) for i in order], [int(new[i]) for i in order]
    assert 32 < (sum(new) * share + len(new) - 1) // len(new) <= 256
    pages, total = tables(rng, lens)
    pool = random_pool(rng, total, h, d, g)
    t = sum(new)
    q = rng.normal(0, 1, (t + 2, h * share, d)).astype(np.float16)
    out = torch.full(q.shape, 9.0, dtype=torch.float16, device=DEV)
    kv4.attention(dev(q), dev(pool), dev(pages), dev(np.array(lens, np.int32)), d ** -0.5, dev(starts_of(new)), out=out)
    out = out.cpu().numpy().astype(np.float64)
    assert np.all(out[t:] == 9.0)
    compare(out, q, pool, pages, lens, new, d, g, h, share, d ** -0.5)


def test_append_to_many_sequences(kv4):
    d, g, h, b = 64, 32, 2, 150
    rng = np.random.default_rng(33)
    lens = rng.integers(1, 300, b).tolist()
    new = [int(min(n, x)) for n, x in zip(lens, rng.integers(0, 100, b))]
    pages, total = tables(rng, lens)
    pool = random_pool(rng, total, h, d, g)
    k, v = (rng.normal(0, 1, (sum(new), h, d)).astype(np.float16) for _ in range(2))
    dpool = dev(pool)
    kv4.append(dev(k), dev(v), dpool, dev(pages), dev(np.array(lens, np.int32)), dev(starts_of(new)))
    want, _ = expect_append(pool, k, v, pages, lens, new, d, g)
    fields = ko.read(dpool.cpu().numpy(), d, g)
    for name in want:
        assert np.array_equal(fields[name], want[name]), name


def test_one_table_row_for_several_sequences(kv4):
    # samples of one prompt: the same pages, lengths of their own; the row need not be repeated in memory
    d, g, h, share = 64, 64, 2, 4
    rng = np.random.default_rng(34)
    pages, total = tables(rng, [500])
    pool, n = dev(random_pool(rng, total, h, d, g)), dev(np.array([500, 129, 64], np.int32))
    q = dev(rng.normal(0, 1, (3, h * share, d)).astype(np.float16))
    one = dev(pages).expand(3, -1)
    assert torch.equal(kv4.attention(q, pool, one, n, 0.1), kv4.attention(q, pool, one.contiguous(), n, 0.1))
    assert torch.equal(kv4.select_pages(q, pool, one, n, 3), kv4.select_pages(q, pool, one.contiguous(), n, 3))
    with pytest.raises(ValueError):
        kv4.attention(q, pool, one, n[:1].expand(3), 0.1)


def test_tokens_that_see_nothing_and_tokens_of_no_sequence(kv4):
    d, g, h, share = 128, 64, 2, 2
    rng = np.random.default_rng(10)
    lens, new = [0, 3, 70, -5], [2, 5, 1, 1]
    pages, total = tables(rng, lens, width=2)
    pool = random_pool(rng, total, h, d, g)
    q = rng.normal(0, 1, (sum(new) + 4, h * share, d)).astype(np.float16)
    out = torch.full(q.shape, 9.0, dtype=torch.float16, device=DEV)
    got = kv4.attention(dev(q), dev(pool), dev(pages), dev(np.array(lens, np.int32)), 0.1, dev(starts_of(new)), out=out)
    assert got is out
    out = out.cpu().numpy().astype(np.float64)
    compare(out, q, pool, pages, lens, new, d, g, h, share, 0.1)
    assert np.all(out[:4] == 0) and np.all(out[8:9] == 0) and np.all(out[9:] == 9.0)


def test_what_nobody_sees_may_hold_anything(kv4):
    # rows behind the last one, pages of no sequence, rows a token does not see yet: NaN scales there reach no output
    d, g, h, share = 128, 32, 1, 4
    rng = np.random.default_rng(11)
    for lens, new in (([70, 33], [1, 1]), ([70, 200], [30, 150])):
        pages, total = tables(rng, lens)
        pool = random_pool(rng, total, h, d, g)
        q = rng.normal(0, 1, (sum(new), share, d)).astype(np.float16)
        st = dev(starts_of(new))
        args = (dev(pages), dev(np.array(lens, np.int32)), 0.1, st)
        before = kv4.attention(dev(q), dev(pool), *args)
        bad = pool.copy()
        view = bad[..., 64 * d:64 * d + 512 * (d // g)].view(np.float16).reshape(total, h, 2, d // g, 16, 2, 4)
        used = set()
        for b, n in enumerate(lens):
            used |= set(pages[b, :(n + 63) // 64].tolist())
            for r in range(n, (n + 63) // 64 * 64):
                view[pages[b, r // 64], ..., r % 64 // 4, :, r % 4] = [np.nan, np.inf, -np.inf][r % 3]
        for p in set(range(total)) - used:
            bad[p] = 255
        bad[..., 64 * d:64 * d + 512 * (d // g)] = view.reshape(total, h, -1).view(np.uint8)
        assert torch.equal(kv4.attention(dev(q), dev(bad), *args), before)
        # the last row of the second sequence: only its last token sees it
        r = lens[1] - 1
        view[pages[1, r // 64], ..., r % 64 // 4, :, r % 4] = np.nan
        bad[..., 64 * d:64 * d + 512 * (d // g)] = view.reshape(total, h, -1).view(np.uint8)
        after = kv4.attention(dev(q), dev(bad), *args)
        assert torch.equal(after[:-1], before[:-1]) and torch.all(torch.isnan(after[-1]))


def test_pages_outside_the_pool_are_not_seen(kv4):
    d, g, h = 64, 64, 2
    rng = np.random.default_rng(12)
    pool = random_pool(rng, 5, h, d, g)
    pages = np.array([[3, -1, 2, 2 ** 31 - 1, 4, 5], [-7, 9, 100, -2 ** 31, 7, 7]], dtype=np.int32)
    lens = [350, 384]
    for c in (1, 20):
        q = rng.normal(0, 1, (2 * c, 2 * h, d)).astype(np.float16)
        out = kv4.attention(dev(q), dev(pool), dev(pages), dev(np.array(lens, np.int32)), 0.2).cpu().numpy()
        for head in range(h):
            full = ko.Rows(pool, [3, 0, 2, 0, 4, 0], 350, head, d, g)
            for i in range(c):
                seen = np.array([r for r in range(350 - c + i + 1) if r // 64 in (0, 2, 4)])
                for j in range(2 * head, 2 * head + 2):
                    want, tol = ko.attend(full, q[i, j].astype(np.float64), 0.2, seen)
                    assert np.all(np.abs(out[i, j] - want) <= tol)
        assert np.all(out[c:] == 0)


def test_lengths_beyond_the_table_are_clamped(kv4):
    d, g, h = 64, 32, 1
    rng = np.random.default_rng(13)
    pool = random_pool(rng, 3, h, d, g)
    pages = np.array([[2, 0]], dtype=np.int32)
    q = rng.normal(0, 1, (1, 2, d)).astype(np.float16)
    a, b = (kv4.attention(dev(q), dev(pool), dev(pages), dev(np.array([n], np.int32)), 0.2) for n in (128, 2 ** 31 - 1))
    assert torch.equal(a, b)


def test_a_table_row_may_lie_in_a_wider_one(kv4):
    d, g, h = 128, 64, 1
    rng = np.random.default_rng(14)
    lens = [200, 130, 64]
    pages, total = tables(rng, lens, width=9)
    pool, q = dev(random_pool(rng, total, h, d, g)), dev(rng.normal(0, 1, (3, 1, d)).astype(np.float16))
    n = dev(np.array(lens, np.int32))
    wide = dev(pages)
    assert torch.equal(kv4.attention(q, pool, wide[:, :4], n, 0.1), kv4.attention(q, pool, wide[:, :4].contiguous(), n, 0.1))
    assert torch.equal(kv4.attention(q[:1], pool, wide[2:, :1], n[2:], 0.1), kv4.attention(q[2:], pool, wide[2:], n[2:], 0.1)) is False


def test_pool_beyond_32_bits(kv4):
    # records whose offsets pass 2^32 bytes
    d, g, h = 128, 64, 32
    per = h * ko.record_bytes(d, g)
    n = 2 ** 32 // per + 40
    pool = torch.empty((n, h, ko.record_bytes(d, g)), dtype=torch.uint8, device=DEV)
    rng = np.random.default_rng(15)
    places = [n - 1, 3, n - 20]
    pages = dev(np.array([places], dtype=np.int32))
    small = kv4.new_pool(3, h, d, g, device=DEV)
    k, v = (dev(rng.normal(0, 1, (150, h, d)).astype(np.float16)) for _ in range(2))
    lens, there = dev(np.array([150], np.int32)), dev(np.arange(3, dtype=np.int32)[None])
    kv4.append(k, v, pool, pages, lens)
    kv4.append(k, v, small, there, lens)
    q = dev(rng.normal(0, 1, (1, h, d)).astype(np.float16))
    want = kv4.attention(q, small, there, lens, 0.1)
    assert torch.equal(kv4.attention(q, pool, pages, lens, 0.1), want)
    assert torch.equal(kv4.select_pages(q, pool, pages, lens, 2), kv4.select_pages(q, small, there, lens, 2))
    kv4.copy_pages(pool, dev(np.array(places, np.int32)), dev(np.array([7, n - 2, 8], np.int32)))
    assert torch.equal(kv4.attention(q, pool, dev(np.array([[7, n - 2, 8]], np.int32)), lens, 0.1), want)


def test_a_refused_call_appends_nothing(kv4):
    pool = kv4.new_pool(2, 2, 64, 32, device=DEV).zero_()
    q, pages, lens = torch.ones((1, 4, 64), dtype=torch.float16, device=DEV), torch.zeros((1, 2), dtype=torch.int32, device=DEV), \
        torch.ones(1, dtype=torch.int32, device=DEV)
    room = torch.zeros(300, dtype=torch.float16, device=DEV)
    for out in (q.float(), q[:, :2], room[4:260].view(1, 4, 64), q.cpu()):
        with pytest.raises(ValueError):
            kv4.attention(q, pool, pages, lens, 1.0, out=out, k_new=q[:, :2], v_new=q[:, :2])
    assert not torch.any(pool)
    kv4.attention(q, pool, pages, lens, 1.0, out=room[8:264].view(1, 4, 64), k_new=q[:, :2], v_new=q[:, :2])
    assert torch.any(pool) and torch.all(room[8:264] == 1) and not torch.any(room[:8]) and not torch.any(room[264:])


def test_strided_queries_and_other_streams(kv4):
    d, g, h, share = 64, 32, 2, 3
    rng = np.random.default_rng(16)
    lens = [300, 90]
    pages, total = tables(rng, lens)
    pool, n, pages = dev(random_pool(rng, total, h, d, g)), dev(np.array(lens, np.int32)), dev(pages)
    big = dev(rng.normal(0, 1, (2, 3, h * share, d + 8)).astype(np.float16))
    want = kv4.attention(big[:, 1, :, :d].contiguous(), pool, pages, n, 0.1)
    assert torch.equal(kv4.attention(big[:, 1, :, :d], pool, pages, n, 0.1), want)
    odd = big[:, 1, :, 3:d + 3]
    assert torch.equal(kv4.attention(odd, pool, pages, n, 0.1), kv4.attention(odd.contiguous(), pool, pages, n, 0.1))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = kv4.attention(big[:, 1, :, :d], pool, pages, n, 0.1)
    b = kv4.attention(big[:, 1, :, :d], pool, pages, n, 0.1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, want) and torch.equal(b, want)


def test_nothing_to_do(kv4):
    pool = kv4.new_pool(2, 2, 64, 32, device=DEV)
    none, pages, lens = (torch.empty((0, 2, 64), dtype=torch.float16, device=DEV), torch.zeros((0, 3), dtype=torch.int32, device=DEV),
                         torch.zeros(0, dtype=torch.int32, device=DEV))
    assert kv4.attention(none, pool, pages, lens, 1.0).shape == (0, 2, 64)
    assert kv4.append(none, none, pool, pages, lens) is None
    assert kv4.select_pages(none, pool, pages, lens, 2).shape == (0, 2, 2)
    two = torch.zeros((2, 3), dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV)
    assert kv4.attention(none, pool, *two, 1.0, torch.zeros(3, dtype=torch.int32, device=DEV)).shape == (0, 2, 64)
    # a table without columns: no rows
    q = torch.ones((2, 2, 64), dtype=torch.float16, device=DEV)
    assert torch.all(kv4.attention(q, pool, two[0][:, :0], two[1], 1.0) == 0)
    kv4.append(q, q, pool, two[0][:, :0], two[1])
    assert torch.all(kv4.select_pages(q, pool, two[0][:, :0], two[1], 2) == -1)


def test_refusals(kv4):
    pool = kv4.new_pool(4, 2, 64, 32, device=DEV)
    q = torch.zeros((2, 4, 64), dtype=torch.float16, device=DEV)
    kv = q[:, :2]
    pages, lens = torch.zeros((2, 3), dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV)
    sel = torch.zeros((2, 2, 2), dtype=torch.int32, device=DEV)
    st = torch.zeros(3, dtype=torch.int32, device=DEV)
    bad = [
        lambda: kv4.attention(q.float(), pool, pages, lens, 1.0),
        lambda: kv4.attention(q[0], pool, pages, lens, 1.0),
        lambda: kv4.attention(q, pool[:, :, :-16], pages, lens, 1.0),
        lambda: kv4.attention(q[:, :3], pool, pages, lens, 1.0),
        lambda: kv4.attention(q, pool, pages.long(), lens, 1.0),
        lambda: kv4.attention(q, pool, pages, lens[:1], 1.0),
        lambda: kv4.attention(q, pool, pages.cpu(), lens, 1.0),
        lambda: kv4.attention(q, pool, pages, lens, 1.0, st[:2]),
        lambda: kv4.attention(q, pool, pages, lens, 1.0, st, sel),
        lambda: kv4.attention(q, pool, pages, lens, 1.0, selected=sel.long()),
        lambda: kv4.attention(q, pool, pages, lens, 1.0, selected=sel[:1]),
        lambda: kv4.attention(q, pool, pages, lens, 1.0, out=q.float()),
        lambda: kv4.attention(torch.cat([q, q[:1]]), pool, pages, lens, 1.0),
        lambda: kv4.attention(q, pool, pages, lens, 1.0, k_new=kv),
        lambda: kv4.attention(q, pool, pages, lens, 1.0, k_new=q, v_new=q),
        lambda: kv4.attention(q, pool, pages, lens, 1.0, k_new=kv, v_new=kv.float()),
        lambda: kv4.attention(q, pool, pages, lens, 1.0, selected=sel, k_new=kv, v_new=kv),
        lambda: kv4.append(q, q, pool, pages, lens),
        lambda: kv4.append(kv, kv[:1], pool, pages, lens),
        lambda: kv4.append(kv, kv.float(), pool, pages, lens),
        lambda: kv4.select_pages(torch.cat([q, q]), pool, pages, lens, 2),
        lambda: kv4.select_pages(q, pool, pages, lens, 1),
        lambda: kv4.select_pages(q, pool, pages, lens, 0, 0, 0),
        lambda: kv4.copy_pages(pool, lens, st),
        lambda: kv4.copy_pages(pool, lens.long(), lens.long()),
        lambda: kv4.copy_pages(pool[:, :1], lens, lens),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            call()
            pytest.fail("call %d was taken" % i)


# ------------------------------------------------------------------------------------------- selection of pages

@pytest.mark.parametrize("d,g", [(64, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("h,share,lens,count,first,last", [
    (1, 1, [640], 3, 1, 1), (2, 4, [64 * 70, 63, 64 * 16 + 1], 16, 1, 1), (3, 9, [5000, 70], 5, 0, 0), (1, 8, [64 * 1030], 40, 2, 3),
    (2, 1, [100, 1, 0], 2, 1, 1), (1, 2, [64 * 3000 + 5], 64, 1, 1), (1, 1, [3000], 1, 0, 1),
], ids=["ten", "several", "nine-queries", "thousand", "short", "three-thousand", "one"])
def test_select(kv4, d, g, h, share, lens, count, first, last):
    rng = np.random.default_rng(d + count)
    pages, total = tables(rng, lens)
    pool = random_pool(rng, total, h, d, g)
    q = rng.normal(0, 1, (len(lens), h * share, d)).astype(np.float16)
    got = kv4.select_pages(dev(q), dev(pool), dev(pages), dev(np.array(lens, np.int32)), count, first, last).cpu().numpy()
    assert got.shape == (len(lens), h, count)
    for b, n in enumerate(lens):
        bounds = ko.read(pool[pages[b, :(n + 63) // 64]], d, g)["bounds"]
        for head in range(h):
            want = ko.select(bounds[:, head], q[b, head * share:(head + 1) * share], count, first, last)
            assert got[b, head].tolist() == want + [-1] * (count - len(want))


def test_select_from_the_widest_table(kv4):
    d, g, h, share, width = 64, 32, 1, 2, 16384
    rng = np.random.default_rng(35)
    pool = random_pool(rng, 997, h, d, g)
    pages = rng.integers(0, 997, (2, width)).astype(np.int32)  # equal scores by the dozen
    lens = [64 * width, 64 * 9000 + 1]
    q = rng.normal(0, 1, (2, h * share, d)).astype(np.float16)
    got = kv4.select_pages(dev(q), dev(pool), dev(pages), dev(np.array(lens, np.int32)), 100).cpu().numpy()
    bounds = ko.read(pool, d, g)["bounds"][:, 0]
    for b, n in enumerate(lens):
        assert got[b, 0].tolist() == ko.select(bounds[pages[b, :(n + 63) // 64]], q[b], 100, 1, 1)
    with pytest.raises((ValueError, RuntimeError)):
        kv4.select_pages(dev(q), dev(pool), dev(np.zeros((2, width + 1), np.int32)), dev(np.array(lens, np.int32)), 100)


def test_select_between_equals_and_without_numbers(kv4):
    d, g = 64, 64
    rng = np.random.default_rng(20)
    pool = random_pool(rng, 40, 1, d, g)
    pool[:, 0, -4 * d:] = pool[0, 0, -4 * d:]  # all alike
    better = [7, 21, 22]
    for p in better:
        pool[p, 0, -4 * d:-2 * d].view(np.float16)[:] += np.float16(1)
    pool[30, 0, -4 * d:].view(np.float16)[:] = np.nan
    pages = np.arange(40, dtype=np.int32)[None]
    pages[0, 9] = -1  # no page: the lowest as well
    q = np.ones((1, 2, d), dtype=np.float16)
    n = dev(np.array([40 * 64], np.int32))
    pick = lambda count, first=0, last=0: kv4.select_pages(dev(q), dev(pool), dev(pages), n, count, first, last)[0, 0].tolist()
    assert pick(3) == better and pick(5) == [0, 1, 7, 21, 22] and pick(2) == [7, 21]
    assert pick(4, 1, 1) == [0, 7, 21, 39] and pick(38) == [i for i in range(40) if i not in (9, 30)]
    assert pick(39) == [i for i in range(40) if i != 30] and pick(6, 0, 4) == [7, 21, 36, 37, 38, 39]


@pytest.mark.parametrize("d,g,h,share,lens,count", [(128, 64, 2, 4, [64 * 40 + 3, 64 * 5, 17], 8), (64, 32, 1, 1, [64 * 200], 33),
                                                     (128, 32, 1, 16, [64 * 9 + 1], 300), (64, 64, 1, 40, [64 * 60, 70], 20)])
def test_attention_over_selected_pages(kv4, d, g, h, share, lens, count):
    rng = np.random.default_rng(count)
    pages, total = tables(rng, lens)
    pool = random_pool(rng, total, h, d, g)
    q = rng.normal(0, 1, (len(lens), h * share, d)).astype(np.float16)
    dq, dpool, dpages, n = dev(q), dev(pool), dev(pages), dev(np.array(lens, np.int32))
    sel = kv4.select_pages(dq, dpool, dpages, n, count)
    out = kv4.attention(dq, dpool, dpages, n, d ** -0.5, selected=sel).cpu().numpy().astype(np.float64)
    sel = sel.cpu().numpy()
    for b, length in enumerate(lens):
        for head in range(h):
            rows = ko.Rows(pool, pages[b, :(length + 63) // 64], length, head, d, g)
            seen = np.concatenate([np.arange(64 * p, min(64 * p + 64, length)) for p in sel[b, head] if p >= 0])
            for j in range(head * share, (head + 1) * share):
                want, tol = ko.attend(rows, q[b, j].astype(np.float64), d ** -0.5, seen)
                assert np.all(np.abs(out[b, j] - want) <= tol)


def test_selected_pages_of_a_callers_own(kv4):
    # any order, one twice, one outside the sequence, none at all
    d, g, h = 128, 64, 1
    rng = np.random.default_rng(22)
    lens = [64 * 6 + 10, 64 * 6 + 10, 64 * 6]
    pages, total = tables(rng, lens)
    pool = random_pool(rng, total, h, d, g)
    sel = np.array([[[6, 2, 2, -1]], [[7, 1000, -5, 2 ** 31 - 1]], [[5, 0, 5, 5]]], dtype=np.int32)
    q = rng.normal(0, 1, (3, 2, d)).astype(np.float16)
    out = kv4.attention(dev(q), dev(pool), dev(pages), dev(np.array(lens, np.int32)), 0.1, selected=dev(sel)).cpu().numpy()
    assert np.all(out[1] == 0)
    for b in (0, 2):
        rows = ko.Rows(pool, pages[b, :(lens[b] + 63) // 64], lens[b], 0, d, g)
        seen = np.concatenate([np.arange(64 * p, min(64 * p + 64, lens[b])) for p in sel[b, 0] if p >= 0])
        for j in range(2):
            want, tol = ko.attend(rows, q[b, j].astype(np.float64), 0.1, seen)
            assert np.all(np.abs(out[b, j] - want) <= tol)


# ---------------------------------------------------------------------------------------------------------- pages

def test_copy_pages(kv4):
    rng = np.random.default_rng(23)
    for shape, src, dst in (((3, 12, 2, ko.record_bytes(64, 32)), [1, 5, 11, 3], [0, 2, 4, 3]),
                            ((6, 8, ko.record_bytes(128, 64)), [0, -1, 2, 7], [1, 3, 6, 4]),
                            ((1, 2, 1, ko.record_bytes(64, 64)), [1], [0])):
        pool = rng.integers(0, 256, shape, dtype=np.uint8)
        d = dev(pool)
        kv4.copy_pages(d, dev(np.array(src, np.int32)), dev(np.array(dst, np.int32)))
        want = pool.copy()
        axis = want if len(shape) == 4 else want[None]
        n = axis.shape[1]
        for a, b in zip(src, dst):
            if 0 <= a < n and 0 <= b < n:
                axis[:, b] = (pool if len(shape) == 4 else pool[None])[:, a]
        assert np.array_equal(d.cpu().numpy(), want)


class Mirror:
    """The rows a cache should hold, kept on the host per sequence."""

    def __init__(self, layers, h, d):
        self.layers, self.h, self.d, self.rows = layers, h, d, {}

    def check(self, cache, rng, g, scale=0.1):
        for layer in range(self.layers):
            seqs = [s for s in self.rows if self.rows[s][0].shape[1]]
            q = rng.normal(0, 1, (len(seqs), 2 * self.h, self.d)).astype(np.float16)
            out = cache.attention(layer, dev(q), scale, seqs).cpu().numpy().astype(np.float64)
            for i, s in enumerate(seqs):
                k, v = (x[layer] for x in self.rows[s])
                f = {}
                for name, x in (("k", k), ("v", v)):
                    c, sc, m = ko.quantise(x, g)
                    f[name] = (c, sc.astype(np.float64), m.astype(np.float64))
                for head in range(self.h):
                    r = ko.Rows.__new__(ko.Rows)
                    kc, ks, km = (x[:, head] for x in f["k"])
                    vc, vs, vm = (x[:, head] for x in f["v"])
                    r.k, r.v, r.k_abs = ks * kc + km, vs * vc + vm, ks * kc + np.abs(km)
                    r.v_mid, r.v_rest = np.abs(vs * (vc - 8)), np.abs(8 * vs + vm)
                    for j in range(2 * head, 2 * head + 2):
                        want, tol = ko.attend(r, q[i, j].astype(np.float64), scale, np.arange(len(r.k)))
                        assert np.all(np.abs(out[i, j] - want) <= tol), (layer, s, j)


def test_a_cache_that_grows_forks_and_is_made_compact(kv4):
    layers, h, d, g = 2, 2, 64, 32
    rng = np.random.default_rng(24)
    cache = kv4.KV4Cache(layers, 24, h, d, g, max_seqs=6, max_rows=64 * 8, device=DEV)
    cache.pool.random_()
    mirror = Mirror(layers, h, d)

    def grow(seqs, counts):
        cache.extend(seqs, counts)
        k, v = (rng.normal(0, 1, (layers, sum(counts), h, d)).astype(np.float16) for _ in range(2))
        for layer in range(layers):
            cache.append(layer, dev(k[layer]), dev(v[layer]), seqs, dev(starts_of(counts)))
        at = 0
        for s, c in zip(seqs, counts):
            old = mirror.rows.get(s, (np.zeros((layers, 0, h, d), np.float16),) * 2)
            mirror.rows[s] = tuple(np.concatenate([o, x[:, at:at + c]], 1) for o, x in zip(old, (k, v)))
            at += c
        assert cache.lengths[seqs].tolist() == [mirror.rows[s][0].shape[1] for s in seqs]

    def fork(s):
        new = cache.fork(s)
        mirror.rows[new] = mirror.rows[s]
        return new

    a, b = cache.add(), cache.add()
    grow([a, b], [100, 64])
    mirror.check(cache, rng, g)
    c = fork(a)                       # shares a part-filled page
    e = fork(b)                       # shares a full one
    assert cache.free_pages() == 24 - 3
    grow([a, c, e], [5, 70, 1])       # a or c writes to a copy; the other keeps the page
    assert len(set(cache.pages(a)) & set(cache.pages(c))) == 1 and cache.pages(e)[0] == cache.pages(b)[0]
    mirror.check(cache, rng, g)
    f = fork(c)
    cache.truncate(f, 130)            # f ends inside a page that it shares with c
    mirror.rows[f] = tuple(x[:, :130] for x in mirror.rows[f])
    grow([f], [3])
    mirror.check(cache, rng, g)
    cache.free(a)
    cache.free(b)
    del mirror.rows[a], mirror.rows[b]
    used = cache.compact()
    assert used == 24 - cache.free_pages() and all(p < used for s in mirror.rows for p in cache.pages(s))
    mirror.check(cache, rng, g)
    again = cache.add()
    mirror.rows[again] = (np.zeros((layers, 0, h, d), np.float16),) * 2
    grow([again, e], [300, 63])
    mirror.check(cache, rng, g)
    assert cache.compact() == 24 - cache.free_pages()
    for s in list(mirror.rows):
        cache.free(s)
    assert cache.free_pages() == 24 and cache.compact() == 0


def test_a_captured_step_follows_lengths_and_tables(kv4):
    # append, selection, attention (dense and over the selection) in one graph, replayed while the cache grows over page
    # borders and its table changes; every replay against the eager calls on a copy
    d, g, h, share, b = 128, 64, 2, 4, 3
    rng = np.random.default_rng(25)
    lens = np.array([60, 700, 127], np.int32)
    pages, total = tables(rng, lens + 20, spare=4)
    pool = dev(random_pool(rng, total, h, d, g))
    n, table = dev(lens), dev(pages)
    kv, q = torch.empty((2, b, h, d), dtype=torch.float16, device=DEV), torch.empty((b, h * share, d), dtype=torch.float16, device=DEV)

    def step(pool, n, table):
        n += 1
        kv4.append(kv[0], kv[1], pool, table, n)
        sel = kv4.select_pages(q, pool, table, n, 4)
        return kv4.attention(q, pool, table, n, 0.1), kv4.attention(q, pool, table, n, 0.1, selected=sel), sel

    kv.normal_(), q.normal_()
    eager = pool.clone(), n.clone(), table.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(pool.clone(), n.clone(), table)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(pool, n, table)
    for i in range(8):
        kv.normal_(), q.normal_()
        if i == 4:  # the first sequence's first page moves elsewhere
            free = next(p for p in range(total) if p not in pages)
            for x, t in ((pool, table), eager[::2]):
                kv4.copy_pages(x, t[0, :1].clone(), torch.tensor([free], dtype=torch.int32, device=DEV))
                t[0, 0] = free
        graph.replay()
        torch.cuda.synchronize()
        want = step(*eager)
        for x, y in zip(got, want):
            assert torch.equal(x, y), i
        assert torch.equal(pool, eager[0]) and torch.equal(n, eager[1])


@pytest.mark.parametrize("each,share,d,g", [(40, 4, 128, 64), (3, 4, 64, 32)], ids=["chunk", "drafts"])
def test_captured_chunks_follow_lengths(kv4, each, share, d, g):
    # tokens appended and attended to in one graph: shares and joins follow the lengths that a replay finds
    h, b = 2, 2
    rng = np.random.default_rng(36)
    lens = np.array([each, 1500], np.int32)
    pages, total = tables(rng, lens + 8 * 640, spare=0)
    pool, n, table = dev(random_pool(rng, total, h, d, g)), dev(lens), dev(pages)
    kv = torch.empty((2, b * each, h, d), dtype=torch.float16, device=DEV)
    q = torch.empty((b * each, h * share, d), dtype=torch.float16, device=DEV)
    call = lambda pool: kv4.attention(q, pool, table, n, 0.1, k_new=kv[0], v_new=kv[1])
    kv.normal_(), q.normal_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(pool.clone())
    torch.cuda.current_stream().wait_stream(side)
    eager = pool.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(pool)
    for more in (0, each, 640, each, 3000):
        n += more
        kv.normal_(), q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, call(eager)) and torch.equal(pool, eager), more


@pytest.mark.parametrize("tokens,share", [(1, 4), (1, 12), (30, 8)], ids=["packed", "rows", "chunk"])
def test_attention_without_a_workspace(kv4, tokens, share):
    # nothing is shared then: one workgroup goes through all of a tile's pages
    from sqamd import capi
    d, g, h = 128, 64, 1
    rng = np.random.default_rng(37)
    lens = [4000, 70]
    pages, total = tables(rng, lens)
    pool = random_pool(rng, total, h, d, g)
    q = rng.normal(0, 1, (2 * tokens, share, d)).astype(np.float16)
    dq, dpool, dpages, n = dev(q), dev(pool), dev(pages), dev(np.array(lens, np.int32))
    out, p = torch.empty_like(dq), capi._ptr
    assert capi.lib().sq_kv4_attention(p(dq), p(out), p(dpool), p(dpages), p(n), None, None, 2 * tokens, 2, h * share, h, d, g, total,
                                       pages.shape[1], pages.shape[1], 0, share * d, d, d ** -0.5, None, None, None, None, 0,
                                       capi._stream()) == 0
    compare(out.cpu().numpy().astype(np.float64), q, pool, pages, lens, [tokens] * 2, d, g, h, share, d ** -0.5)


def test_two_graphs_at_once(kv4):
    # each captured call has a workspace of its own: graphs on two streams do not disturb each other
    d, g, h, share = 128, 64, 8, 4
    rng = np.random.default_rng(26)
    lens = np.array([20000], np.int32)
    pages, total = tables(rng, lens)
    pool, n, table = dev(random_pool(rng, total, h, d, g)), dev(lens), dev(pages)
    qs = [dev(rng.normal(0, 1, (1, h * share, d)).astype(np.float16)) for _ in range(2)]
    want = [kv4.attention(q, pool, table, n, 0.1) for q in qs]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(kv4.attention(q, pool, table, n, 0.1))
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(3):
                    graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


@pytest.mark.parametrize("d,g", SIZES)
@pytest.mark.parametrize("h,share,lens,new", [
    (2, 4, [1, 64, 65, 640], None), (4, 1, [33, 32, 700, 128], None), (1, 7, [97, 3000], None), (2, 16, [129, 1025], None),
    (1, 24, [200, 64], None), (1, 40, [300], None), (8, 4, [5000], None), (2, 2, [30, 200], [30, 70]), (1, 3, [0, 70, 129], None),
], ids=["edges", "unshared", "seven", "sixteen", "two-tiles", "many-rows", "split", "chunks", "none"])
def test_rows_appended_by_the_attention_itself(kv4, d, g, h, share, lens, new):
    # the cache and the result are those of an append followed by the attention, bit for bit
    rng = np.random.default_rng(d + g + share)
    new = new or [1] * len(lens)
    pages, total = tables(rng, lens)
    pool = dev(random_pool(rng, total, h, d, g))
    t = sum(new)
    kv = dev(rng.normal(0, 1, (t, 2, h, d)).astype(np.float16))
    q = dev(rng.normal(0, 1, (t, h * share, d)).astype(np.float16))
    n, table = dev(np.array(lens, np.int32)), dev(pages)
    st = None if max(new) == 1 else dev(starts_of(new))
    other = pool.clone()
    kv4.append(kv[:, 0], kv[:, 1], pool, table, n, st)
    want = kv4.attention(q, pool, table, n, 0.1, st)
    for _ in range(2):  # (once more: the same rows in the same places)
        got = kv4.attention(q, other, table, n, 0.1, st, k_new=kv[:, 0], v_new=kv[:, 1])
        assert torch.equal(got, want) and torch.equal(other, pool)
    odd = kv.clone().flatten()
    shifted = torch.cat([odd.new_zeros(3), odd])[3:].view(kv.shape)  # rows that have to be copied first
    assert torch.equal(kv4.attention(q, other, table, n, 0.1, st, k_new=shifted[:, 0], v_new=shifted[:, 1]), want)


def test_a_new_row_without_a_page(kv4):
    d, g, h = 64, 32, 1
    rng = np.random.default_rng(30)
    pool = random_pool(rng, 3, h, d, g)
    pages = np.array([[0, 9], [1, -1], [2, 2]], dtype=np.int32)
    lens = np.array([100, 65, 129], np.int32)  # a page outside the pool, none, a row beyond the table
    q, kv = rng.normal(0, 1, (3, 2, d)).astype(np.float16), rng.normal(0, 1, (2, 3, h, d)).astype(np.float16)
    a, b = dev(pool), dev(pool)
    got = kv4.attention(dev(q), a, dev(pages), dev(lens), 0.1, k_new=dev(kv[0]), v_new=dev(kv[1]))
    kv4.append(dev(kv[0]), dev(kv[1]), b, dev(pages), dev(lens))
    assert torch.equal(a, b) and torch.equal(got, kv4.attention(dev(q), b, dev(pages), dev(lens), 0.1))


def test_results_repeat_bit_for_bit(kv4):
    rng = np.random.default_rng(27)
    lens = [9000, 300, 64]
    pages, total = tables(rng, lens)
    pool, n, table = dev(random_pool(rng, total, 2, 128, 64)), dev(np.array(lens, np.int32)), dev(pages)
    q = dev(rng.normal(0, 1, (3, 8, 128)).astype(np.float16))
    first = kv4.attention(q, pool, table, n, 0.1)
    assert all(torch.equal(kv4.attention(q, pool, table, n, 0.1), first) for _ in range(5))


@pytest.mark.parametrize("c,h,share,equal", [(4, 2, 1, True), (4, 1, 6, True), (33, 1, 4, True), (40, 2, 4, False), (5, 2, 2, False)],
                         ids=["packed", "two-tiles", "chunk", "ragged-chunk", "ragged"])
def test_tokens_beyond_the_table_leave_the_others_where_they_are(kv4, c, h, share, equal):
    # rows that the table has no place for are not stored and not seen; the call's other tokens are the rows that append
    # stored, and see what lies up to their own
    d, g = 128, 64
    rng = np.random.default_rng(c + share)
    lens, new = [130, 128 + c, 200, 128 + c // 2, 101], [c, c, c, c, c if equal else 2]
    pages, total = np.arange(10, dtype=np.int32).reshape(5, 2), 11
    pool = random_pool(rng, total, h, d, g)
    q = rng.normal(0, 1, (sum(new), h * share, d)).astype(np.float16)
    kv = rng.normal(0, 1, (2, sum(new), h, d)).astype(np.float16)
    st = None if equal else dev(starts_of(new))
    dpool, args = dev(pool), (dev(pages), dev(np.array(lens, np.int32)))
    kv4.append(dev(kv[0]), dev(kv[1]), dpool, *args, st)
    want, written = expect_append(pool, kv[0], kv[1], pages, lens, new, d, g)
    stored = dpool.cpu().numpy()
    assert np.array_equal(ko.read(stored, d, g)["kc"], want["kc"]) and written.any()
    out = kv4.attention(dev(q), dpool, *args, 0.1, st).cpu().numpy().astype(np.float64)
    both = dev(pool)
    assert torch.equal(kv4.attention(dev(q), both, *args, 0.1, st, k_new=dev(kv[0]), v_new=dev(kv[1])).double().cpu(),
                       torch.from_numpy(out)) and torch.equal(both, dpool)
    at = 0
    for b, (n, count) in enumerate(zip(lens, new)):
        for head in range(h):
            rows = ko.Rows(stored, pages[b], 128, head, d, g)
            for i in range(count):
                for j in range(head * share, (head + 1) * share):
                    expect, tol = ko.attend(rows, q[at + i, j].astype(np.float64), 0.1, np.arange(min(128, n, n - count + i + 1)))
                    assert not np.sum(np.abs(out[at + i, j] - expect) > tol), (b, i, j)
        at += count


def test_sequences_that_overlap_far_beyond_the_tokens(kv4):
    # starts that go back and forth: thousands of sequences on the same tokens, more pages in all than 39 bits count.  Which
    # of them a token's result comes from is open, but one that has its tokens alone gets its own
    d, g, h, share, t, alone, b, width = 64, 32, 8, 4, 1 << 15, 4096, 4096, 1 << 16
    rng = np.random.default_rng(40)
    starts = np.where(np.arange(b + 1) % 2 == 0, t, alone).astype(np.int32)
    starts[0] = 0
    lens = np.where(np.arange(b) < 13, 0, 64 * width).astype(np.int32)
    lens[0] = 1280
    pool = random_pool(rng, 20, h, d, g)
    pages = torch.full((b, width), -1, dtype=torch.int32, device=DEV)
    pages[0, :20] = torch.arange(20, dtype=torch.int32, device=DEV)
    q = dev(rng.normal(0, 1, (t, h * share, d)).astype(np.float16))
    out = torch.full_like(q, 9.0)
    kv4.attention(q, dev(pool), pages, dev(lens), 0.1, dev(starts), out=out)
    own = out[:alone].cpu().numpy().astype(np.float64)
    compare(own, q[:alone].cpu().numpy(), pool, pages[:1, :20].cpu().numpy(), [1280], [alone], d, g, h, share, 0.1)
    assert not torch.any(out[alone:])


@pytest.mark.parametrize("d,g,c,share", [(64, 32, 1, 4), (128, 64, 1, 12), (128, 128, 1, 24), (64, 64, 5, 4), (128, 64, 40, 4), (64, 32, 70, 2)],
                         ids=["packed", "rows", "two-tiles", "drafts", "chunk", "chunk-64"])
@pytest.mark.parametrize("where", ["first", "middle", "hidden"])
def test_one_row_of_large_values_that_hardly_counts(kv4, d, g, c, share, where):
    # values of 60000 in one row of no weight (or that most of the call's tokens do not see) beside rows of 0.01: the small ones
    # are as exact as they are without it.  Scores come from two elements of a query, so that their own rounding is small
    rng = np.random.default_rng(41)
    n = 1000 if where != "hidden" else 64 if c < 64 else 128  # (hidden in a page that the tokens see most of)
    at = {"first": 3, "middle": 500, "hidden": n - 1}[where]
    k, v = rng.normal(0, 1, (n, 1, d)), rng.normal(0, 0.01, (n, 1, d))
    v[at] = 60000 * np.where(np.arange(d) % 2, 1, -1)
    if where != "hidden":
        k[at] = 0
        k[at, 0, 0] = -14
    q = np.zeros((c, share, d))
    q[..., 0], q[..., d // 2] = rng.uniform(2.5, 3.5, (c, share)), rng.uniform(-0.5, 0.5, (c, share))
    k, v, q = (x.astype(np.float16) for x in (k, v, q))
    pool, pages, lens = kv4.new_pool(16, 1, d, g, device=DEV), np.arange(16, dtype=np.int32)[None], dev(np.array([n], np.int32))
    pool.zero_()
    kv4.append(dev(k), dev(v), pool, dev(pages), lens)
    out = kv4.attention(dev(q), pool, dev(pages), lens, 1.0).cpu().numpy().astype(np.float64)
    rows = ko.Rows(pool.cpu().numpy(), pages[0], n, 0, d, g)
    worst = 0.0
    for i in sorted({0, 1, 2, 30, c - 2, c - 1} & set(range(c))):
        seen = np.arange(n - c + i + 1)
        if where == "hidden" and at in seen:
            continue
        for j in range(share):
            want, tol = ko.attend(rows, q[i, j].astype(np.float64), 1.0, seen, 2.0 ** -11 if c * share > 32 else 0.0)
            worst = max(worst, float(np.max(np.abs(out[i, j] - want) / tol)))
    assert worst <= 1, worst


def test_one_sequence_of_a_wider_table(kv4):
    # views of one row: the row's distance is not read from the table then, the columns may be cut
    d, g, h, share = 128, 64, 2, 2
    rng = np.random.default_rng(42)
    lens = [200, 130, 64]
    pages, total = tables(rng, lens, width=9)
    pool, q = random_pool(rng, total, h, d, g), dev(rng.normal(0, 1, (3, h * share, d)).astype(np.float16))
    kv = dev(rng.normal(0, 1, (2, 3, h, d)).astype(np.float16))
    n, wide = dev(np.array(lens, np.int32)), dev(pages)
    for i, cut in ((2, 1), (2, 9), (1, 3), (1, 4), (0, 4)):
        a, b = dev(pool), dev(pool)
        views = (wide[i:i + 1, :cut], n[i:i + 1])
        copies = (dev(pages[i:i + 1, :(lens[i] + 63) // 64]), dev(np.array(lens[i:i + 1], np.int32)))
        assert views[0].stride(0) == 9
        assert torch.equal(kv4.attention(q[i:i + 1], a, *views, 0.1), kv4.attention(q[i:i + 1], b, *copies, 0.1))
        assert torch.equal(kv4.select_pages(q[i:i + 1], a, *views, 2), kv4.select_pages(q[i:i + 1], b, *copies, 2))
        kv4.append(kv[0, i:i + 1], kv[1, i:i + 1], a, *views)
        kv4.append(kv[0, i:i + 1], kv[1, i:i + 1], b, *copies)
        assert torch.equal(a, b) and not torch.equal(a, dev(pool))
    every = kv4.attention(q, dev(pool), wide, n, 0.1)
    for i in range(3):
        assert torch.equal(kv4.attention(q[i:i + 1], dev(pool), wide[i:i + 1], n[i:i + 1], 0.1), every[i:i + 1])


@pytest.mark.parametrize("d,g,h,share,lens,new", [
    (128, 64, 2, 4, [2300, 1, 1700, 640, 3000, 5], [2000, 1, 1500, 1, 1, 0]),
    (64, 32, 1, 1, [4000, 33, 700], [4000, 5, 1]),
    (128, 128, 1, 16, [900, 400], [900, 1]),
], ids=["four", "one", "sixteen"])
def test_long_prompts_beside_single_tokens(kv4, d, g, h, share, lens, new):
    rng = np.random.default_rng(43)
    assert sum(new) * share > 1024 * len(new)
    pages, total = tables(rng, lens)
    pool = random_pool(rng, total, h, d, g)
    t = sum(new)
    q = rng.normal(0, 1, (t + 2, h * share, d)).astype(np.float16)
    out = torch.full(q.shape, 9.0, dtype=torch.float16, device=DEV)
    kv4.attention(dev(q), dev(pool), dev(pages), dev(np.array(lens, np.int32)), d ** -0.5, dev(starts_of(new)), out=out)
    out = out.cpu().numpy().astype(np.float64)
    assert np.all(out[t:] == 9.0)
    compare(out, q, pool, pages, lens, new, d, g, h, share, d ** -0.5, few=16)


def test_a_row_appended_behind_many_pages(kv4):
    # more pages in one workgroup than are looked up at once, and the row's page among the last of them
    d, g, h, b = 64, 32, 8, 130
    rng = np.random.default_rng(44)
    lens = (64 * 65 + rng.integers(1, 65, b)).tolist()
    pages = np.concatenate([np.broadcast_to(rng.permutation(65), (b, 65)), 65 + rng.permutation(b)[:, None]], 1).astype(np.int32)
    pool = dev(random_pool(rng, 65 + b, h, d, g))
    kv, q = (dev(rng.normal(0, 1, s).astype(np.float16)) for s in ((2, b, h, d), (b, h, d)))
    n, table, other = dev(np.array(lens, np.int32)), dev(pages), pool.clone()
    kv4.append(kv[0], kv[1], pool, table, n)
    want = kv4.attention(q, pool, table, n, 0.1)
    assert torch.equal(kv4.attention(q, other, table, n, 0.1, k_new=kv[0], v_new=kv[1]), want) and torch.equal(other, pool)
    compare(want[:3].cpu().numpy().astype(np.float64), q[:3].cpu().numpy(), pool.cpu().numpy(), pages[:3], lens[:3], [1] * 3, d, g,
            h, 1, 0.1)
