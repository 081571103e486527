"""The 4-bit cache without a GPU: refusals of the C ABI before any launch, sizes, and the oracle against itself."""
import ctypes

import numpy as np
import pytest
import torch

import kv4_oracle as ko

SIZES = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)]


@pytest.mark.parametrize("d,g", SIZES)
def test_every_code_and_scale_has_its_own_place(d, g):
    p = ko.places(d, g)
    nibbles = np.concatenate([(2 * p["kb"] + p["ks"] // 4).ravel(), (2 * p["vb"] + p["vs"] // 4).ravel()])
    assert np.array_equal(np.sort(nibbles), np.arange(2 * 64 * d))  # all nibbles of the first 64 D bytes, each once
    halves = np.unique(np.concatenate([(p[n] + o).ravel() for n in ("ksm", "vsm") for o in (0, 8)]))
    assert np.array_equal(halves, 64 * d + 2 * np.arange(256 * (d // g)))
    for n in ("ksm", "vsm"):
        assert np.array_equal(p[n][:, ::g].repeat(g, 1), p[n])
    assert ko.record_bytes(d, g) == 64 * d + 512 * (d // g) + 4 * d


def test_quantisation_of_the_oracle():
    x = np.array([[0.0, 1.5, 15.0, 7.5] * 8, [2.0] * 32, [-3.0, 12.0] * 16, [0.0, np.nan] + [1.0] * 30,
                  [np.inf] + [0.0] * 31], dtype=np.float16)
    c, s, m = ko.quantise(x, 32)
    assert c[0, :4].tolist() == [0, 2, 15, 8]  # 1.5 and 7.5 are halves: to the even code
    assert np.all(c[1] == 0) and np.all(s[1] == 0) and np.all(m[1] == 2.0)
    assert np.all(s[2] == 1.0) and np.all(m[2] == -3.0) and c[2, :2].tolist() == [0, 15]
    with np.errstate(invalid="ignore"):
        assert np.all(np.isnan(ko.values(c, s, m)[3:]))


@pytest.fixture(scope="module")
def L(built_lib):
    from sqamd import capi
    return capi.lib()


@pytest.fixture(scope="module")
def p():
    buf = np.zeros(64, dtype=np.uint8)
    test_p = ctypes.c_void_p(buf.ctypes.data - buf.ctypes.data % 16 + 16)
    test_p.keep = buf
    return test_p


def test_record_bytes(L):
    from sqamd import kv4
    for d, g in SIZES:
        assert L.sq_kv4_record_bytes(d, g) == kv4.record_bytes(d, g) == ko.record_bytes(d, g)
    for d, g in ((96, 32), (64, 128), (128, 16), (0, 0), (128, 48)):
        assert L.sq_kv4_record_bytes(d, g) == 0
        with pytest.raises(ValueError):
            kv4.record_bytes(d, g)


def test_append_refuses(L, p):
    from sqamd import capi
    strides = (ctypes.c_long * 4)(1024, 128, 1024, 128)

    def call(k=p, v=p, kh=None, vh=None, pool=p, pages=p, lengths=p, starts=None, T=4, B=4, H=8, D=128, g=64, n=10, width=5,
             stride=5, st=strides):
        return L.sq_kv4_append(k, v, kh, vh, pool, pages, lengths, starts, T, B, H, D, g, n, width, stride, st, None)

    odd = ctypes.c_void_p(p.value + 2)
    null, shape, group, misaligned = (capi.SQ_ERR_NULL_POINTER, capi.SQ_ERR_BAD_SHAPE, capi.SQ_ERR_BAD_GROUP,
                                      capi.SQ_ERR_MISALIGNED)
    assert call(T=0) == capi.SQ_OK and call(T=0, B=0) == capi.SQ_OK and call(width=0, stride=0) == capi.SQ_OK
    for bad in (dict(k=None), dict(v=None), dict(pool=None), dict(pages=None), dict(lengths=None), dict(kh=p), dict(vh=p),
                dict(st=None)):
        assert call(**bad) == null, bad
    for bad in (dict(T=-1), dict(B=-1), dict(H=0), dict(D=96), dict(n=0), dict(width=-1), dict(width=6), dict(T=5),
                dict(st=(ctypes.c_long * 4)(-8, 128, 1024, 128)), dict(T=1 << 28, B=1 << 28)):
        assert call(**bad) == shape, bad
    for bad in (dict(g=16), dict(g=128, D=64), dict(g=0)):
        assert call(**bad) == group, bad
    for bad in (dict(k=odd), dict(v=odd), dict(kh=odd, vh=odd), dict(pool=odd), dict(lengths=odd), dict(starts=odd),
                dict(st=(ctypes.c_long * 4)(1024, 128, 1020, 128))):
        assert call(**bad) == misaligned, bad


def test_attention_refuses(L, p):
    from sqamd import capi

    def call(q=p, out=p, pool=p, pages=p, lengths=p, starts=None, sel=None, T=4, B=4, Hq=16, H=8, D=128, g=64, n=10, width=5,
             stride=5, count=0, qt=2048, qh=128, k=None, v=None, st=None, ws=None, size=0):
        return L.sq_kv4_attention(q, out, pool, pages, lengths, starts, sel, T, B, Hq, H, D, g, n, width, stride, count, qt, qh,
                                  0.1, k, v, st, ws, size, None)

    strides = (ctypes.c_long * 4)(1024, 128, 1024, 128)
    assert call(k=p) == call(v=p, st=strides) == call(k=p, v=p) == capi.SQ_ERR_NULL_POINTER
    assert call(k=p, v=p, st=strides, sel=p, count=2) == capi.SQ_ERR_BAD_SHAPE
    assert call(k=ctypes.c_void_p(p.value + 2), v=p, st=strides) == capi.SQ_ERR_MISALIGNED
    assert call(k=p, v=p, st=(ctypes.c_long * 4)(1024, 128, 1020, 128)) == capi.SQ_ERR_MISALIGNED
    assert call(k=p, v=p, st=(ctypes.c_long * 4)(1024, -128, 1024, 128)) == capi.SQ_ERR_BAD_SHAPE

    odd = ctypes.c_void_p(p.value + 2)
    assert call(T=0) == capi.SQ_OK and call(T=0, B=0) == capi.SQ_OK
    for bad in (dict(q=None), dict(out=None), dict(pool=None), dict(lengths=None), dict(pages=None)):
        assert call(**bad) == capi.SQ_ERR_NULL_POINTER, bad
    for bad in (dict(Hq=12), dict(Hq=0), dict(T=6), dict(D=80), dict(n=0), dict(stride=4), dict(qt=-8), dict(sel=p, count=0),
                dict(sel=p, count=2, starts=p), dict(sel=p, count=2, T=8), dict(T=1 << 27, B=1, Hq=64, H=1)):
        assert call(**bad) == capi.SQ_ERR_BAD_SHAPE, bad
    for bad in (dict(q=odd), dict(out=odd), dict(qh=100), dict(sel=odd, count=2)):
        assert call(**bad) == capi.SQ_ERR_MISALIGNED, bad
    assert call(g=256) == capi.SQ_ERR_BAD_GROUP
    need = L.sq_kv4_attention_workspace_bytes
    assert call(ws=p, size=16, width=500, stride=500) == capi.SQ_ERR_WORKSPACE
    assert call(ws=odd, size=1 << 30) == capi.SQ_ERR_WORKSPACE
    assert call(ws=p, size=need(4, 4, 16, 8, 128, 500, 0) - 1, width=500, stride=500) == capi.SQ_ERR_WORKSPACE
    assert need(4, 4, 16, 8, 128, 4, 0) == 0 == need(4, 4, 16, 8, 128, 500, 4)  # too short to be dealt out
    assert need(4, 4, 16, 8, 96, 500, 0) == 0 < need(4, 4, 16, 8, 64, 500, 0) < need(4, 4, 16, 8, 128, 500, 0)
    assert need(0, 4, 16, 8, 128, 500, 0) == 0 == need(4, 4, 12, 8, 128, 500, 0)


def test_select_refuses(L, p):
    from sqamd import capi

    def call(q=p, sel=p, B=4, Hq=16, H=8, D=128, g=64, n=10, width=50, stride=50, count=4, first=1, last=1, qt=2048, qh=128,
             ws=p, size=1 << 20):
        return L.sq_kv4_select(q, sel, p, p, p, B, Hq, H, D, g, n, width, stride, count, first, last, qt, qh, ws, size, None)

    assert call(B=0) == capi.SQ_OK
    for bad in (dict(count=0), dict(count=1), dict(first=-1), dict(last=-1), dict(first=4), dict(width=16385, stride=16385),
                dict(B=1 << 14), dict(Hq=20), dict(first=2 ** 31 - 1, last=2 ** 31 - 1)):
        assert call(**bad) == capi.SQ_ERR_BAD_SHAPE, bad
    for bad in (dict(q=None), dict(sel=None)):
        assert call(**bad) == capi.SQ_ERR_NULL_POINTER, bad
    need = L.sq_kv4_select_workspace_bytes(4, 8, 50)
    assert need > 0 and call(ws=None) == capi.SQ_ERR_WORKSPACE and call(size=need - 1) == capi.SQ_ERR_WORKSPACE
    assert L.sq_kv4_select_workspace_bytes(0, 8, 50) == 0


def test_copy_refuses(L, p):
    from sqamd import capi

    def call(pool=p, src=p, dst=p, n=3, pages=8, layers=2, page=4864, layer=8 * 4864):
        return L.sq_kv4_copy_pages(pool, src, dst, n, pages, layers, page, layer, None)

    assert call(n=0) == capi.SQ_OK
    for bad in (dict(n=-1), dict(pages=0), dict(layers=0), dict(page=0), dict(page=4860), dict(layer=8 * 4864 - 16),
                dict(layer=8 * 4864 + 8), dict(layers=1 << 16)):
        assert call(**bad) == capi.SQ_ERR_BAD_SHAPE, bad
    for bad in (dict(pool=None), dict(src=None), dict(dst=None)):
        assert call(**bad) == capi.SQ_ERR_NULL_POINTER, bad
    assert call(src=ctypes.c_void_p(p.value + 2)) == capi.SQ_ERR_MISALIGNED


def test_python_refuses_host_tensors():
    from sqamd import kv4
    pool = kv4.new_pool(4, 2, 64, 32, device="cpu")
    pages, lengths = torch.zeros((1, 4), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x = torch.zeros((1, 2, 64), dtype=torch.float16)
    for call in (lambda: kv4.append(x, x, pool, pages, lengths), lambda: kv4.attention(x, pool, pages, lengths, 1.0),
                 lambda: kv4.select_pages(x, pool, pages, lengths, 2), lambda: kv4.copy_pages(pool, lengths, lengths)):
        with pytest.raises(ValueError):
            call()


def test_bookkeeping_without_copies():
    # sequences that share nothing need no device work but the tables': the host's side runs anywhere
    from sqamd import kv4
    c = kv4.KV4Cache(2, 10, 1, 64, 64, max_seqs=3, max_rows=300, device="cpu")
    a, b = c.add(), c.add()
    c.extend([a, b], [130, 1])
    assert c.pages(a) == [0, 1, 2] and c.pages(b) == [3] and c.free_pages() == 6
    assert c.lengths.tolist() == [130, 1, 0] and c.table[a, :3].tolist() == [0, 1, 2]
    c.extend([b], 63)
    assert c.pages(b) == [3]
    c.extend([b], 1)
    assert c.pages(b) == [3, 4]
    c.truncate(a, 64)
    assert c.pages(a) == [0] and c.rows(a) == 64 and c.free_pages() == 7
    with pytest.raises(ValueError):
        c.truncate(a, 65)
    with pytest.raises(ValueError):
        c.extend([a], 300)
    with pytest.raises(ValueError):
        c.extend([a, a], 1)
    with pytest.raises(ValueError):
        c.rows(2)
    f = c.fork(a)  # a full page: shared, no copy
    assert c.pages(f) == [0] and c.free_pages() == 7
    c.extend([f, a], 1)
    assert c.pages(f) == [0, 1] and c.pages(a) == [0, 2] and c.free_pages() == 5
    c.free(a)
    assert c.free_pages() == 6
    c.free(f)
    assert c.free_pages() == 8 and c.pages(b) == [3, 4]
    with pytest.raises(ValueError):
        c.free(f)
    big, more = c.add(), c.add()
    c.reserve([big], 300)
    assert c.free_pages() == 3 and c.rows(big) == 0
    with pytest.raises(RuntimeError):
        c.reserve([more, b], [130, 130])
    assert c.free_pages() == 3 and c.pages(more) == [] and c.pages(b) == [3, 4]
    with pytest.raises(RuntimeError):
        c.add()


def test_bookkeeping_refuses_what_would_write_into_shared_or_unknown_pages():
    from sqamd import kv4
    c = kv4.KV4Cache(1, 10, 1, 64, 64, max_seqs=3, max_rows=300, device="cpu")
    a = c.add()
    c.reserve([a], 200)
    c.set_lengths([a], [70])
    b = c.fork(a)
    for seq in (a, b):  # the page of rows 64 to 69 is shared: no more rows in it before one of them has its own
        with pytest.raises(ValueError):
            c.set_lengths([seq], 71)
    c.set_lengths([a], 64)
    with pytest.raises(ValueError):
        c.set_lengths([a], 65)
    c.free(b)
    c.set_lengths([a], 200)
    x = torch.zeros((2, 1, 64), dtype=torch.float16)
    for call in (lambda: c.batch([0, 1]), lambda: c.batch([3]), lambda: c.batch([-1]), lambda: c.batch(4), lambda: c.batch(-1),
                 lambda: c.append(0, x, x, [a, a]), lambda: c.attention(0, x, 1.0, [a, a], k_new=x, v_new=x)):
        with pytest.raises(ValueError):
            call()
    c.set_lengths(iter([a]), (n for n in [199]))  # any iterable of numbers
    c.set_lengths(torch.tensor([a]), torch.tensor([200]))
    with pytest.raises(ValueError):
        c.append(0, x, x, torch.tensor([a, a]))
    assert c.batch(iter([a]))[1].tolist() == [200]
    assert [t.shape[0] for t in c.batch([a, a])] == [2, 2] and c.batch(3)[1].tolist() == [200, 0, 0]
    for wrong in ((0, 10, 1, 64, 64, 3, 300), (1, 0, 1, 64, 64, 3, 300), (1, 10, 1, 64, 64, 0, 300), (1, 10, 1, 64, 64, 3, 0),
                  (1, 10, 1, 64, 128, 3, 300), (1, 10, 1, 96, 32, 3, 300)):
        with pytest.raises(ValueError):
            kv4.KV4Cache(*wrong, device="cpu")


@pytest.fixture
def host_copies(monkeypatch):
    """Page copies of a pool on the host, so that the bookkeeping around them runs without a GPU."""
    from sqamd import kv4

    def copy(pool, src, dst):
        pool[:, dst.long()] = pool[:, src.long()]
    monkeypatch.setattr(kv4, "copy_pages", copy)


def only_own_pages(c):
    """Every place of the device's table names the sequence's own page there, or none."""
    for seq, row in enumerate(c.table.tolist()):
        own = c._pages[seq] or []
        if row != own + [-1] * (c.width - len(own)):
            return False
    return True


def test_places_without_a_page_name_none(host_copies):
    # a place that no sequence owns must not name a page: a length counted on the device past it would reach others' rows
    from sqamd import kv4
    c = kv4.KV4Cache(1, 10, 1, 64, 64, max_seqs=3, max_rows=256, device="cpu")
    assert only_own_pages(c)
    a, b = c.add(), c.add()
    c.extend([a, b], [64, 130])
    assert only_own_pages(c)
    c.free(b)
    assert only_own_pages(c)
    c.extend([a], 64)  # on a page that was b's
    assert only_own_pages(c)
    c.extend([a], 70)
    c.truncate(a, 60)
    assert c.pages(a) == [0] and only_own_pages(c)
    b = c.add()
    f = c.fork(a)
    assert only_own_pages(c)
    c.reserve([f, a, b], [200, 61, 64])
    assert only_own_pages(c)
    c.truncate(f, 0)
    c.free(a)
    c.extend([b], 10)
    assert only_own_pages(c)


def test_rows_that_the_device_counts_are_known_to_the_host(host_copies):
    # a decode step counts `lengths` up where the host does not see it: what the host does next starts from there
    from sqamd import kv4, opt_decode
    c = kv4.KV4Cache(1, 20, 1, 64, 64, max_seqs=4, max_rows=400, device="cpu")
    a, b = c.add(), c.add()
    c.reserve([a, b], 200)
    opt_decode._per_layer(c, 2, 60, 0)                      # a prompt: counted by the host
    assert c.rows(a) == 60
    for pos in range(60, 131):                              # steps: by the device
        opt_decode._per_layer(c, 2, 1, torch.tensor([pos]))
    assert c.lengths.tolist() == [131, 131, 0, 0] and c.rows(a) == c.rows(b) == 131
    c.pool.copy_(torch.randint(0, 256, c.pool.shape, dtype=torch.uint8))
    f = c.fork(a)
    assert c.rows(f) == 131 and c.lengths[f] == 131 and c.pages(f)[:2] == c.pages(a)[:2]
    # the step of the first two may be a captured one: the page it goes on writing to is not shared, and no page was lost
    assert c.pages(f)[2] != c.pages(a)[2] and torch.equal(c.pool[0, c.pages(f)[2]], c.pool[0, c.pages(a)[2]])
    assert only_own_pages(c)
    c.extend([a, f], 4)
    assert c.lengths.tolist() == [135, 131, 135, 0]
    c.truncate(a, 130)
    with pytest.raises(ValueError):
        c.truncate(a, 131)
    c.lengths[a] = 190
    c.truncate(a, 180)
    assert c.rows(a) == 180
    c.lengths[a] = 193                                      # past its pages, which end at 192
    for call in (lambda: c.rows(a), lambda: c.fork(a), lambda: c.extend([a], 1), lambda: c.reserve([a], 300)):
        with pytest.raises(RuntimeError):
            call()
    c.truncate(a, 192)
    c.extend([a], 1)
    assert c.rows(a) == 193 and only_own_pages(c)
    c.lengths[b] = 500
    c.set_lengths([b], 190)
    assert c.rows(b) == 190


def test_the_device_never_counts_into_a_shared_page(host_copies):
    from sqamd import kv4
    c = kv4.KV4Cache(1, 6, 1, 64, 64, max_seqs=3, max_rows=256, device="cpu")
    a = c.add()
    c.reserve([a], 128)
    c.set_lengths([a], 70)
    f = c.fork(a)
    for n in (1, 2, [f]):
        with pytest.raises(ValueError):
            c.counted_on_device(n)
    with pytest.raises(ValueError):
        c.counted_on_device([3])
    c.reserve([f], 71)
    c.counted_on_device(3)                                  # the third does not exist yet
    pages, uses = c.pages(a), list(c._uses)
    g = c.fork(f)
    assert g == 2 and c.pages(g)[0] == pages[0] and c._uses[c.pages(g)[1]] == c._uses[c.pages(f)[1]] == 1
    c.free(g)
    assert c._uses == uses
    # back into a shared full page: by truncate and by set_lengths
    c.truncate(f, 64)
    g = c.fork(f)
    c.truncate(g, 30)
    assert c.pages(g)[0] != pages[0] and c.pages(f)[0] == pages[0]
    c.set_lengths([f], 10)
    assert c.pages(f)[0] != pages[0] and c.pages(a) == pages and only_own_pages(c)


def test_a_shared_page_without_a_free_one_leaves_everything_as_it_was(host_copies):
    from sqamd import kv4
    for rows, cut in ((100, None), (128, 100)):
        c = kv4.KV4Cache(1, 2, 1, 64, 64, max_seqs=2, max_rows=256, device="cpu")
        c.counted_on_device(2)
        a = c.add()
        c.extend([a], rows)
        if cut:
            c.fork(a)
        state = lambda: (c._pages[:], c._rows[:], c._uses[:], c._free[:], c.table.tolist(), c.lengths.tolist())
        before = state()
        with pytest.raises(RuntimeError):
            c.truncate(1, cut) if cut else c.fork(a)
        assert state() == before
    c = kv4.KV4Cache(1, 3, 1, 64, 64, max_seqs=2, max_rows=256, device="cpu")
    c.counted_on_device(2)
    a = c.add()
    c.extend([a], 128)
    f = c.fork(a)
    c.extend([f], 64)
    c.truncate(f, 100)  # the page that goes is the one that comes
    assert c.pages(a) == [0, 1] and c.pages(f) == [0, 2] and c.free_pages() == 0 and only_own_pages(c)


def test_a_prompt_is_not_stored_again_over_shared_pages(host_copies):
    from sqamd import kv4, opt_decode
    c = kv4.KV4Cache(1, 10, 1, 64, 64, max_seqs=2, max_rows=300, device="cpu")
    a = c.add()
    c.reserve([a], 200)
    opt_decode._per_layer(c, 1, 130, 0)
    opt_decode._per_layer(c, 1, 130, 0)             # again, on pages of its own
    f = c.fork(a)
    c.reserve([f], 150)
    before = c.lengths.tolist(), c.table.tolist()
    for first, tokens in ((0, 130), (0, 20), (127, 3), (64, 64)):
        with pytest.raises(ValueError):             # the first two pages are the fork's too
            opt_decode._per_layer(c, 1, tokens, first)
    assert (c.lengths.tolist(), c.table.tolist()) == before
    opt_decode._per_layer(c, 2, 5, 130)             # behind them
    opt_decode._per_layer(c, 2, 5, 128)             # again
    opt_decode._per_layer(c, 2, 0, 10)              # nothing is stored
    assert c.lengths.tolist() == [10, 10]
    c.truncate(a, 0)
    c.reserve([a], 130)
    opt_decode._per_layer(c, 1, 130, 0)
    assert not set(c.pages(a)) & set(c.pages(f))


@pytest.mark.parametrize("seed", range(8))
def test_a_random_life_of_a_cache(host_copies, seed):
    # every sequence finds its own rows, whatever the others do, with some counted by the host and some by the device; a row is
    # one byte here, stored where the device's table says
    import random
    from sqamd import kv4
    rng = random.Random(seed)
    c = kv4.KV4Cache(1, 14, 1, 64, 64, max_seqs=5, max_rows=250, device="cpu")
    c.counted_on_device(rng.choice([0, 0, 2, 5]))
    rows = {}

    def store(seq, first, values):
        for r, value in enumerate(values, first):
            page = int(c.table[seq, r // 64]) if r // 64 < c.width else -1
            if page >= 0:
                c.pool[0, page, 0, r % 64] = value

    def check():
        assert only_own_pages(c)
        uses = [0] * c.num_pages
        for seq, own in rows.items():
            assert c.rows(seq) == len(own) == int(c.lengths[seq]) <= 64 * len(c.pages(seq))
            assert [int(c.pool[0, int(c.table[seq, r // 64]), 0, r % 64]) for r in range(len(own))] == own
            for page in c.pages(seq):
                uses[page] += 1
        assert uses == c._uses and sorted(c._free) == [p for p, n in enumerate(uses) if not n]

    for step in range(120):
        seq = rng.choice(sorted(rows)) if rows else None
        what = rng.choice(["add", "extend", "extend", "extend", "fork", "truncate", "free", "compact", "reserve", "device", "device"])
        try:
            if what == "add":
                rows[c.add()] = []
            elif seq is None:
                continue
            elif what == "extend":
                some = sorted(rng.sample(sorted(rows), rng.randint(1, len(rows))))
                more = [rng.randint(0, 70) for _ in some]
                c.extend(some, more)
                for s, n in zip(some, more):
                    new = [rng.randrange(256) for _ in range(n)]
                    store(s, len(rows[s]), new)
                    rows[s] = rows[s] + new
            elif what == "fork":
                rows[c.fork(seq)] = list(rows[seq])
            elif what == "truncate":
                n = rng.randint(0, len(rows[seq]))
                c.truncate(seq, n)
                rows[seq] = rows[seq][:n]
            elif what == "free":
                c.free(seq)
                del rows[seq]
            elif what == "compact":
                assert c.compact() == c.num_pages - c.free_pages()
            elif what == "reserve":
                c.reserve([seq], rng.randint(0, 250))
            elif c._device_counts:  # steps of all that the device counts, as a replayed graph takes them
                room = [64 * len(c.pages(s)) - len(rows[s]) for s in rows if s in c._device_counts]
                for _ in range(min([rng.randint(0, 20)] + room)):
                    for s in sorted(c._device_counts):
                        if s in rows:
                            value = rng.randrange(256)
                            store(s, len(rows[s]), [value])
                            rows[s] = rows[s] + [value]
                            c.lengths[s] += 1
        except (RuntimeError, ValueError) as e:
            assert any(word in str(e) for word in ("wanted", "in use", "in a cache of")), e
        check()
