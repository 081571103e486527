"""The decoder harness behind a shared prefix, over a cache that evicts, and with rules on its logits."""
import numpy as np
import pytest
import torch

import serving_oracle as so

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOL = 3 * 2.0 ** -11 * 1.02  # of sum P |v|: as in test_gpu_prefix.py


@pytest.fixture(scope="module")
def opt(built_lib):
    from sqamd import opt_decode
    return opt_decode


def small(opt, heads=4, hd=128, layers=2, seed=0, vocab=1000):
    model = opt.OPTDecoder(layers=layers, hidden=heads * hd, heads=heads, ffn=2 * heads * hd, vocab=vocab, max_pos=512, group=128,
                           dev=DEV, seed=seed)
    for layer in model.layers:
        layer.fuse_qkv()
        layer.capture = {}
    return model


def ids_of(seed, *shape):
    return torch.randint(0, 1000, shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))


def captured(layer):
    return [layer.capture[n].cpu().numpy() for n in "qkva"]


def check_causal(a, q, k, v, pos0, what):
    """a [B, H, T, D] against attention over the rows k, v [B, H, N, D], query i seeing rows 0 .. pos0 + i."""
    b, h, t, d = q.shape
    for i in range(t):
        n = pos0 + i + 1
        s = np.einsum("bhd,bhnd->bhn", q[:, :, i].astype(np.float64), k[:, :, :n].astype(np.float64)) / np.sqrt(d)
        p = so._softmax(s)
        want = np.einsum("bhn,bhnd->bhd", p, v[:, :, :n].astype(np.float64))
        size = np.einsum("bhn,bhnd->bhd", p, np.abs(v[:, :, :n].astype(np.float64)))
        assert (np.abs(a[:, :, i] - want) <= TOL * size + 1e-6).all(), (what, i, np.abs(a[:, :, i] - want).max())


def capture_graph(step, warm):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        warm()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    warm()
    torch.cuda.synchronize()
    return graph


@pytest.mark.parametrize("hd,heads,p,own", [(128, 4, 70, 33), (64, 8, 130, 1)])
def test_prompts_and_steps_behind_a_prefix(opt, hd, heads, p, own):
    model = small(opt, heads, hd)
    prefix_ids, ids = ids_of(1, p), ids_of(2, 3, own)
    cache = model.prefix_cache(prefix_ids, 3, p + own + 20)
    shared = [[x.cpu().numpy()[None].repeat(3, 0) for x in (cache.k_prefix[i], cache.v_prefix[i])] for i in range(2)]
    tok = model(ids, cache, p).argmax(-1)
    rows = []
    for i, layer in enumerate(model.layers):
        q, k, v, a = captured(layer)
        rows.append([np.concatenate([s, x], 2) for s, x in zip(shared[i], (k, v))])
        check_causal(a, q, *rows[i], p, "prompt")
        assert np.array_equal(cache.k[i, :, :, :own].cpu().numpy(), k)
    # the same as every sequence running prefix and prompt through a cache of its own: its first layer's rows differ by the
    # linears' summation order alone, so what it attends to is checked here, not its logits
    pos = p + own
    for step in range(3):
        if step < 2:
            model.greedy_step(tok, cache, torch.tensor([pos], device=DEV))
            t = 1
        else:  # several tokens at once
            t = 4
            model(ids_of(3, 3, t), cache, pos)
        for i, layer in enumerate(model.layers):
            q, k, v, a = captured(layer)
            rows[i] = [np.concatenate([s, x], 2) for s, x in zip(rows[i], (k, v))]
            check_causal(a, q, *rows[i], pos, step)
        pos += t
    with pytest.raises(ValueError):
        model(ids_of(4, 3, 40), cache, pos)
    with pytest.raises(ValueError):
        model(ids_of(4, 3, 1), cache, p - 1)
    with pytest.raises(ValueError):
        model(ids_of(4, 4, 1), cache, pos)
    model.set_prefill_lut(own + 1, 0.5)
    with pytest.raises(ValueError):
        model(ids_of(4, 3, 2), cache, p)


@pytest.mark.parametrize("window", [None, 16])
def test_prompt_and_steps_over_a_cache_that_evicts(opt, window):
    heads, hd, room, first, last, n = 4, 128, 40, 2, 10, 75
    model = small(opt, heads, hd)
    cache = model.new_cache(2, 400, rows=room, keep_first=first, keep_last=last, window=window)
    tok = model(ids_of(5, 2, n), cache, 0).argmax(-1)
    for i, layer in enumerate(model.layers):
        q, k, v, a = captured(layer)
        check_causal(a, q, k, v, 0, "prompt")
        w = so.attention_weights(q, k, [n, n], hd ** -0.5, window)
        pos, weight = cache.position[i].cpu().numpy(), cache.weight[i].cpu().numpy()
        for b in range(2):
            for h in range(heads):
                kept = pos[b, h]
                assert (np.diff(kept) > 0).all() and set(range(first)) <= set(kept) and set(range(n - last, n)) <= set(kept)
                assert np.allclose(weight[b, h], w[b, h, kept], rtol=2e-4, atol=0)  # the bound of test_gpu_evict.py, rounded up
                # none that went weighs more than one that stayed, but for that error
                others = [r for r in range(first, n - last) if r not in set(kept)]
                stayed = [r for r in kept if first <= r < n - last]
                assert w[b, h, others].max() <= w[b, h, stayed].min() * (1 + 4e-4)
                assert np.array_equal(cache.k[i, b, h].cpu().numpy(), k[b, h, kept])
                assert np.array_equal(cache.v[i, b, h].cpu().numpy(), v[b, h, kept])
    pos = n
    for step in range(3):
        before = [[x[i].cpu().numpy() for x in (cache.k, cache.v, cache.weight, cache.position)] for i in range(2)]
        if step == 1:
            model(tok, cache, pos)
        else:
            model.greedy_step(tok, cache, torch.tensor([pos], device=DEV))
        pos += 1
        for i, layer in enumerate(model.layers):
            q, k, v, a = (x[:, :, 0] for x in captured(layer))
            out, size, _, kr, vr, wr, pr = so.evict_step(q, k, v, *before[i], np.array([pos, pos]), hd ** -0.5, first, last)
            assert (np.abs(a - out) <= TOL * size + 1e-6).all()
            assert np.array_equal(cache.k[i].cpu().numpy(), kr) and np.array_equal(cache.v[i].cpu().numpy(), vr)
            assert np.array_equal(cache.position[i].cpu().numpy(), pr)
            assert np.allclose(cache.weight[i].cpu().numpy(), wr, rtol=2e-4, atol=0)
    with pytest.raises(ValueError):
        model(ids_of(6, 2, 3), cache, pos)
    with pytest.raises(ValueError):
        model(ids_of(6, 3, 1), cache, pos)
    with pytest.raises(ValueError):
        model.new_cache(2, 400, kv_bits=4, rows=16)
    with pytest.raises(ValueError):
        model.new_cache(2, 400, rows=16, keep_first=10, keep_last=10)


@pytest.mark.parametrize("kind", ["prefix", "evict"])
def test_captured_steps_generate_what_eager_ones_do(opt, kind):
    model = small(opt)
    for layer in model.layers:
        layer.capture = None
    tokens = {}
    for graphed in (False, True):
        if kind == "prefix":
            cache, pos0 = model.prefix_cache(ids_of(7, 60), 2, 200), 60
        else:
            cache, pos0 = model.new_cache(2, 200, rows=24), 0
        ids = ids_of(8, 2, 30)
        start = model(ids, cache, pos0).argmax(-1)
        tok, pos, hist, at = start.clone(), torch.tensor([pos0 + 30], device=DEV), torch.zeros((12, 2), dtype=torch.long, device=DEV), \
            torch.zeros(1, dtype=torch.long, device=DEV)

        def step():
            model.greedy_step(tok, cache, pos, hist, at)

        def back():  # (the warm-up took a step: the prompt again puts the cache back)
            model(ids, cache, pos0)
            tok.copy_(start)
            pos.fill_(pos0 + 30)
            at.zero_()

        run = capture_graph(step, back).replay if graphed else step
        for _ in range(12):
            run()
        torch.cuda.synchronize()
        tokens[graphed] = hist.cpu()
        assert int(pos) == pos0 + 42 and int(at) == 12
    assert torch.equal(tokens[False], tokens[True])


def test_steps_under_rules(opt):
    from sqamd import logits
    model = small(opt)
    for layer in model.layers:
        layer.capture = None
    b, n, steps, v = 3, 10, 6, 1000
    ids = ids_of(9, b, n)
    start = model(ids, model.new_cache(b, 64), 0).argmax(-1)
    banned = torch.full((b, 32), -1, dtype=torch.int32, device=DEV)
    rules = logits.Rules(repetition=torch.full((b,), 1.3, device=DEV), presence=torch.full((b,), 0.5, device=DEV),
                         frequency=torch.full((b,), 0.2, device=DEV), generated_from=torch.full((b,), n, device=DEV),
                         bias_ids=torch.tensor([[5, 7]] * b, dtype=torch.int32, device=DEV),
                         bias=torch.tensor([[1.0, -2.0]] * b, device=DEV), mask=banned)
    seen = {}
    for graphed in (False, True):
        cache = model.new_cache(b, 64)
        model(ids, cache, 0)
        hist = torch.zeros((n + 1 + steps, b), dtype=torch.long, device=DEV)
        hist[:n], hist[n] = ids.t(), start.view(-1)
        tok, pos, at = start.clone(), torch.tensor([n], device=DEV), torch.tensor([n + 1], device=DEV)
        out = torch.empty((b, v), dtype=torch.float16, device=DEV)
        banned.fill_(-1)

        def step():
            out.copy_(model.greedy_step(tok, cache, pos, hist, at, rules))

        def back():
            hist[n + 1:] = 0
            tok.copy_(start)
            pos.fill_(n)
            at.fill_(n + 1)

        run = capture_graph(step, back).replay if graphed else step
        got = []
        for i in range(steps):
            text = hist[:n + 1 + i].t().cpu().numpy()
            run()
            torch.cuda.synchronize()
            got.append(out.clone())
            assert torch.equal(tok.view(-1), hist[n + 1 + i]) and int(pos) == n + 1 + i and int(at) == n + 2 + i
            assert tok.view(-1).tolist() == so.best_token(out.cpu().numpy()).tolist()
            if not graphed:
                # the same step without rules gives the logits that the oracle applies them to
                plain_tok = torch.from_numpy(text[:, -1:].copy()).to(DEV)
                plain = model.greedy_step(plain_tok, cache, torch.tensor([n + i], device=DEV)).cpu().numpy()
                want = so.logit_rules(plain, text, None, np.full(b, n), np.full(b, 1.3, np.float32), np.full(b, 0.5, np.float32),
                                      np.full(b, 0.2, np.float32), np.array([[5, 7]] * b), np.array([[1.0, -2.0]] * b, np.float32),
                                      banned.cpu().numpy(), dtype=np.float32).astype(np.float16)
                assert np.array_equal(out.cpu().numpy(), want)
            # the token just chosen is banned from now on
            for r, t in enumerate(tok.view(-1).tolist()):
                word = int(banned[r, t // 32]) & 0xffffffff & ~(1 << (t % 32))
                banned[r, t // 32] = word - (1 << 32) if word >= 1 << 31 else word
        seen[graphed] = hist.cpu(), torch.stack(got).cpu()
        assert all(len(set(hist[n + 1:, r].tolist())) == steps for r in range(b))  # nothing twice
    assert torch.equal(seen[False][0], seen[True][0]) and torch.equal(seen[False][1], seen[True][1])


def test_end_to_end_figures(opt):
    for kw, what in (({"shared": 64}, "shared_prefix"), ({"rows": 48}, "cache_rows")):
        got = opt.run_e2e(batch=2, prompt=40, new_tokens=6, layers=1, return_tokens=True, **kw)
        eager = opt.run_e2e(batch=2, prompt=40, new_tokens=6, layers=1, return_tokens=True, use_graph=False, **kw)
        assert got[what] == list(kw.values())[0] and got["logits_finite"] and torch.equal(got["tokens"], eager["tokens"])
    with pytest.raises(ValueError):
        opt.run_e2e(batch=1, prompt=8, new_tokens=2, layers=1, shared=4, rows=4)


def test_end_to_end_over_a_cache_that_evicts_from_the_prompt_on(opt, monkeypatch):
    # fewer rows than the prompt has: a step in front of the first would leave its token's row and its weights in the cache
    caches, plain = [], opt.OPTDecoder.new_cache

    def new_cache(self, *args, **kw):
        caches.append(plain(self, *args, **kw))
        return caches[-1]

    monkeypatch.setattr(opt.OPTDecoder, "new_cache", new_cache)
    for rows in (24, 44):  # (44: more than the prompt's, but not than all)
        got = [opt.run_e2e(batch=2, prompt=40, new_tokens=9, layers=2, rows=rows, use_graph=graph, return_tokens=True)["tokens"]
               for graph in (True, False)]
        a, b = caches[-2:]
        assert torch.equal(*got)
        assert torch.equal(a.position, b.position) and torch.equal(a.weight, b.weight) and torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
        for i in range(2):
            for j in range(2):
                kept = a.position[i, j].cpu().numpy()
                assert all(len(set(kept[h])) == rows for h in range(kept.shape[0]))  # no token twice


def test_rules_without_texts_are_refused_before_the_step(opt):
    from sqamd import logits
    model = small(opt)
    cache = model.new_cache(2, 64, rows=20)
    tok = model(ids_of(10, 2, 30), cache, 0).argmax(-1)
    before = [x.clone() for x in (cache.k, cache.v, cache.weight, cache.position, tok)]
    pos = torch.tensor([30], device=DEV)
    with pytest.raises(ValueError):
        model.greedy_step(tok, cache, pos, rules=logits.Rules(presence=torch.ones(2, device=DEV)))
    assert int(pos) == 30 and all(torch.equal(a, c) for a, c in zip(before, (cache.k, cache.v, cache.weight, cache.position, tok)))


@pytest.mark.parametrize("heads,h,d,n", [(8, 2, 64, 50), (6, 1, 128, 131), (4, 4, 64, 50), (8, 2, 64, 1), (8, 2, 64, 0)])
def test_an_evicting_cache_with_shared_heads(opt, heads, h, d, n):
    from sqamd import evict
    rng = np.random.default_rng(heads + n)
    b, room, first, last, scale = 2, 40, 2, 8, 0.11
    cache = evict.EvictCache(1, b + 1, h, d, room, first, last, device=DEV)

    def rows(t):
        x = rng.normal(0, 1, (b, t, heads + 2 * h, d)).astype(np.float16)
        y = torch.from_numpy(x).to(DEV).transpose(1, 2)
        return [v.transpose(0, 2, 1, 3) for v in np.split(x, [heads, heads + h], 2)], (y[:, :heads], y[:, heads:heads + h], y[:, heads + h:])

    (q, k, v), given = rows(n)
    cache.set_position(b, 0, n)
    a = cache.attention(0, *given, scale)
    assert a.shape == (b, n, heads, d)
    share = heads // h
    if n:
        a = a.transpose(1, 2).cpu().numpy()
        for i in range(n):
            p = so._softmax(np.einsum("bhd,bhnd->bhn", q[:, :, i].astype(np.float64), k[:, :, :i + 1].repeat(share, 1).astype(np.float64)) * scale)
            wide = v[:, :, :i + 1].repeat(share, 1).astype(np.float64)
            want, size = np.einsum("bhn,bhnd->bhd", p, wide), np.einsum("bhn,bhnd->bhd", p, np.abs(wide))
            assert (np.abs(a[:, :, i] - want) <= TOL * size + 1e-6).all(), i
        w = so.attention_weights(q, k, [n] * b, scale)
        weight, pos = cache.weight[0].cpu().numpy(), cache.position[0].cpu().numpy()
        for i in range(b):
            for j in range(h):
                kept = pos[i, j, :min(n, room)]
                assert np.allclose(weight[i, j, :len(kept)], w[i, j, kept], rtol=4e-4, atol=0)
                assert np.array_equal(cache.k[0, i, j, :len(kept)].cpu().numpy(), k[i, j, kept])
    for step in range(3):
        before = [x[0, :b].cpu().numpy() for x in (cache.k, cache.v, cache.weight, cache.position)]
        (q, k, v), given = rows(1)
        cache.set_position(b, n + step, 1)
        a = cache.attention(0, *given, scale)[:, 0].cpu().numpy()
        out, size, _, kr, vr, wr, pr = so.evict_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], *before, np.full(b, n + step + 1), scale, first, last)
        assert (np.abs(a - out) <= TOL * size + 1e-6).all()
        assert np.array_equal(cache.k[0, :b].cpu().numpy(), kr) and np.array_equal(cache.position[0, :b].cpu().numpy(), pr)
        assert np.allclose(cache.weight[0, :b].cpu().numpy(), wr, rtol=4e-4, atol=0)
    assert (cache.k[0, b:] == 0).all() and (cache.weight[0, b:] == 0).all()


def test_a_prompt_of_too_many_rows_for_one_call(built_lib):
    # 2^21 tokens of 32 heads are twice what a call takes: sequences and heads are dealt to several, and agree with one of the parts
    from sqamd import evict, prefix
    gen = torch.Generator(device=DEV).manual_seed(0)
    b, heads, h, t, d = 2100, 32, 16, 512, 64
    q, k = (torch.randn((b, n, 1, d), device=DEV, generator=gen).half().expand(b, n, t, d) for n in (heads, h))
    v = torch.randn((1, h, t, d), device=DEV, generator=gen).half().expand(b, h, t, d)
    assert b * t * heads > 1 << 25
    out = evict._prompt_attention(q, k, v, 0.125)
    # all keys of a sequence are one, so the rows are the means of the values so far
    want = v[0].double().cumsum(1) / torch.arange(1, t + 1, device=DEV)[:, None]
    size = v[0].double().abs().cumsum(1) / torch.arange(1, t + 1, device=DEV)[:, None]
    off = (out.view(b, t, h, 2, d) - want.transpose(0, 1)[None, :, :, None]).abs().amax((0, 3))
    assert (off <= TOL * size.transpose(0, 1) + 1e-6).all()


@pytest.mark.parametrize("rows", [1, 50 * 2 * 3, 50 * 8 * 2])
def test_a_prompt_dealt_to_several_calls(built_lib, monkeypatch, rows):
    # a head at a time, three heads, two sequences of three
    from sqamd import evict
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn((3, 50, 16, 64), device=DEV, generator=gen).half().transpose(1, 2)
    q, k, v = x[:, :8], x[:, 8:12], x[:, 12:]
    monkeypatch.setattr(evict, "_MOST_ROWS", rows)
    a = evict._prompt_attention(q, k, v, 0.125).transpose(1, 2).cpu().numpy()
    q, k, v = (y.cpu().numpy() for y in (q, k.repeat_interleave(2, 1), v.repeat_interleave(2, 1)))
    check_causal(a, q, k, v, 0, rows)


def test_positions_behind_the_models_last_are_refused(opt):
    model = small(opt)
    cache = model.new_cache(2, 64, rows=20)
    last = model.pos.shape[0] - 2  # (512)
    model(ids_of(11, 2, 30), cache, 0)
    seen = cache.seen.clone()
    for ids, pos in ((ids_of(12, 2, 1), last), (ids_of(12, 2, 1), 1 << 40), (ids_of(12, 2, last + 1), 0)):
        with pytest.raises(ValueError):
            model(ids, cache, pos)
    assert torch.equal(cache.seen, seen)
    model(ids_of(12, 2, 1), cache, last - 1)
