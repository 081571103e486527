"""The decoder harness over a cache held in 4 bits: prompts, steps, look-up tables, a captured step, a fork."""
import numpy as np
import pytest
import torch

import kv4_oracle as ko

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def opt(built_lib):
    from sqamd import opt_decode
    return opt_decode


def small(opt, heads=4, hd=128, layers=2, seed=0):
    model = opt.OPTDecoder(layers=layers, hidden=heads * hd, heads=heads, ffn=2 * heads * hd, vocab=1000, max_pos=512, group=128,
                           dev=DEV, seed=seed)
    for layer in model.layers:
        layer.fuse_qkv()
    return model


def quantised(x, g):
    """fp16 [T, D] -> an oracle's fields."""
    c, s, m = ko.quantise(x, g)
    return c, s.astype(np.float64), m.astype(np.float64)


def rows_of(k, v, g):
    r = ko.Rows.__new__(ko.Rows)
    (kc, ks, km), (vc, vs, vm) = quantised(k, g), quantised(v, g)
    r.k, r.v, r.k_abs = ks * kc + km, vs * vc + vm, ks * kc + np.abs(km)
    r.v_mid, r.v_rest, r.v_code = np.abs(vs * (vc - 8)), np.abs(8 * vs + vm), vs * (vc + 8)
    return r


def check_layer(cap, k_all, v_all, pos0, g, tokens=None):
    """The captured attention of one call against the oracle over the rows so far (k_all, v_all [B, H, N, D])."""
    q, a = cap["q"].cpu().numpy(), cap["a"].cpu().numpy().astype(np.float64)
    b, h, t, d = q.shape
    for i in range(b):
        for j in range(h):
            r = rows_of(k_all[i, j], v_all[i, j], g)
            for n in tokens if tokens is not None else range(t):
                want, tol = ko.attend(r, q[i, j, n].astype(np.float64), d ** -0.5, np.arange(pos0 + n + 1))
                assert np.all(np.abs(a[i, j, n] - want) <= tol), (i, j, n)


@pytest.mark.parametrize("hd,heads", [(128, 4), (64, 8)])
def test_prompt_then_steps(opt, hd, heads):
    model = small(opt, heads, hd)
    gen = torch.Generator(device=DEV).manual_seed(1)
    ids = torch.randint(0, 1000, (3, 70), device=DEV, generator=gen)
    cache = model.new_cache(3, 200, kv_bits=4)
    g = cache.group_size
    for layer in model.layers:
        layer.capture = {}
    tok = model(ids, cache, 0).argmax(-1)
    kept = [[x.cpu().numpy() for x in (l.capture["k"], l.capture["v"])] for l in model.layers]
    for l, (k, v) in zip(model.layers, kept):
        check_layer(l.capture, k, v, 0, g, tokens=(0, 1, 31, 63, 64, 69))
    pos = 70
    for step in range(3):
        if step == 1:  # several tokens behind a prompt: a chunk
            tok = ids[:, :5].contiguous()
        t = tok.shape[1]
        out = model(tok, cache, pos) if t > 1 else model.greedy_step(tok, cache, torch.tensor([pos], device=DEV))
        for l, kv in zip(model.layers, kept):
            for i, name in enumerate("kv"):
                kv[i] = np.concatenate([kv[i], l.capture[name].cpu().numpy()], 2)
            check_layer(l.capture, *kv, pos, g)
        assert torch.isfinite(out).all() and cache.lengths.tolist() == [pos + t] * 3
        pos += t
        tok = ids[:, :1].contiguous()


def test_prompt_over_a_table_sees_what_the_cache_holds(opt):
    from sqamd import capi
    model = small(opt)
    gen = torch.Generator(device=DEV).manual_seed(2)
    ids = torch.randint(0, 1000, (2, 150), device=DEV, generator=gen)
    model.set_prefill_lut(150, 0.5)
    cache = model.new_cache(2, 160, kv_bits=4, kv_group=32)
    for layer in model.layers:
        layer.capture = {}
    model(ids, cache, 0)
    for layer in model.layers:
        hats = []
        for x in (layer.capture["k"], layer.capture["v"]):
            c, s, m = ko.quantise(x.cpu().numpy(), 32)
            hats.append(torch.from_numpy((s.astype(np.float32) * c + m.astype(np.float32)).astype(np.float16)).to(DEV))
        want = capi.lut_attention_strided(layer.capture["q"].contiguous(), *hats, layer.lut, 128 ** -0.5, True)
        assert torch.equal(layer.capture["a"], want)


def test_captured_steps_are_the_eager_ones(opt):
    model = small(opt, layers=3)
    gen = torch.Generator(device=DEV).manual_seed(3)
    ids = torch.randint(0, 1000, (4, 60), device=DEV, generator=gen)
    runs = []
    for captured in (False, True):
        cache = model.new_cache(4, 100, kv_bits=4)
        tok = model(ids, cache, 0).argmax(-1)
        pos = torch.tensor([60], device=DEV)
        step = torch.zeros(1, dtype=torch.long, device=DEV)
        history = torch.zeros((12, 4), dtype=torch.long, device=DEV)
        if captured:
            first = tok.clone()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                model.greedy_step(tok, cache, pos, history, step)
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                logits = model.greedy_step(tok, cache, pos, history, step)
            tok.copy_(first)
            pos.fill_(60)
            step.zero_()
        for i in range(12):  # over the border of a page
            if captured:
                graph.replay()
            else:
                logits = model.greedy_step(tok, cache, pos, history, step)
        torch.cuda.synchronize()
        runs.append((history.clone(), logits.clone(), cache.lengths.clone()))
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_a_forked_sequence_continues_on_its_own(opt):
    # two continuations of one prompt, decoded as a batch, are what two separate prompts give
    model = small(opt)
    gen = torch.Generator(device=DEV).manual_seed(4)
    ids = torch.randint(0, 1000, (1, 90), device=DEV, generator=gen)
    nxt = torch.randint(0, 1000, (2, 5), device=DEV, generator=gen)
    from sqamd import kv4
    cache = kv4.KV4Cache(len(model.layers), 8, model.heads, 128, max_seqs=2, max_rows=128, device=DEV)
    cache.add()
    cache.reserve([0], 90)
    model(ids, cache, 0)
    assert cache.fork(0) == 1 and cache.pages(1) == cache.pages(0)
    cache.reserve([0, 1], 95)
    assert cache.pages(1)[0] == cache.pages(0)[0] and cache.pages(1)[1] != cache.pages(0)[1]
    out = model(nxt, cache, 90)
    for i in range(2):
        alone = model.new_cache(1, 128, kv_bits=4)
        model(ids, alone, 0)
        # (one row of tokens fewer takes the linears' other kernels: fp16 roundings apart)
        want = model(nxt[i:i + 1], alone, 90)
        assert torch.allclose(out[i].float(), want[0].float(), atol=2e-2, rtol=2e-2)
        for layer in range(len(model.layers)):
            for p, q in zip(cache.pages(i)[:1], alone.pages(0)[:1]):
                assert torch.equal(cache.pool[layer, p], alone.pool[layer, q])


def test_other_widths_are_refused(opt):
    model = small(opt)
    with pytest.raises(ValueError):
        model.new_cache(1, 64, kv_bits=8)
    with pytest.raises(ValueError):
        model.new_cache(1, 64, kv_bits=4, kv_group=256)


def test_steps_past_the_reserved_pages_leave_other_sequences_alone(opt):
    # the device counts every sequence of the batch: one that has ended, and one at the end of its pages, store nowhere
    model = small(opt)
    from sqamd import kv4
    gen = torch.Generator(device=DEV).manual_seed(5)
    ids = torch.randint(0, 1000, (3, 60), device=DEV, generator=gen)
    cache = kv4.KV4Cache(len(model.layers), 8, model.heads, 128, max_seqs=4, max_rows=256, device=DEV)
    cache.pool.zero_()
    for _ in range(3):
        cache.add()
    cache.reserve([0, 1, 2], 60)
    model(ids, cache, 0)
    cache.free(1)
    cache.reserve([0], 200)          # the first gets the page that was the second's; the third has rows up to 64 only
    assert cache.pages(0)[1] == 1
    tok, pos = ids[:, :1].contiguous(), torch.tensor([60], device=DEV)
    for _ in range(4):
        model.greedy_step(tok, cache, pos)
    before = cache.pool.clone()
    for _ in range(6):               # rows 64 to 69
        logits = model.greedy_step(tok, cache, pos)
    assert torch.isfinite(logits[0]).all()
    # what has changed: six rows of the first sequence's second page and its bounds, in every layer
    changed = torch.nonzero((cache.pool != before).flatten(2).any(2))
    assert sorted(set(changed[:, 1].tolist())) == [1] and len(changed) == len(model.layers)
    new, old = (ko.read(x[:, 1].cpu().numpy(), 128, 64) for x in (cache.pool, before))
    for name in ("kc", "vc", "ks", "vs", "km", "vm"):
        assert np.array_equal(new[name][..., 6:, :], old[name][..., 6:, :]), name
    assert np.any(new["kc"][..., :6, :] != old["kc"][..., :6, :])


@pytest.mark.parametrize("captured", [False, True], ids=["eager", "captured"])
def test_steps_then_a_fork(opt, captured):
    # the device has counted rows that the host did not see: a fork has them all, and steps that go on (replays cannot be
    # refused) leave it alone
    model = small(opt)
    from sqamd import kv4
    gen = torch.Generator(device=DEV).manual_seed(6)
    ids = torch.randint(0, 1000, (2, 60), device=DEV, generator=gen)
    runs = []
    for forked in (False, True):
        cache = kv4.KV4Cache(len(model.layers), 16, model.heads, 128, max_seqs=3, max_rows=192, device=DEV)
        cache.pool.zero_()
        cache.add(), cache.add()
        cache.reserve([0, 1], 192)
        tok, pos = model(ids, cache, 0).argmax(-1), torch.tensor([60], device=DEV)
        first, step = tok.clone(), lambda: model.greedy_step(tok, cache, pos)
        if captured:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step()
            tok.copy_(first)
            pos.fill_(60)
            step = graph.replay
        for _ in range(10):
            step()
        if forked:
            assert cache.rows(0) == 70 and cache.fork(0) == 2 and cache.rows(2) == 70
            pages = cache.pages(2)
            assert len(pages) == 2 and pages[0] == cache.pages(0)[0] and pages[1] != cache.pages(0)[1]
            new, old = (ko.read(cache.pool[:, p].cpu().numpy(), 128, 64) for p in (pages[1], cache.pages(0)[1]))
            for name in ("kc", "vc", "ks", "vs", "km", "vm"):
                assert np.array_equal(new[name][..., :6, :], old[name][..., :6, :])
            kept = cache.pool[:, pages].clone()
        for _ in range(10):
            step()
        assert cache.rows(0) == cache.rows(1) == 80
        if forked:
            assert cache.rows(2) == 70 and torch.equal(cache.pool[:, pages], kept)
        runs.append((tok.clone(), [cache.pool[:, cache.pages(i)[:2]].clone() for i in range(2)]))
    assert torch.equal(runs[0][0], runs[1][0]) and all(torch.equal(a, b) for a, b in zip(*(r[1] for r in runs)))
