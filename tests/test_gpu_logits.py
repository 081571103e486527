"""Rules on logits on the device against the oracle: bit for bit against its steps in fp32, and against 64 bits."""
import numpy as np
import pytest
import torch

import serving_oracle as so

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def logits(built_lib):
    from sqamd import logits as m
    return m


def dev(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def make(rng, m, v, length, nb, dtype, mask_rows):
    d = {"ids": rng.integers(-2, v + 2, (m, length)) if length else None}
    if length:
        d["ids"][:, ::3] = d["ids"][:, :1]  # tokens that stand there often
        d["lengths"] = rng.integers(-1, length + 2, m)
        d["generated"] = rng.integers(-1, length + 2, m)
        for name, low, high in (("repetition", 0.8, 1.5), ("presence", -0.5, 0.5), ("frequency", -0.2, 0.3)):
            d[name] = rng.uniform(low, high, m).astype(np.float32)
    if nb:
        d["bias_ids"] = rng.integers(-2, min(v + 2, 3 * nb), (m, nb)).astype(np.int32)  # some named twice
        d["bias"] = rng.normal(0, 4, (m, nb)).astype(np.float32)
    if mask_rows:
        d["mask"] = rng.integers(-2 ** 31, 2 ** 31, (mask_rows, (v + 31) // 32)).astype(np.int32)
    return rng.normal(0, 3, (m, v)).astype(dtype), d


def call(logits, x, d, **kw):
    return logits.apply_rules(x, dev(d.get("ids")), dev(d.get("lengths")), dev(d.get("generated")), dev(d.get("repetition")),
                              dev(d.get("presence")), dev(d.get("frequency")), dev(d.get("bias_ids")), dev(d.get("bias")),
                              dev(d.get("mask")), **kw)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("m,v", [(1, 1), (2, 7), (3, 33), (1, 2048), (5, 2049), (2, 10007), (300, 9000), (1, 50272), (2, 65528),
                                 (2, 65529), (40, 70001)])
@pytest.mark.parametrize("length,nb,mask_rows", [(0, 0, 0), (1, 0, 0), (300, 5, 1), (0, 700, 0), (40, 0, 2)])
def test_rules(logits, dtype, m, v, length, nb, mask_rows):
    rng = np.random.default_rng(v + length)
    x, d = make(rng, m, v, length, nb, dtype, m if mask_rows == 2 else mask_rows)
    y, token = call(logits, dev(x), d)
    y = y.cpu().numpy()
    with np.errstate(over="ignore"):
        steps = so.logit_rules(x, dtype=np.float32, **d).astype(dtype)
        exact = so.logit_rules(x, **d)
    assert np.array_equal(y, steps)
    # four steps in fp32 and the rounding to the type, of values that grow by no more than their operands
    fin = np.isfinite(exact)
    size = 8 * 2.0 ** -24 * (np.abs(exact) + 80) + np.finfo(dtype).eps / 2 * np.abs(exact)
    assert (np.abs(y.astype(np.float64) - exact)[fin] <= size[fin]).all() and np.array_equal(np.isfinite(y), fin)
    assert np.array_equal(token.cpu().numpy(), so.best_token(steps))


@pytest.mark.parametrize("length,nb", [(16383, 512), (16384, 5), (300, 513), (70000, 6), (20, 33000)])
def test_long_texts_and_many_biases(logits, length, nb):
    # one token fills the text: its count passes what a half word, then what a word's half holds
    rng = np.random.default_rng(length)
    m, v = 2, 5000
    x, d = make(rng, m, v, length, nb, np.float32, 0)
    d["ids"][0], d["lengths"][:], d["generated"][:] = 77, length, 1
    d["frequency"][:] = 2.0 ** -10
    y, token = call(logits, dev(x), d)
    want = so.logit_rules(x, dtype=np.float32, **d)
    assert np.array_equal(y.cpu().numpy(), want) and np.array_equal(token.cpu().numpy(), so.best_token(want))


def test_ties_nan_and_rows_without_a_token(logits):
    x = np.full((6, 5000), -1.0, np.float16)
    x[0, [4321, 77, 2050]] = 2.0
    x[1, 3] = np.nan
    x[1, 4000] = 0.5
    x[2] = -np.inf
    x[3] = np.nan
    x[4, 4999] = np.inf
    x[5, :] = np.nan
    x[5, 4998] = -np.inf
    y, token = call(logits, dev(x), {})
    assert np.array_equal(y.cpu().numpy(), x, equal_nan=True)
    assert token.tolist() == [77, 4000, 0, 0, 4999, 4998]
    none = torch.zeros((6, 157), dtype=torch.int32, device=DEV)
    y, token = logits.apply_rules(dev(x), mask=none)
    assert (y == -torch.inf).all() and token.tolist() == [0] * 6


def test_each_penalty_alone_and_strides(logits):
    rng = np.random.default_rng(3)
    m, v, length = 4, 3001, 50
    x, d = make(rng, m, v, length, 6, np.float16, 0)
    history = dev(d["ids"].T.copy())  # [place, row], as a decoder keeps it
    wide = torch.zeros((m, v + 11), dtype=torch.float16, device=DEV)
    wide[:, 5:5 + v] = dev(x)
    for name in ("repetition", "presence", "frequency"):
        e = {"ids": d["ids"], name: d[name]}
        want = so.logit_rules(x, dtype=np.float32, **e).astype(np.float16)
        y, token = logits.apply_rules(wide[:, 5:5 + v], history.t(), **{name: dev(d[name])})
        assert np.array_equal(y.cpu().numpy(), want) and np.array_equal(token.cpu().numpy(), so.best_token(want))
    # one length for all rows, results in place and into given tensors
    steps = torch.tensor([20], device=DEV)
    e = dict(d, lengths=np.full(m, 20), generated=None)
    want = so.logit_rules(x, dtype=np.float32, **{k: g for k, g in e.items() if g is not None}).astype(np.float16)
    token = torch.zeros(m, dtype=torch.int64, device=DEV)
    view = wide[:, 5:5 + v]
    got = logits.apply_rules(view, history.t(), steps.expand(m), None, dev(d["repetition"]), dev(d["presence"]), dev(d["frequency"]),
                             dev(d["bias_ids"]), dev(d["bias"]), out=view, token=token)
    assert got[0] is view and got[1] is token and np.array_equal(view.cpu().numpy(), want)
    assert (wide[:, :5] == 0).all() and (wide[:, 5 + v:] == 0).all()
    # rows that lie across, and a bias that does
    across = dev(x.T.copy()).t()
    y, _ = logits.apply_rules(across, bias_ids=dev(d["bias_ids"].T.copy()).t(), bias=dev(d["bias"].T.copy()).t())
    assert np.array_equal(y.cpu().numpy(), so.logit_rules(x, bias_ids=d["bias_ids"], bias=d["bias"], dtype=np.float32).astype(np.float16))


def test_captured(logits):
    rng = np.random.default_rng(4)
    m, v = 8, 50272
    x, d = make(rng, m, v, 60, 4, np.float16, m)
    given = {k: dev(a) for k, a in d.items()}
    rows = dev(x)
    lengths = torch.full((m,), 10, device=DEV)

    def step():
        return logits.apply_rules(rows, given["ids"], lengths, None, given["repetition"], given["presence"], given["frequency"],
                                  given["bias_ids"], given["bias"], given["mask"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y, token = step()
    for i in range(4):
        rows.copy_(dev(rng.normal(0, 3, (m, v)).astype(np.float16)))
        lengths += 7
        want = [a.clone() for a in step()]
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(y, want[0]) and torch.equal(token, want[1]), i


def test_refusals(logits):
    x = torch.zeros((2, 100), dtype=torch.float16, device=DEV)
    ids, one = torch.zeros((2, 5), dtype=torch.int64, device=DEV), torch.ones(2, device=DEV)
    mask, b = torch.zeros((2, 4), dtype=torch.int32, device=DEV), torch.zeros((2, 3), dtype=torch.int32, device=DEV)
    bad = [((x.double(),), {}), ((x.cpu(),), {}), ((x[0],), {}), ((x, ids.int()), {}), ((x, ids[:1]), {}), ((x, ids, one), {}),
           ((x,), {"repetition": one}), ((x, ids), {"repetition": one.half()}), ((x, ids), {"presence": one[:1]}),
           ((x,), {"bias_ids": b}), ((x,), {"bias_ids": b, "bias": b}), ((x,), {"mask": mask[:, :3]}), ((x,), {"mask": mask.long()}),
           ((x,), {"out": x.float()}), ((x,), {"out": x[:1].expand(2, -1)}), ((x,), {"token": one}), ((x[:, :0],), {}),
           ((x,), {"mask": torch.zeros((3, 4), dtype=torch.int32, device=DEV)}),
           ((x.view(-1)[:198].view(2, 99),), {"out": x.view(-1)[1:199].view(2, 99)}), ((x[:, :50],), {"out": x.view(-1)[:100].view(2, 50)})]
    for args, kw in bad:
        with pytest.raises(ValueError):
            logits.apply_rules(*args, **kw)
    y, token = logits.apply_rules(x[:0])
    assert y.shape == (0, 100) and token.shape == (0,)


@pytest.mark.parametrize("v,allowed", [(40, [3, 17]), (9000, [0, 5, 2100, 8999])])
def test_rows_of_which_nothing_may_be_chosen(logits, v, allowed):
    # all that the mask leaves is NaN: the lowest of the masked ones; with one number among them, that
    x = np.full((3, v), 1.0, np.float32)
    x[:2, allowed] = np.nan
    x[1, allowed[1]] = -7.0
    x[2] = np.nan
    bits = np.zeros(((v + 31) // 32) * 32, np.uint64)
    bits[allowed] = 1
    mask = (bits.reshape(-1, 32) << np.arange(32, dtype=np.uint64)).sum(1).astype(np.uint32).view(np.int32)[None]
    y, token = logits.apply_rules(dev(x), mask=dev(mask))
    want = so.logit_rules(x, mask=mask, dtype=np.float32)
    assert np.array_equal(y.cpu().numpy(), want, equal_nan=True)
    lowest = next(i for i in range(v) if i not in allowed)
    assert token.tolist() == so.best_token(want).tolist() == [lowest, allowed[1], lowest]
