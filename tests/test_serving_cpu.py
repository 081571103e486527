"""What serving over fp16 caches can be checked for without a GPU: refusals of the C ABI, and the oracle against itself."""
import ctypes

import numpy as np
import pytest

import serving_oracle as so


@pytest.fixture(scope="module")
def L(built_lib):
    from sqamd import capi
    return capi.lib()


def pointers():
    buf = np.zeros(64, dtype=np.uint8)
    p = buf.ctypes.data - (buf.ctypes.data % 16) + 16
    return buf, ctypes.c_void_p(p), ctypes.c_void_p(p + 2)


def longs(*values):
    return (ctypes.c_long * len(values))(*values)


def test_prefix_attention_refuses_before_any_launch(L):
    from sqamd import capi
    keep, p, odd = pointers()
    ok = longs(512, 128, 12800, 128, 25600, 12800, 128, 512, 128)

    def call(q=p, kp=p, vp=p, kc=p, vc=p, lengths=p, starts=None, kn=p, vn=p, out=p, T=4, B=4, Hq=4, H=2, D=128, P=100, Lmax=100,
             strides=ok, ws=p, size=1 << 40):
        return L.sq_prefix_attention(q, kp, vp, kc, vc, lengths, starts, kn, vn, out, T, B, Hq, H, D, P, Lmax, strides, 1.0, ws, size, None)

    for kw in ({"D": 96}, {"Hq": 3}, {"H": 0}, {"T": 5}, {"T": -4}, {"B": -1}, {"P": -1}, {"Lmax": -1}, {"P": 1 << 30, "Lmax": (1 << 30) + 1},
               {"T": 1 << 27, "B": 1 << 27}, {"T": (1 << 23) + 4}, {"T": 1 << 22, "B": 1 << 22},
               {"strides": longs(*ok[:3], 1 << 23, *ok[4:])}, {"strides": longs(*ok[:6], -8, *ok[7:])}):
        assert call(**kw) == capi.SQ_ERR_BAD_SHAPE, kw
    for name in ("q", "kp", "vp", "kc", "vc", "lengths", "out", "vn", "strides"):
        assert call(**{name: None}) == capi.SQ_ERR_NULL_POINTER, name
    for name in ("q", "kp", "vp", "kc", "vc", "out", "kn", "vn", "lengths", "starts"):
        assert call(**{name: odd}) == capi.SQ_ERR_MISALIGNED, name
    assert call(strides=longs(*ok[:7], 4, 128)) == capi.SQ_ERR_MISALIGNED
    for kw in ({"ws": None}, {"ws": odd}, {"size": 16}):
        assert call(**kw) == capi.SQ_ERR_WORKSPACE, kw
    assert call(T=0, B=0) == capi.SQ_OK and call(T=0, q=None) == capi.SQ_OK
    assert L.sq_prefix_attention_workspace_bytes(0, 1, 1, 1, 64, 1, 1, 0) == 0


def test_evict_refuses_before_any_launch(L):
    from sqamd import capi
    keep, p, odd = pointers()
    ok = longs(512, 128, 512, 128, 25600, 12800, 128)

    def step(q=p, kn=p, vn=p, kc=p, vc=p, w=p, pos=p, seen=p, out=p, slot=p, B=4, Hq=4, H=2, D=64, R=100, first=4, last=10, strides=ok,
             ws=p, size=1 << 40):
        return L.sq_evict_attention(q, kn, vn, kc, vc, w, pos, seen, out, slot, B, Hq, H, D, R, first, last, strides, 1.0, ws, size, None)

    for kw in ({"D": 32}, {"Hq": 5}, {"R": 0}, {"first": -1}, {"last": 0}, {"first": 91}, {"B": -1}, {"B": 1 << 22},
               {"strides": longs(*ok[:6], 1 << 23)}):
        assert step(**kw) == capi.SQ_ERR_BAD_SHAPE, kw
    for name in ("q", "kn", "vn", "kc", "vc", "w", "pos", "seen", "out", "slot", "strides"):
        assert step(**{name: None}) == capi.SQ_ERR_NULL_POINTER, name
    for name in ("q", "kn", "vn", "kc", "vc", "w", "pos", "seen", "out", "slot"):
        assert step(**{name: odd}) == capi.SQ_ERR_MISALIGNED, name
    for kw in ({"ws": None}, {"size": 16}):
        assert step(**kw) == capi.SQ_ERR_WORKSPACE, kw
    assert step(B=0) == capi.SQ_OK

    def weights(q=p, k=p, lengths=None, w=p, B=2, Hq=4, H=2, D=64, S=50, window=0, strides=longs(*[1024] * 6), ws=p, size=1 << 40):
        return L.sq_attention_weights(q, k, lengths, w, B, Hq, H, D, S, window, strides, 1.0, ws, size, None)

    for kw in ({"D": 80}, {"Hq": 3}, {"window": -1}, {"S": -1}, {"S": 1 << 30, "B": 16}, {"S": (1 << 27) + 1},
               {"strides": longs(*[1024] * 5, 1 << 23)}):
        assert weights(**kw) == capi.SQ_ERR_BAD_SHAPE, kw
    for name in ("q", "k", "w", "strides"):
        assert weights(**{name: None}) == capi.SQ_ERR_NULL_POINTER, name
    assert weights(lengths=odd) == weights(q=odd) == capi.SQ_ERR_MISALIGNED
    assert weights(ws=None) == capi.SQ_ERR_WORKSPACE and weights(S=0) == weights(B=0) == capi.SQ_OK

    def keep_rows(k=p, v=p, w=p, lengths=None, kc=p, vc=p, cw=p, cp=p, rows=p, B=2, H=2, D=64, S=50, R=20, first=2, last=4,
                  strides=longs(*[64] * 3, 50, 25, *[64] * 3)):
        return L.sq_evict_keep(k, v, w, lengths, kc, vc, cw, cp, rows, B, H, D, S, R, first, last, strides, None)

    for kw in ({"D": 16}, {"R": 0}, {"first": 17}, {"last": -1}, {"B": 40000}, {"strides": longs(*[64] * 3, -1, 25, *[64] * 3)}):
        assert keep_rows(**kw) == capi.SQ_ERR_BAD_SHAPE, kw
    for name in ("k", "v", "w", "kc", "vc", "cw", "cp", "rows", "strides"):
        assert keep_rows(**{name: None}) == capi.SQ_ERR_NULL_POINTER, name
    for name in ("k", "v", "w", "lengths", "kc", "vc", "cw", "cp", "rows"):
        assert keep_rows(**{name: odd}) == capi.SQ_ERR_MISALIGNED, name
    assert keep_rows(B=0) == capi.SQ_OK


def test_logit_rules_refuse_before_any_launch(L):
    from sqamd import capi
    keep, p, odd = pointers()
    ok = longs(100, 100, 10, 1, 1, 1, 3, 3, 4)

    def call(x=p, y=p, elem=2, ids=p, lengths=None, gen=None, rep=p, pres=None, freq=None, bias_ids=p, bias=p, mask=None, token=p, M=2,
             V=100, nids=10, nb=3, strides=ok, ws=p, size=1 << 30):
        return L.sq_logit_rules(x, y, elem, ids, lengths, gen, rep, pres, freq, bias_ids, bias, mask, token, M, V, nids, nb, strides, ws,
                                size, None)

    for kw in ({"elem": 3}, {"V": 0}, {"M": -1}, {"M": 65536}, {"nids": -1}, {"nids": (1 << 30) + 1}, {"nb": 65536},
               {"strides": longs(100, 99, *ok[2:])},
               {"strides": longs(-1, *ok[1:])}):
        assert call(**kw) == capi.SQ_ERR_BAD_SHAPE, kw
    for name in ("x", "y", "ids", "bias", "bias_ids", "token", "strides"):
        assert call(**{name: None}) == capi.SQ_ERR_NULL_POINTER, name
    for name in ("ids", "lengths", "gen", "rep", "pres", "freq", "bias_ids", "bias", "mask", "token"):
        assert call(**{name: odd}) == capi.SQ_ERR_MISALIGNED, name
    assert call(x=odd, elem=4) == capi.SQ_ERR_MISALIGNED
    assert call(ws=None) == call(size=4) == call(ws=odd) == capi.SQ_ERR_WORKSPACE
    assert call(M=0) == capi.SQ_OK


def test_python_refuses_what_is_not_on_the_device():
    import torch
    from sqamd import evict, logits, prefix
    q, kp, kc = torch.zeros(2, 2, 64).half(), torch.zeros(2, 5, 64).half(), torch.zeros(2, 2, 8, 64).half()
    n = torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        prefix.attention(q, kp, kp, kc, kc, n, 1.0)
    with pytest.raises(ValueError):
        evict.attention(q, q, q, kc, kc.clone(), torch.zeros(2, 2, 8), torch.zeros(2, 2, 8, dtype=torch.int32), n, 1.0, 1, 2)
    with pytest.raises(ValueError):
        evict.attention_weights(kc, kc, 1.0)
    with pytest.raises(ValueError):
        evict.keep(kc, kc, torch.zeros(2, 2, 8), kc.clone(), kc.clone(), torch.zeros(2, 2, 8), torch.zeros(2, 2, 8, dtype=torch.int32), 1, 2)
    with pytest.raises(ValueError, match="memory"):
        evict.keep(kc, kc, torch.zeros(2, 2, 8), kc[:, :, :4], kc.clone(), torch.zeros(2, 2, 4), torch.zeros(2, 2, 4, dtype=torch.int32), 1, 2)
    w = torch.zeros(2, 2, 8)
    with pytest.raises(ValueError, match="memory"):
        evict.keep(kc, kc, w, kc.clone()[:, :, :4], kc.clone(), w[:, :, :4], torch.zeros(2, 2, 4, dtype=torch.int32), 1, 2)
    with pytest.raises(ValueError):
        logits.apply_rules(torch.zeros(2, 10))


def test_the_oracle_joins_what_it_cuts():
    # attention over prefix and own rows is attention over their concatenation, and the weights are its columns' sums
    rng = np.random.default_rng(0)
    b, h, heads, d, p, n = 2, 2, 4, 8, 5, 7
    q, kp, vp = rng.normal(size=(b * n, heads, d)), rng.normal(size=(h, p, d)), rng.normal(size=(h, p, d))
    kc, vc = rng.normal(size=(b, h, n, d)), rng.normal(size=(b, h, n, d))
    out, _, _, _ = so.prefix_attention(q, kp, vp, kc, vc, [n] * b, [n] * b, 0.3)
    for i in range(b):
        for g in range(heads):
            k, v = (np.concatenate([x[g // 2], y[i, g // 2]]) for x, y in ((kp, kc), (vp, vc)))
            s = q[i * n:(i + 1) * n, g] @ k.T * 0.3
            s[np.arange(p + n)[None] > p + np.arange(n)[:, None]] = -np.inf
            e = np.exp(s)
            assert np.allclose(out[i * n:(i + 1) * n, g], e / e.sum(1, keepdims=True) @ v)
    w = so.attention_weights(q.reshape(b, n, heads, d).transpose(0, 2, 1, 3), kc, [n, 3], 0.3)
    assert np.allclose(w.sum(-1), [[n * 2] * h, [3 * 2] * h]) and (w[1, :, 3:] == 0).all()


def test_the_oracle_on_rules_by_hand():
    x = np.array([[2.0, -2.0, 1.0, 0.5]])
    y = so.logit_rules(x, np.array([[1, 0, 0, 9]]), None, np.array([1]), np.array([2.0]), np.array([0.25]), np.array([0.5]),
                       np.array([[2, 2, -1]]), np.array([[5.0, 3.0, 9.0]]), np.array([[0b0111]], dtype=np.int32))
    # token 0 stands twice in the generated part, token 1 in the prompt; the last bias of token 2 counts; token 3 is masked
    assert y.tolist() == [[2.0 / 2 - 0.5 * 2 - 0.25, -4.0, 4.0, -np.inf]]
    assert so.best_token(y).tolist() == [2]
    assert so.keep_rows(np.array([5.0, 1.0, np.nan, 3.0, 3.0, 0.0]), 6, 3, 0, 1) == [0, 3, 5]


def test_the_oracle_on_rows_without_a_token():
    inf, nan = np.inf, np.nan
    y = np.array([[nan, -inf, -inf], [nan, nan, nan], [-inf, -inf, -inf], [nan, -inf, -3.0], [nan, 2.0, 2.0]])
    assert so.best_token(y).tolist() == [1, 0, 0, 2, 1] and so.best_token(y[:0]).shape == (0,)


def test_a_launch_that_failed_is_no_refusal(built_lib):
    # a refusal is looked into and may be called again; what may have run in part is not
    import torch  # noqa: F401
    import quant
    from sqamd import capi
    assert quant.taken(capi.SQ_OK, "call")
    assert not any(quant.taken(rc, "call") for rc in (capi.SQ_ERR_BAD_SHAPE, capi.SQ_ERR_MISALIGNED, capi.SQ_ERR_WORKSPACE))
    with pytest.raises(RuntimeError, match="call"):
        quant.taken(capi.SQ_ERR_LAUNCH, "call")
