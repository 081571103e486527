"""A key/value cache of a fixed number of rows a head that evicts by accumulated attention weight.

    attention          a decode step: the token's row is stored (where the cache is full, in the place of the row that has
                       gathered the least attention), the token attends, the rows' weights grow by what it gave them
    attention_weights  the weights that a prompt's queries give to its keys
    keep               of a prompt's rows those with the highest weights into such a cache
    EvictCache         a model's cache of this kind

A cache is k_cache, v_cache fp16 [B, kv_heads, rows, D] with, for each row, weight fp32 and position int32 [B, kv_heads, rows]
(of which token it is); the rows of a head are in no order.  All are device tensors, and the step takes the number of tokens
from the device, so that a captured HIP graph follows it.  Nothing here has a counterpart in the reference, whose cache grows.
"""
import torch

import quant
from . import capi, prefix
from .prefix import _alike, _check_ints, _check_written, _readable, _rows_like


def _check_state(name, x, dtype, shape, like):
    if x.dtype != dtype or tuple(x.shape) != shape or x.device != like.device or not x.is_contiguous():
        raise ValueError("%s must be a contiguous %s %s on the device of the rows, got %s %s"
                         % (name, dtype, list(shape), x.dtype, tuple(x.shape)))


def _check_cache(k_cache, v_cache, weight, position, b, h, d, like):
    for name, x in (("k_cache", k_cache), ("v_cache", v_cache)):
        _rows_like(x, like, 4, name)
        if x.shape[:2] != (b, h) or x.shape[3] != d or x.shape != k_cache.shape or x.shape[2] < 1:
            raise ValueError("%s %s for %d sequences, %d heads of %d" % (name, tuple(x.shape), b, h, d))
    if d not in (64, 128):
        raise ValueError("heads are of 64 or 128, not %d" % d)
    _check_written(k_cache, v_cache)
    r = k_cache.shape[2]
    _check_state("weight", weight, torch.float32, (b, h, r), like)
    _check_state("position", position, torch.int32, (b, h, r), like)
    return r


def attention(q, k_new, v_new, k_cache, v_cache, weight, position, seen, sm_scale, keep_first, keep_last, out=None):
    """The next token of each sequence: q fp16 [B, heads, D], its row k_new, v_new fp16 [B, kv_heads, D]; seen int32 [B] counts
    the sequence's tokens, this one among them.  The row goes to place seen - 1 while the cache has room, afterwards to that of
    the row of the lowest weight which is neither of the first keep_first nor of the last keep_last tokens (this one is one of
    those; keep_first + keep_last at most the cache's rows).  Returns (out fp16 [B, heads, D], slot int32 [B, kv_heads], the
    place taken); caches, weight and position are updated."""
    got = quant.evict_attention(q, k_new, v_new, k_cache, v_cache, weight, position, seen, sm_scale, keep_first, keep_last, out)
    if got is not None:
        return got if out is None else (out, got[1])
    _rows_like(q, q, 3, "q")
    _rows_like(k_new, q, 3, "k_new")
    _rows_like(v_new, q, 3, "v_new")
    b, heads, d = q.shape
    h = k_new.shape[1]
    if h < 1 or heads % h or k_new.shape != (b, h, d) or v_new.shape != k_new.shape:
        raise ValueError("rows %s and %s for queries %s" % (tuple(k_new.shape), tuple(v_new.shape), tuple(q.shape)))
    r = _check_cache(k_cache, v_cache, weight, position, b, h, d, q)
    _check_ints("seen", seen, (b,), q)
    _check_kept(keep_first, keep_last, r, 1)
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous()
                            or out.data_ptr() % 16):
        raise ValueError("out must be a contiguous fp16 %s at a multiple of 16 bytes on the device of q" % (tuple(q.shape),))
    k_new, v_new = _alike(k_new, v_new)
    got = quant.evict_attention(_readable(q, 3), k_new, v_new, k_cache, v_cache, weight, position, seen, sm_scale, keep_first,
                                keep_last, out)
    if got is None:
        raise ValueError("a step over caches %s: too large, or rows too far apart" % (tuple(k_cache.shape),))
    return got if out is None else (out, got[1])


def _check_kept(keep_first, keep_last, rows, least_last):
    if keep_first < 0 or keep_last < least_last or keep_first + keep_last > rows:
        raise ValueError("cannot keep the first %d and the last %d tokens in %d rows" % (keep_first, keep_last, rows))


def attention_weights(q, k, sm_scale, window=None, lengths=None):
    """fp32 [B, kv_heads, S]: the attention weight that the queries q fp16 [B, heads, S, D] of a prompt (the last `window` of
    each sequence, or all) give to each key of k fp16 [B, kv_heads, S, D], causally, summed over queries and query heads.
    lengths int32 [B] on the device: the sequences' rows, where they are fewer than S; 0 behind them."""
    if window is not None and window < 1:
        raise ValueError("a window of %d queries" % window)
    got = quant.evict_weights(q, k, sm_scale, window or 0, lengths)
    if got is not None:
        return got
    _rows_like(q, q, 4, "q")
    _rows_like(k, q, 4, "k")
    b, heads, s, d = q.shape
    h = k.shape[1]
    if h < 1 or heads % h or k.shape != (b, h, s, d) or d not in (64, 128):
        raise ValueError("keys %s for queries %s" % (tuple(k.shape), tuple(q.shape)))
    if lengths is not None:
        _check_ints("lengths", lengths, (b,), q)
    got = quant.evict_weights(_readable(q, 4), _readable(k, 4), sm_scale, window or 0, lengths)
    if got is None:
        raise ValueError("weights of %s queries: too large, or rows too far apart" % (tuple(q.shape),))
    return got


def keep(k, v, weight, k_cache, v_cache, cache_weight, cache_position, keep_first, keep_last, lengths=None):
    """Of the rows k, v fp16 [B, kv_heads, S, D] of a prompt (the first lengths[b], int32 on the device, or all S) those with
    the highest weight, fp32 [B, kv_heads, S], into the first rows of a cache, as many as it has; the first keep_first and the
    last keep_last are always among them.  They keep their order; their weights and places in the prompt become the cache's
    weights and positions.  Returns the places, int32 [B, kv_heads, rows], -1 behind the last.  The caches must not overlap k
    and v."""
    if any(_overlap(cache, x) for cache in (k_cache, v_cache) for x in (k, v)) or _overlap(cache_weight, weight):
        raise ValueError("rows cannot be kept in the memory that they are read from")
    got = quant.evict_keep(k, v, weight, k_cache, v_cache, cache_weight, cache_position, keep_first, keep_last, lengths)
    if got is not None:
        return got
    _rows_like(k, k, 4, "k")
    _rows_like(v, k, 4, "v")
    b, h, s, d = k.shape
    if v.shape != k.shape:
        raise ValueError("keys %s and values %s" % (tuple(k.shape), tuple(v.shape)))
    r = _check_cache(k_cache, v_cache, cache_weight, cache_position, b, h, d, k)
    if weight.dtype != torch.float32 or weight.shape != (b, h, s) or weight.device != k.device:
        raise ValueError("weight must be fp32 [%d, %d, %d] on the device of the rows" % (b, h, s))
    _check_kept(keep_first, keep_last, r, 0)
    if lengths is not None:
        _check_ints("lengths", lengths, (b,), k)
    k, v = _alike(k, v)
    got = quant.evict_keep(k, v, weight.contiguous(), k_cache, v_cache, cache_weight, cache_position, keep_first, keep_last, lengths)
    if got is None:
        raise ValueError("rows %s into caches %s: too large" % (tuple(k.shape), tuple(k_cache.shape)))
    return got


_MOST_ROWS, _MOST_HEADS = 1 << 25, 1 << 22  # (token, query head) and (sequence, query head) pairs of a call of prefix.attention


def _prompt_attention(q, k, v, sm_scale):
    """Causal attention of prompts q fp16 [B, heads, T, D] over k, v [B, kv_heads, T, D] -> [B, T, heads, D]: that of a batch whose
    own rows are all there is, in as many calls as its limits on tokens and heads ask for."""
    b, heads, t, d = q.shape
    h = k.shape[1]
    if h < 1 or heads % h:
        raise ValueError("%d query heads over %d key/value heads" % (heads, h))
    share = heads // h
    at_once = max(1, min(h, _MOST_ROWS // max(t * share, 1)))                                       # key/value heads
    most = max(1, min(_MOST_ROWS // max(t * share * at_once, 1), _MOST_HEADS // (share * at_once)))  # sequences
    none = torch.empty((h, 0, d), dtype=q.dtype, device=q.device)
    lengths = torch.full((b,), t, dtype=torch.int32, device=q.device)
    if b <= most and h <= at_once:
        return prefix.attention(q.transpose(1, 2).reshape(b * t, heads, d), none, none, k, v, lengths, sm_scale).view(b, t, heads, d)
    out = torch.empty((b, t, heads, d), dtype=q.dtype, device=q.device)
    for i in range(0, b, most):
        for j in range(0, h, at_once):
            mine = slice(j * share, (j + at_once) * share)
            rows = q[i:i + most, mine].transpose(1, 2)
            n, _, g, _ = rows.shape
            got = prefix.attention(rows.reshape(n * t, g, d), none[j:j + at_once], none[j:j + at_once], k[i:i + most, j:j + at_once],
                                   v[i:i + most, j:j + at_once], lengths[i:i + most], sm_scale)
            out[i:i + most, :, mine] = got.view(n, t, g, d)
    return out


def _extent(x):
    last = sum((n - 1) * st for n, st in zip(x.shape, x.stride())) if x.numel() else 0
    return x.data_ptr(), x.data_ptr() + (last + 1) * x.element_size() if x.numel() else x.data_ptr()


def _overlap(a, b):
    """Whether the extents of two tensors of one storage meet (rows of one may lie between those of the other: refused too)."""
    if a.untyped_storage().data_ptr() != b.untyped_storage().data_ptr():
        return False
    (a0, a1), (b0, b1) = _extent(a), _extent(b)
    return a0 < b1 and b0 < a1


class EvictCache:
    """A model's cache of `rows` rows a head in every layer: a prompt's rows of the highest weights stay, by all its queries or
    its last `window`, and later tokens take the places of those of the lowest.  The first keep_first and the last keep_last
    tokens are never given up.  `seen` counts the sequences' tokens on the device; `OPTDecoder` keeps it, or whoever drives the
    layers by hand.  It takes one prompt, at the beginning, and then single tokens, each once: a step changes the weights and may
    give up a row, so that running it again (a warm-up in front of a capture, say) leaves its token there twice.  A prompt at
    position 0 begins anew."""

    def __init__(self, layers, batch, kv_heads, head_dim, rows, keep_first=4, keep_last=None, window=None, device="cuda"):
        keep_last = max(1, rows // 4) if keep_last is None else keep_last
        if min(layers, batch, kv_heads, rows) < 1 or head_dim not in (64, 128) or (window is not None and window < 1):
            raise ValueError("a cache of %d layers, %d sequences, %d heads of %d, %d rows" % (layers, batch, kv_heads, head_dim, rows))
        _check_kept(keep_first, keep_last, rows, 1)
        self.layers, self.batch, self.rows = layers, batch, rows
        self.keep_first, self.keep_last, self.window = keep_first, keep_last, window
        shape = (layers, batch, kv_heads, rows)
        self.k = torch.zeros(shape + (head_dim,), dtype=torch.float16, device=device)
        self.v = torch.zeros_like(self.k)
        self.weight = torch.zeros(shape, dtype=torch.float32, device=device)
        self.position = torch.zeros(shape, dtype=torch.int32, device=device)
        self.seen = torch.zeros(batch, dtype=torch.int32, device=device)

    def set_position(self, batch, pos0, tokens):
        """The next `tokens` tokens of the first `batch` sequences are those of positions pos0 on: an int, or (one token) an
        int64 tensor of one element on the device.  Positions are not compared with those that came before: each step is for
        the position behind the last one's."""
        if batch > self.batch:
            raise ValueError("%d sequences in a cache for %d" % (batch, self.batch))
        if tokens != 1 and not (isinstance(pos0, int) and pos0 == 0):
            raise ValueError("a cache that evicts takes a prompt at the beginning, and then single tokens")
        if isinstance(pos0, int) and pos0 < 0:
            raise ValueError("position %d" % pos0)
        self.seen[:batch] = pos0 + tokens

    def attention(self, layer, q, k, v, sm_scale):
        """q, k, v fp16 [B, heads, T, D] of a prompt, or of the next token -> [B, T, heads, D]; their rows are stored."""
        b, h, t, d = q.shape
        cache = self.k[layer, :b], self.v[layer, :b], self.weight[layer, :b], self.position[layer, :b]
        if t == 1:
            q, k, v = (x[:, :, 0] for x in (q, k, v))
            return attention(q, k, v, *cache, self.seen[:b], sm_scale, self.keep_first, self.keep_last)[0].view(b, 1, h, d)
        if capi.lut_attention_strided_ok(q, k, v):
            out = capi.lut_attention_strided(q, k, v, None, sm_scale, True, rows_first=True)
        else:
            out = _prompt_attention(q, k, v, sm_scale)
        weight = attention_weights(q, k, sm_scale, self.window)
        keep(k, v, weight, *cache, self.keep_first, self.keep_last)
        return out
