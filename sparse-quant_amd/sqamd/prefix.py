"""Attention of a batch of sequences that share a long prefix: the prefix is held once and read once for all of them.

    attention     causal attention of the sequences' last tokens over the prefix and over rows of their own
    PrefixCache   a model's cache of both: the prefix's rows of every layer, and room for each sequence's own

Tokens of several sequences lie one behind the other, `starts` int32 [sequences + 1] says where each begins (None: equally many
each); `lengths` int32 [sequences] counts a sequence's own rows, those of the present call among them.  Both are device tensors
that the kernels read, so that a captured HIP graph follows them.

The reference attends to one sequence's cache at a time (sparse-attention/nvidia/playground/kernels/
block_sparse_attention_lut.py:272-300); nothing here has a counterpart there.
"""
import torch

import quant


def _rows_like(x, like, dims, what):
    if x.dtype != torch.float16 or x.dim() != dims or x.device != like.device or not x.is_cuda:
        raise ValueError("%s must be fp16 with %d dimensions on the device of the queries, got %s %s on %s"
                         % (what, dims, x.dtype, tuple(x.shape), x.device))


def _readable(x, dims):
    """x as the kernels can address it: rows of 16-byte chunks (a copy where it is not)."""
    ok = x.stride(-1) == 1 and x.data_ptr() % 16 == 0 and all(x.shape[d] < 2 or x.stride(d) % 8 == 0 for d in range(dims - 1))
    return x if ok else x.clone(memory_format=torch.contiguous_format)


def _alike(k, v):
    """Keys and values with the same strides (copies where they differ)."""
    k, v = _readable(k, k.dim()), _readable(v, v.dim())
    if any(k.shape[d] > 1 and k.stride(d) != v.stride(d) for d in range(k.dim())):
        k, v = (x.clone(memory_format=torch.contiguous_format) for x in (k, v))
    return k, v


def _check_written(k_cache, v_cache):
    """Caches that rows are stored in have to be addressable as they lie."""
    for x in (k_cache, v_cache):
        if x.stride(-1) != 1 or x.data_ptr() % 16 or any(x.shape[d] > 1 and (x.stride(d) % 8 or x.stride(d) < x.shape[-1])
                                                         for d in range(3)):
            raise ValueError("caches must hold rows of 16-byte chunks, no two in one place, got strides %s" % (x.stride(),))
    if any(k_cache.shape[d] > 1 and k_cache.stride(d) != v_cache.stride(d) for d in range(4)):
        raise ValueError("k_cache and v_cache must have the same strides")


def _check_ints(name, x, shape, like):
    if x.dtype != torch.int32 or tuple(x.shape) != shape or x.device != like.device or not x.is_contiguous():
        raise ValueError("%s must be a contiguous int32 %s on the device of the queries, got %s %s" % (name, list(shape), x.dtype,
                                                                                                   tuple(x.shape)))


def attention(q, k_prefix, v_prefix, k_cache, v_cache, lengths, sm_scale, starts=None, out=None, k_new=None, v_new=None):
    """Causal attention of q fp16 [T, heads, D], the last tokens of their sequences, over the rows k_prefix, v_prefix fp16
    [kv_heads, P, D] that all sequences begin with and the first lengths[b] rows of k_cache, v_cache fp16 [B, kv_heads, room,
    D]; query head h reads key/value head h // (heads // kv_heads); heads of 64 or 128.  k_new, v_new fp16 [T, kv_heads, D]:
    the tokens' own rows, which are stored in the caches first; without them they are there.  Any strides with adjacent
    elements of a row.  Returns fp16 [T, heads, D]; a token that sees no row gets 0, tokens behind the last sequence's are left
    as `out` had them.  Rows outside the caches' room are neither stored nor seen."""
    got = quant.prefix_attention(q, k_prefix, v_prefix, k_cache, v_cache, lengths, sm_scale, starts, out, k_new, v_new)
    if got is not None:
        return got if out is None else out
    # something has to be copied first, or is refused
    _rows_like(q, q, 3, "q")
    for name, x, dims in (("k_prefix", k_prefix, 3), ("v_prefix", v_prefix, 3), ("k_cache", k_cache, 4), ("v_cache", v_cache, 4)):
        _rows_like(x, q, dims, name)
    t, heads, d = q.shape
    b, h = k_cache.shape[:2]
    if d not in (64, 128) or h < 1 or heads % h:
        raise ValueError("%d query heads of %d over %d key/value heads; heads are of 64 or 128" % (heads, d, h))
    if k_prefix.shape != v_prefix.shape or k_prefix.shape[0] != h or k_prefix.shape[2] != d:
        raise ValueError("a prefix %s and %s for %d heads of %d" % (tuple(k_prefix.shape), tuple(v_prefix.shape), h, d))
    if k_cache.shape != v_cache.shape or k_cache.shape[3] != d:
        raise ValueError("caches %s and %s for heads of %d" % (tuple(k_cache.shape), tuple(v_cache.shape), d))
    _check_ints("lengths", lengths, (b,), q)
    if starts is not None:
        _check_ints("starts", starts, (b + 1,), q)
    elif t % b if b else t:
        raise ValueError("%d tokens cannot be dealt equally to %d sequences; pass starts" % (t, b))
    if (k_new is None) != (v_new is None):
        raise ValueError("k_new and v_new come together")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous()
                            or out.data_ptr() % 16):
        raise ValueError("out must be a contiguous fp16 %s at a multiple of 16 bytes on the device of q" % (tuple(q.shape),))
    if k_new is not None:
        _rows_like(k_new, q, 3, "k_new")
        _rows_like(v_new, q, 3, "v_new")
        if k_new.shape != (t, h, d) or v_new.shape != k_new.shape:
            raise ValueError("rows %s and %s for %d tokens, %d heads of %d" % (tuple(k_new.shape), tuple(v_new.shape), t, h, d))
        _check_written(k_cache, v_cache)
        k_new, v_new = _alike(k_new, v_new)
    else:
        k_cache, v_cache = _alike(k_cache, v_cache)
    k_prefix, v_prefix = _alike(k_prefix, v_prefix)
    got = quant.prefix_attention(_readable(q, 3), k_prefix, v_prefix, k_cache, v_cache, lengths, sm_scale, starts, out, k_new, v_new)
    if got is None:
        raise ValueError("prefix attention of %d tokens over %s behind %s: too large, or rows too far apart"
                         % (t, tuple(k_cache.shape), tuple(k_prefix.shape)))
    return got if out is None else out


class PrefixCache:
    """A model's keys and values behind a shared prefix: its rows in every layer, held once, and room for `max_rows` own rows of
    each of `batch` sequences.  k_prefix, v_prefix: a tensor [kv_heads, P, D] of each layer.  `lengths` counts the sequences' own
    rows on the device; `OPTDecoder` keeps it, or whoever drives the layers by hand (rows of the present call among them)."""

    def __init__(self, k_prefix, v_prefix, batch, max_rows):
        if not k_prefix or len(k_prefix) != len(v_prefix) or batch < 1 or max_rows < 1:
            raise ValueError("a cache of %d layers, %d sequences of %d rows" % (len(k_prefix), batch, max_rows))
        h, p, d = k_prefix[0].shape
        if any(x.shape != (h, p, d) for x in (*k_prefix, *v_prefix)):
            raise ValueError("the prefix has as many rows in every layer")
        self.k_prefix, self.v_prefix = list(k_prefix), list(v_prefix)
        self.layers, self.batch, self.max_rows, self.prefix_rows = len(k_prefix), batch, max_rows, p
        shape = (self.layers, batch, h, max_rows, d)
        self.k = torch.zeros(shape, dtype=torch.float16, device=k_prefix[0].device)
        self.v = torch.zeros_like(self.k)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=self.k.device)

    def set_position(self, batch, pos0, tokens):
        """The next `tokens` rows of the first `batch` sequences are those of positions pos0 on (the prefix's counted): an int, or
        an int64 tensor of one element on the device."""
        if batch > self.batch:
            raise ValueError("%d sequences in a cache for %d" % (batch, self.batch))
        if isinstance(pos0, int):
            if pos0 < self.prefix_rows or pos0 + tokens > self.prefix_rows + self.max_rows:
                raise ValueError("positions %d .. %d in a cache of %d rows behind a prefix of %d"
                                 % (pos0, pos0 + tokens - 1, self.max_rows, self.prefix_rows))
            self.lengths[:batch] = pos0 + tokens - self.prefix_rows
        else:
            self.lengths[:batch] = pos0 + (tokens - self.prefix_rows)

    def attention(self, layer, q, k, v, sm_scale):
        """q, k, v fp16 [B, heads, T, D] of the next tokens -> [B, T, heads, D]; their rows are stored."""
        b, h, t, d = q.shape
        q, k, v = (x.transpose(1, 2).reshape(b * t, x.shape[1], d) for x in (q, k, v))
        return attention(q, self.k_prefix[layer], self.v_prefix[layer], self.k[layer, :b], self.v[layer, :b], self.lengths[:b],
                         sm_scale, k_new=k, v_new=v).view(b, t, h, d)
