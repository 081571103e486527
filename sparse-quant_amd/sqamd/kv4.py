"""A key/value cache held in 4 bits, in pages: the operators on it and its bookkeeping.

The cache is a pool of pages of 64 rows, uint8 [pages, kv_heads, record] (`new_pool`); the record's layout is written down
with sq_kv4_append in include/sq_w4a16.h.  A sequence's pages stand in a row of `pages` int32 [sequences, width], its rows
are counted by `lengths` int32 [sequences], the rows of the present call among them; tokens of several sequences lie one
behind the other, `starts` int32 [sequences + 1] says where each begins (None: equally many each).  All are device tensors,
read by the kernels, so that a captured HIP graph follows them.

    append        quantise the key and value rows of new tokens into their pages
    attention     causal attention of the tokens over their sequence's rows, or over the rows of selected pages
    select_pages  for one token of each sequence, the pages whose keys can score highest
    copy_pages    copy pages in every layer

`KV4Cache` keeps pools of all layers, tables and free pages: sequences that grow, fork (pages are shared until one of them
is written to), shrink and end, and a pool made compact.

The reference keeps its cache in fp16 tensors that grow by torch.cat (sparse-attention/nvidia/playground/kernels/
block_sparse_attention_lut.py:272-300 reads them); nothing here has a counterpart there.
"""
import ctypes
import heapq

import torch

import quant
from . import capi
from .capi import _check, _ptr, _stream

PAGE = 64
GROUPS = (32, 64, 128)


def record_bytes(head_dim, group_size):
    """Bytes of one page of one key/value head."""
    if head_dim not in (64, 128) or group_size not in GROUPS or group_size > head_dim:
        raise ValueError("a 4-bit cache has heads of 64 or 128 and groups of 32, 64 or 128 within a head, not %d and %d"
                         % (head_dim, group_size))
    return 68 * head_dim + 512 * (head_dim // group_size)


def new_pool(num_pages, kv_heads, head_dim, group_size=64, layers=None, device="cuda"):
    """uint8 [num_pages, kv_heads, record], or [layers, ...]; of any content: what no row was stored to is never seen."""
    shape = (num_pages, kv_heads, record_bytes(head_dim, group_size))
    return torch.empty(shape if layers is None else (layers,) + shape, dtype=torch.uint8, device=device)


def _group_size(pool, head_dim):
    for g in GROUPS:
        if head_dim in (64, 128) and g <= head_dim and record_bytes(head_dim, g) == pool.shape[-1]:
            return g
    raise ValueError("a pool with records of %d bytes holds no heads of %d" % (pool.shape[-1], head_dim))


def _check_cache(x, pool, pages, lengths, starts):
    """The cache's tensors against rows or queries x [T, heads, D]; returns (T, B, group size)."""
    if x.dim() != 3 or x.dtype != torch.float16 or not x.is_cuda:
        raise ValueError("expected fp16 [tokens, heads, dim] on the device, got %s %s" % (x.dtype, tuple(x.shape)))
    if pool.dim() != 3 or pool.dtype != torch.uint8 or not pool.is_contiguous() or pool.shape[0] < 1:
        raise ValueError("the pool must be a contiguous uint8 [pages, kv_heads, record] of at least one page")
    for name, t, dims in (("pages", pages, 2), ("lengths", lengths, 1), ("starts", starts, 1)):
        if t is None:
            continue
        if t.dtype != torch.int32 or t.dim() != dims or (t.numel() and t.stride(-1) != 1):
            raise ValueError("%s must be int32 with %d dimensions and adjacent elements" % (name, dims))
    for t in (pool, pages, lengths, starts):
        if t is not None and t.device != x.device:
            raise ValueError("all tensors must be on %s" % x.device)
    b = lengths.shape[0]
    if pages.shape[0] != b or (starts is not None and starts.shape[0] != b + 1):
        raise ValueError("%d lengths, but pages %s%s" % (b, tuple(pages.shape), "" if starts is None else
                                                         " and starts %s" % (tuple(starts.shape),)))
    t = x.shape[0]
    if starts is None and (t % b if b else t):
        raise ValueError("%d tokens cannot be dealt equally to %d sequences; pass starts" % (t, b))
    return t, b, _group_size(pool, x.shape[-1])


def _readable(x):
    """x [T, heads, D] as the kernels can address it: rows of 16-byte chunks (a copy where it is not)."""
    ok = x.stride(2) == 1 and x.data_ptr() % 16 == 0 and all(s % 8 == 0 for s in x.stride()[:2])
    return x if ok else x.clone(memory_format=torch.contiguous_format)


def _table(pages):
    """pages with rows that lie apart (a copy where they do not: an expanded row), and their distance."""
    if pages.shape[0] > 1 and pages.stride(0) < pages.shape[1]:
        pages = pages.contiguous()
    return pages, max(pages.stride(0), pages.shape[1]) if pages.shape[0] > 1 else pages.shape[1]


def append(k, v, pool, pages, lengths, starts=None, values=False):
    """Quantise the rows k, v fp16 [T, kv_heads, D] (any token and head strides) of new tokens into their pages; they are
    the last rows of their sequences (two sequences that get rows must not share the page these go to).  With `values` returns
    (k_hat, v_hat) fp16 [T, kv_heads, D], what the cache holds of them, rounded (of no defined content where a token has no
    page); otherwise None."""
    got = quant.kv4_append(k, v, pool, pages, lengths, starts, values)
    if got is not None:
        return tuple(got) if values else None
    # something is empty, has to be copied first, or is refused
    t, b, g = _check_cache(k, pool, pages, lengths, starts)
    if v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
        raise ValueError("k and v must be alike, got %s %s and %s %s" % (k.dtype, tuple(k.shape), v.dtype, tuple(v.shape)))
    h, d = k.shape[1:]
    if pool.shape[1] != h:
        raise ValueError("rows of %d heads for a pool of %d" % (h, pool.shape[1]))
    k, v = _readable(k), _readable(v)
    hats = torch.empty((2, t, h, d), dtype=k.dtype, device=k.device).unbind(0) if values else (None, None)
    strides = (ctypes.c_long * 4)(k.stride(0), k.stride(1), v.stride(0), v.stride(1))
    pages, pitch = _table(pages)
    with torch.cuda.device(k.device):
        _check(capi.lib().sq_kv4_append(_ptr(k), _ptr(v), _ptr(hats[0]), _ptr(hats[1]), _ptr(pool), _ptr(pages), _ptr(lengths),
                                        _ptr(starts), t, b, h, d, g, pool.shape[0], pages.shape[1], pitch,
                                        strides, _stream()), "sq_kv4_append")
    return hats if values else None


def attention(q, pool, pages, lengths, sm_scale, starts=None, selected=None, out=None, k_new=None, v_new=None):
    """Causal attention of q fp16 [T, heads, D], the last tokens of their sequences (their own rows are in the cache), over
    the cached rows; query head h reads key/value head h // (heads // kv_heads).  selected int32 [sequences, kv_heads,
    count] (one token per sequence): over the rows of these pages only, as select_pages gives them.  Returns fp16
    [T, heads, D]; a token that sees no row gets 0, tokens behind the last sequence's are left as `out` had them.
    k_new, v_new fp16 [T, kv_heads, D]: the tokens' rows are not in the cache yet and are appended first (for one token per
    sequence in the same launch); not with selected pages."""
    got = quant.kv4_attention(q, pool, pages, lengths, sm_scale, starts, selected, out, k_new, v_new)
    if got is not None:
        return got if out is None else out
    t, b, g = _check_cache(q, pool, pages, lengths, starts)
    hq, d = q.shape[1:]
    h = pool.shape[1]
    if hq % h:
        raise ValueError("%d query heads over %d key/value heads" % (hq, h))
    count = 0
    if selected is not None:
        if starts is not None or t != b:
            raise ValueError("selected pages are for one token per sequence")
        if selected.dtype != torch.int32 or not selected.is_contiguous() or selected.device != q.device \
                or selected.dim() != 3 or tuple(selected.shape[:2]) != (b, h) or selected.shape[2] < 1:
            raise ValueError("selected must be a contiguous int32 [sequences, kv_heads, count] on the device of q")
        count = selected.shape[2]
    if (k_new is None) != (v_new is None):
        raise ValueError("k_new and v_new come together")
    if k_new is not None:
        if selected is not None:
            raise ValueError("rows are appended before pages are selected")
        if k_new.shape != (t, h, d) or k_new.device != q.device:
            raise ValueError("rows of shape %s for %d tokens, %d heads of %d on the device of q"
                             % (tuple(k_new.shape), t, h, d))
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous()
                            or out.data_ptr() % 16):
        raise ValueError("out must be a contiguous fp16 %s at a multiple of 16 bytes on the device of q" % (tuple(q.shape),))
    if k_new is not None:
        append(k_new, v_new, pool, pages, lengths, starts)
    q = _readable(q)
    if out is None:
        out = torch.empty((t, hq, d), dtype=q.dtype, device=q.device)
    pages, pitch = _table(pages)
    need = capi.lib().sq_kv4_attention_workspace_bytes(t, b, hq, h, d, pages.shape[1], count)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    with torch.cuda.device(q.device):
        _check(capi.lib().sq_kv4_attention(_ptr(q), _ptr(out), _ptr(pool), _ptr(pages), _ptr(lengths), _ptr(starts),
                                           _ptr(selected), t, b, hq, h, d, g, pool.shape[0], pages.shape[1], pitch, count,
                                           q.stride(0), q.stride(1), float(sm_scale), None, None, None, _ptr(ws), need,
                                           _stream()), "sq_kv4_attention")
    return out


def select_pages(q, pool, pages, lengths, count, keep_first=1, keep_last=1):
    """int32 [sequences, kv_heads, count]: for the next token of each sequence, q fp16 [sequences, heads, D], the places of
    the `count` pages that can hold the highest scores, ascending, -1 behind the last where there are fewer; the first
    keep_first and the last keep_last are always among them.  With attention over 64 pages it takes less time than attention over
    all rows where the sequences have more than some 100000 rows together (8 key/value heads), and more below."""
    got = quant.kv4_select(q, pool, pages, lengths, count, keep_first, keep_last)
    if got is not None:
        return got
    t, b, g = _check_cache(q, pool, pages, lengths, None)
    hq, d = q.shape[1:]
    h = pool.shape[1]
    if t != b:
        raise ValueError("pages are selected for one token per sequence, got %d tokens for %d" % (t, b))
    if hq % h:
        raise ValueError("%d query heads over %d key/value heads" % (hq, h))
    if count < 1 or keep_first < 0 or keep_last < 0 or keep_first + keep_last > count:
        raise ValueError("cannot keep the first %d and the last %d among %d pages" % (keep_first, keep_last, count))
    q = _readable(q)
    pages, pitch = _table(pages)
    selected = torch.empty((b, h, count), dtype=torch.int32, device=q.device)
    width = pages.shape[1]
    need = capi.lib().sq_kv4_select_workspace_bytes(b, h, width) if width > count else 0
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    with torch.cuda.device(q.device):
        _check(capi.lib().sq_kv4_select(_ptr(q), _ptr(selected), _ptr(pool), _ptr(pages), _ptr(lengths), b, hq, h, d, g,
                                        pool.shape[0], width, pitch, int(count), int(keep_first), int(keep_last),
                                        q.stride(0), q.stride(1), _ptr(ws), need, _stream()),
               "sq_kv4_select")
    return selected


def copy_pages(pool, src, dst):
    """Copy page src[i] to page dst[i], int32 on the device, in a pool [pages, ...] or in every layer of [layers, pages,
    kv_heads, record].  No page may be a destination twice, or a destination and another pair's source."""
    if quant.kv4_copy_pages(pool, src, dst):
        return
    if pool.dim() not in (3, 4) or pool.dtype != torch.uint8 or not pool.is_contiguous() or not pool.is_cuda:
        raise ValueError("the pool must be a contiguous uint8 [pages, kv_heads, record] or [layers, ...] on the device")
    if src.shape != dst.shape or src.dim() != 1 or any(i.dtype != torch.int32 or i.device != pool.device
                                                       or not i.is_contiguous() for i in (src, dst)):
        raise ValueError("src and dst must be int32 vectors of one length on the device of the pool")
    layers, (n, h, rec) = (1, pool.shape) if pool.dim() == 3 else (pool.shape[0], pool.shape[1:])
    with torch.cuda.device(pool.device):
        _check(capi.lib().sq_kv4_copy_pages(_ptr(pool), _ptr(src), _ptr(dst), src.numel(), n, layers, h * rec, n * h * rec,
                                            _stream()), "sq_kv4_copy_pages")


class KV4Cache:
    """The 4-bit cache of a model: pools of all layers, and which pages belong to which sequence.

    Sequences are numbered 0 .. max_seqs - 1 (`add`, `fork`, `free`).  Rows are given room with `extend` (which also counts
    them) or ahead of time with `reserve`; `append`, `attention` and `select_pages` then work on one layer for a list of
    sequences, or for all of the first n (`seqs` an int).  Pages may be shared between sequences (`fork`): a page is copied
    before a sequence that shares it gets rows in it, by `reserve` (and so by `extend`), which therefore follows a fork.
    `lengths` and `table` are the device's view of it and change in place.  The table has as many columns as `max_rows` takes,
    and the operators choose by them: where sequences stay below 1024 rows, max_rows up to 1024 (or the table's first 16 columns)
    make the attention of a step 2.5 us faster.

    With rows reserved the device may count `lengths` up itself, as a captured graph does and every decode step that takes
    its position from the device.  `counted_on_device` says so, once, before the first such step.  From then on the host asks
    the device for the rows of these sequences where it needs them (`rows`, `fork`, `truncate`, `reserve`, `extend`), which
    waits for the current stream; and where `fork`, `truncate` or `set_lengths` leaves them at the end of a shared page it
    gives them their own at once, since a replayed step cannot be refused.  Rows counted beyond the reserved pages, or of a
    sequence that has ended, are left out."""

    def __init__(self, layers, num_pages, kv_heads, head_dim, group_size=64, max_seqs=8, max_rows=2048, device="cuda"):
        if min(layers, num_pages, kv_heads, max_seqs, max_rows) < 1:
            raise ValueError("a cache of %d layers, %d pages, %d heads, %d sequences of %d rows"
                             % (layers, num_pages, kv_heads, max_seqs, max_rows))
        self.pool = new_pool(num_pages, kv_heads, head_dim, group_size, layers, device)
        self.layers, self.num_pages, self.max_seqs, self.max_rows = layers, num_pages, max_seqs, max_rows
        self.kv_heads, self.head_dim, self.group_size = kv_heads, head_dim, group_size
        self.width = (max_rows + PAGE - 1) // PAGE
        # Places without a page hold -1, which the kernels know as no page: a sequence whose length is counted on the device
        # past its pages, or after it has ended, neither stores nor sees rows there.
        self.table = torch.full((max_seqs, self.width), -1, dtype=torch.int32, device=self.pool.device)
        self.lengths = torch.zeros(max_seqs, dtype=torch.int32, device=self.pool.device)
        self._pages = [None] * max_seqs  # of a sequence, in their order; None: no such sequence
        self._rows = [0] * max_seqs
        self._device_counts = set()  # sequences (their numbers, whoever has them) whose lengths the device counts as well
        self._uses = [0] * num_pages
        self._free = list(range(num_pages))  # a heap: the lowest page first

    # ------------------------------------------------------------------------------------------------ bookkeeping

    def _known(self, seq):
        if not 0 <= seq < self.max_seqs or self._pages[seq] is None:
            raise ValueError("no sequence %r" % (seq,))
        return self._pages[seq]

    def counted_on_device(self, seqs):
        """Something on the device counts `lengths` of these sequences from now on (an int n: of the first n, whether they
        exist or not).  Refused where the next rows would go to a page that another sequence shares."""
        seqs = [seq for seq in (range(seqs) if isinstance(seqs, int) else map(int, seqs)) if seq not in self._device_counts]
        for seq in seqs:
            if not 0 <= seq < self.max_seqs:
                raise ValueError("no sequence %r" % (seq,))
            if self._pages[seq] and any(self._uses[page] > 1 for page in self._pages[seq][self._rows[seq] // PAGE:]):
                raise ValueError("rows of sequence %d would go to a page that another shares; reserve gives it its own" % seq)
        self._device_counts.update(seqs)

    def _ask_device(self, seqs, beyond=False):
        """Bring the host's row counts after the device's; more rows than pages hold are an error unless `beyond`."""
        asked = [seq for seq in seqs if seq in self._device_counts and self._pages[seq] is not None]
        if not asked:
            return
        lengths = self.lengths.tolist()
        for seq in asked:
            room = len(self._pages[seq]) * PAGE
            if lengths[seq] > room and not beyond:
                raise RuntimeError("the device counted sequence %d to %d rows, of which its pages hold %d: truncate or "
                                   "set_lengths says how many it keeps" % (seq, lengths[seq], room))
            self._rows[seq] = max(0, min(lengths[seq], room))

    def free_pages(self):
        return len(self._free)

    def rows(self, seq):
        self._known(seq)
        self._ask_device([seq])
        return self._rows[seq]

    def pages(self, seq):
        """The pages of a sequence, in their order."""
        return list(self._known(seq))

    def add(self):
        """A new, empty sequence; returns its number (the lowest that is free)."""
        for seq, pages in enumerate(self._pages):
            if pages is None:
                self._pages[seq] = []
                self._rows[seq] = 0
                self.lengths[seq:seq + 1].zero_()
                return seq
        raise RuntimeError("all %d sequences are in use" % self.max_seqs)

    def _release(self, page):
        self._uses[page] -= 1
        if self._uses[page] == 0:
            heapq.heappush(self._free, page)

    def free(self, seq):
        """End a sequence; pages that no other shares become free."""
        for page in self._known(seq):
            self._release(page)
        self._pages[seq] = None
        self._rows[seq] = 0
        self.lengths[seq:seq + 1].zero_()
        self.table[seq].fill_(-1)

    def fork(self, seq):
        """A new sequence with the rows of `seq`, on the same pages; returns its number."""
        pages = self._known(seq)
        rows = self.rows(seq)
        new = self.add()
        used = pages[:(rows + PAGE - 1) // PAGE]
        for page in used:
            self._uses[page] += 1
        self._pages[new] = list(used)
        self._write([new])
        self._count([new], [rows])
        if self._device_counts & {seq, new}:
            try:
                self._give({new: (rows, len(used) * PAGE)})
            except RuntimeError:
                self.free(new)
                raise
        return new

    def truncate(self, seq, rows):
        """Keep the first `rows` rows of a sequence and release the pages behind them.  (The bounds of the page that becomes
        its last still cover the rows that went, until its row 0 is stored again.)"""
        pages = self._known(seq)
        self._ask_device([seq], beyond=True)
        if not 0 <= rows <= self._rows[seq]:
            raise ValueError("cannot keep %d of %d rows" % (rows, self._rows[seq]))
        keep = (rows + PAGE - 1) // PAGE
        own = seq in self._device_counts and rows % PAGE and self._uses[pages[keep - 1]] > 1
        if own and not self._free and all(self._uses[page] > 1 for page in pages[keep:]):
            raise RuntimeError("1 page wanted, 0 free of %d" % self.num_pages)
        for page in pages[keep:]:
            self._release(page)
        del pages[keep:]
        self.table[seq, keep:].fill_(-1)
        if own:
            self._give({seq: (rows, keep * PAGE)})
        self._count([seq], [rows])

    def reserve(self, seqs, rows):
        """Pages for the first rows[i] rows of seqs[i], of their own from the row behind the last one on."""
        seqs, rows = self._per_sequence(seqs, rows)
        for seq, n in zip(seqs, rows):
            self._known(seq)
            if n > self.max_rows:
                raise ValueError("%d rows in a cache of %d" % (n, self.max_rows))
        self._ask_device(seqs)
        self._give({seq: (self._rows[seq], n) for seq, n in zip(seqs, rows)})

    def _give(self, wanted):
        """{sequence: (held, rows)}: pages of its own for the rows from `held`, the last it has, to `rows`."""
        fresh = {}   # sequence -> places that get a new page
        for seq, (held, n) in wanted.items():
            if n > held:
                pages = self._pages[seq]
                fresh[seq] = [j for j in range(held // PAGE, (n + PAGE - 1) // PAGE)
                              if j >= len(pages) or self._uses[pages[j]] > 1]
        # a page shared by sequences of this very call is copied for all but the last of them
        want = []
        shared = dict()
        for seq, places in fresh.items():
            pages = self._pages[seq]
            for j in places:
                if j < len(pages):
                    left = shared.get(pages[j], self._uses[pages[j]])
                    if left == 1:
                        continue
                    shared[pages[j]] = left - 1
                want.append((seq, j))
        if len(want) > len(self._free):
            raise RuntimeError("%d pages wanted, %d free of %d" % (len(want), len(self._free), self.num_pages))
        src, dst = [], []
        for seq, j in want:
            pages = self._pages[seq]
            page = heapq.heappop(self._free)
            self._uses[page] = 1
            if j < len(pages):
                if j * PAGE < wanted[seq][0]:  # it holds rows
                    src.append(pages[j])
                    dst.append(page)
                self._release(pages[j])
                pages[j] = page
            else:
                pages.append(page)
        if src:
            copy_pages(self.pool, *self._vectors(src, dst))
        if want:
            self._write(sorted({seq for seq, _ in want}))

    def extend(self, seqs, rows):
        """Room for rows[i] (or `rows`) more rows of seqs[i], and count them."""
        seqs, more = self._per_sequence(seqs, rows)
        for seq in seqs:
            self._known(seq)
        self._ask_device(seqs)
        total = [self._rows[seq] + n for seq, n in zip(seqs, more)]
        if any(n < 0 for n in more):
            raise ValueError("a sequence shrinks by truncate")
        self.reserve(seqs, total)
        self.set_lengths(seqs, total)

    def set_lengths(self, seqs, rows, stored=0):
        """Count rows that have pages already, new ones pages that no other sequence shares.  stored: the last so many rows of
        each will be stored, again where they are not new; their pages must not be shared either."""
        seqs, rows = self._per_sequence(seqs, rows)
        for seq, n in zip(seqs, rows):
            pages = self._known(seq)
            if not 0 <= n <= len(pages) * PAGE:
                raise ValueError("%d rows on %d pages" % (n, len(pages)))
            if n > self._rows[seq] and any(self._uses[p] > 1 for p in pages[self._rows[seq] // PAGE:(n + PAGE - 1) // PAGE]):
                raise ValueError("rows of sequence %d would go to a page that another shares; reserve gives it its own" % seq)
            if stored and any(self._uses[p] > 1 for p in pages[max(0, n - stored) // PAGE:(n + PAGE - 1) // PAGE]):
                raise ValueError("rows of sequence %d would be stored again on a page that another shares; truncate and reserve "
                                 "give it its own" % seq)
        self._give({seq: (n, len(self._pages[seq]) * PAGE) for seq, n in zip(seqs, rows) if seq in self._device_counts})
        self._count(seqs, rows)

    def _count(self, seqs, rows):
        for seq, n in zip(seqs, rows):
            self._rows[seq] = n
        at, n = self._vectors(seqs, rows)
        self.lengths[at.long()] = n

    def compact(self):
        """Move the pages in use to the front of the pool; returns how many they are.  Behind it the pool's tail is free."""
        used = sum(1 for n in self._uses if n)
        holes = [p for p in range(used) if not self._uses[p]]
        tail = [p for p in range(used, self.num_pages) if self._uses[p]]
        if not tail:
            return used
        to = dict(zip(tail, holes))
        copy_pages(self.pool, *self._vectors(list(to), list(to.values())))
        for a, b in to.items():
            self._uses[b], self._uses[a] = self._uses[a], 0
        touched = []
        for seq, pages in enumerate(self._pages):
            if pages and any(p in to for p in pages):
                self._pages[seq] = [to.get(p, p) for p in pages]
                touched.append(seq)
        self._free = list(range(used, self.num_pages))
        self._write(touched)
        return used

    @staticmethod
    def _per_sequence(seqs, rows):
        seqs = [int(seq) for seq in seqs]
        rows = [rows] * len(seqs) if isinstance(rows, int) else [int(n) for n in rows]
        if len(rows) != len(seqs) or len(set(seqs)) != len(seqs):
            raise ValueError("%d row counts for the sequences %s" % (len(rows), seqs))
        return seqs, rows

    def _vectors(self, *lists):
        return torch.tensor(lists, dtype=torch.int32).to(self.pool.device).unbind(0)

    def _write(self, seqs):
        """The device's table of these sequences."""
        rows = torch.full((len(seqs), self.width), -1, dtype=torch.int32)
        for i, seq in enumerate(seqs):
            rows[i, :len(self._pages[seq])] = torch.tensor(self._pages[seq], dtype=torch.int32)
        self.table[torch.tensor(seqs, device=self.table.device)] = rows.to(self.table.device)

    # -------------------------------------------------------------------------------------------------- operators

    def batch(self, seqs):
        """(pages, lengths) of these sequences; views of the cache's own where seqs is an int n (sequences 0 .. n - 1)."""
        if isinstance(seqs, int):
            if not 0 <= seqs <= self.max_seqs:
                raise ValueError("%d sequences of a cache for %d" % (seqs, self.max_seqs))
            return self.table[:seqs], self.lengths[:seqs]
        seqs = [int(seq) for seq in seqs]
        for seq in seqs:
            self._known(seq)
        at = torch.tensor(seqs, dtype=torch.int64, device=self.table.device)
        return self.table[at], self.lengths[at]

    @staticmethod
    def _once(seqs):
        """The sequences of a call that stores rows."""
        if isinstance(seqs, int):
            return seqs
        seqs = [int(seq) for seq in seqs]
        if len(set(seqs)) != len(seqs):
            raise ValueError("sequences that get rows stand once each, not %s" % (seqs,))
        return seqs

    def layer(self, index, seqs):
        """One layer's operators for these sequences (an int n: the first n), bound to the cache's tables as they are."""
        return LayerOf(self.pool[index], *self.batch(seqs))

    def append(self, layer, k, v, seqs, starts=None, values=False):
        return self.layer(layer, self._once(seqs)).append(k, v, starts, values)

    def attention(self, layer, q, sm_scale, seqs, starts=None, selected=None, out=None, k_new=None, v_new=None):
        if k_new is not None:
            seqs = self._once(seqs)
        return self.layer(layer, seqs).attention(q, sm_scale, starts, selected, out, k_new, v_new)

    def select_pages(self, layer, q, count, seqs, keep_first=1, keep_last=1):
        return self.layer(layer, seqs).select_pages(q, count, keep_first, keep_last)


class LayerOf:
    """A pool with the tables of some sequences: append, attention and select_pages without naming them again."""

    def __init__(self, pool, pages, lengths):
        self.pool, self.pages, self.lengths = pool, pages, lengths

    def append(self, k, v, starts=None, values=False):
        return append(k, v, self.pool, self.pages, self.lengths, starts, values)

    def attention(self, q, sm_scale, starts=None, selected=None, out=None, k_new=None, v_new=None):
        return attention(q, self.pool, self.pages, self.lengths, sm_scale, starts, selected, out, k_new, v_new)

    def select_pages(self, q, count, keep_first=1, keep_last=1):
        return select_pages(q, self.pool, self.pages, self.lengths, count, keep_first, keep_last)
