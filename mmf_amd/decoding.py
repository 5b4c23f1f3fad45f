"""Decoding with a paged key / value cache and several beams per request: the operators of one step, on the GPU from the lengths to the chosen tokens.

    plan_pages     pages for the new tokens, from a free list, and the slot of each new token
    write_pages    new keys and values into their slots
    attend_pages   attention of the new tokens (one each, or a chunk) over the pages of their request
    select_beams   the best continuations of each group of beams, with the token histories
    reorder_pages  the block tables after a selection; copy_pages for the pages that two beams would go on writing
    PagedCache     the pool, the tables and the lengths of a decoder, and the calls above on them

The reference decodes M4C greedily by re-running the whole transformer (mmf/models/m4c.py:284-304) and selects beams on the host (mmf/utils/text.py BeamSearch).
`M4C` with `num_beams` in its config decodes through this module.

A cache pool is [pages, kv_heads, page_size, head_dim] (any strides with contiguous head_dim), page_size a power of two up to 1024, bf16 or fp32.  Requests come
in groups of `beams` rows of the same length; a block table [groups * beams, blocks] int32 names the page of every block of a row.  Lengths stay on the device: no
call here waits for the GPU, and every call can be captured into a hipGraph.  An index outside its table (a page, a slot, a parent) is left out and reported by
`mmf_amd._native.take_index_error()`.  Forward only: tensors that require gradients are refused while gradients are on."""
from collections import namedtuple

import torch

from mmf_amd import _native as nat
from mmf_amd._native import NativeLibraryError

I32, I64 = torch.int32, torch.int64

PagePlan = namedtuple("PagePlan", "q_start q_lens kv_lens slots positions copies free_top refused beams")
PagePlan.__doc__ = """A step's plan.  q_start int32 [groups * beams] (shared: [groups]) first token row of each; q_lens [groups] planned new tokens (0: the group
waits); kv_lens [groups] new lengths; slots int64 [rows] and positions int32 [rows], -1 where a row holds no planned token; copies int32 [groups * beams, 3] for
`copy_pages`; free_top, refused int32 [1]; beams: rows per length in this plan (1 when shared)."""
BeamStep = namedtuple("BeamStep", "scores parents tokens finished history")
BeamStep.__doc__ = "scores fp32, parents int64, tokens int64, finished bool, each [groups, beams], best first; history int64 [groups, beams, length] or None."


def _need(ok, *message):
    if not ok:
        raise NativeLibraryError(message[0] % message[1:] if len(message) > 1 else message[0])


def _check(t, name, dtype, shape=None, dense=True):
    _need(isinstance(t, torch.Tensor), "%s must be a tensor", name)
    _need(t.dtype == dtype if isinstance(dtype, torch.dtype) else t.dtype in dtype, "%s must be %s, got %s", name, dtype, t.dtype)
    if shape is not None:
        _need(t.dim() == len(shape) and all(a is None or a == b for a, b in zip(shape, t.shape)), "%s must be %s, got %s", name,
              list(shape), list(t.shape))
    _need(not dense or t.is_contiguous(), "%s must be contiguous", name)
    _need(not (t.requires_grad and torch.is_grad_enabled()), "%s requires a gradient: decoding is forward only (torch.no_grad)", name)


class _on:
    """The device of the tensors for the duration of a call (its current stream takes the work); every tensor has to live there."""

    def __init__(self, *tensors):
        self.device = tensors[0].device
        _need(all(t is None or t.device == self.device for t in tensors), "tensors on different devices: %s", sorted({str(t.device) for t in tensors if t is not None}))
        _need(self.device.type == "cuda", "tensors must live in HBM (cuda/hip tensors), got %s; there is no CPU path", self.device)
        self.guard = torch.cuda.device(self.device) if self.device.index != torch.cuda.current_device() else None

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _page_size(n):
    _need(isinstance(n, int) and 1 <= n <= nat.PAGE_MAX and n & (n - 1) == 0, "page_size must be a power of two up to %d, got %s", nat.PAGE_MAX, n)


def _beams(n):
    _need(isinstance(n, int) and 1 <= n <= nat.BEAMS_MAX, "beams must be 1 .. %d, got %s", nat.BEAMS_MAX, n)


FLOATS = (torch.bfloat16, torch.float32)


def _pool(t, name, dtype=FLOATS):
    _check(t, name, dtype, dense=False)
    _need(t.dim() == 4 and t.stride(3) == 1 and t.numel() > 0, "%s must be [pages, kv_heads, page_size, head_dim] with contiguous head_dim, got %s", name, list(t.shape))
    _page_size(t.shape[2])


def plan_pages(q_lens, kv_lens, tables, owned, free_pages, free_top, *, page_size, rows, beams=1, shared=False, out=None):
    """Pages and slots of a step, from lengths on the device.

    q_lens int32 [groups]: new tokens of each row of a group (`shared`: of the group, all of whose rows see them, as a prompt); negative: the group is done, the
    pages its rows own go back on the free list and its length becomes 0.  kv_lens int32 [groups]: tokens in the cache.  tables, owned int32 [groups * beams,
    blocks]: the block tables, and which page each row took itself (both written in place).  free_pages int32 [capacity], free_top int32 [1]: the free list, pages
    are taken from its top.  rows: rows of the step's token buffers; the tokens of a group (of each of its beams) follow those of the group before.

    A group is served whole or waits (no page, no slot, q_lens 0): when its tokens do not fit its table row or `rows`, or when it and the groups before it need
    more pages than are free.  Not shared, a row that still shares the block it goes on writing gets a page of its own and a line in `copies`: call
    `copy_pages(plan.copies, cache)` before the write.  `out`: a PagePlan whose tensors take the results; its kv_lens and free_top may be the inputs."""
    _page_size(page_size); _beams(beams)
    _check(q_lens, "q_lens", I32, (None,))
    G = q_lens.numel()
    _need(G > 0 and isinstance(rows, int) and 0 < rows <= 1 << 30, "plan_pages needs groups and 1 .. 2**30 rows, got %s and %s", G, rows)
    _check(kv_lens, "kv_lens", I32, (G,)); _check(tables, "tables", I32, (G * beams, None)); _check(owned, "owned", I32, tuple(tables.shape))
    _check(free_pages, "free_pages", I32, (None,)); _check(free_top, "free_top", I32, (1,))
    _need(tables.shape[1] > 0 and free_pages.numel() > 0, "tables and free_pages must not be empty")
    _need(tables.shape[1] * page_size <= 1 << 30, "a table row names more than 2**30 tokens")
    n = G if shared else G * beams
    with _on(q_lens, kv_lens, tables, owned, free_pages, free_top, *((t for t in out[:8]) if out is not None else ())):
        if out is None:
            # one buffer for the small outputs: an allocation costs as much time as a small plan
            dev = q_lens.device
            ints = torch.empty(n + 2 * G + rows + 3 * G * beams + 2, dtype=I32, device=dev)
            parts = ints.split((n, G, G, rows, 3 * G * beams, 1, 1))
            out = PagePlan(parts[0], parts[1], parts[2], torch.empty(rows, dtype=I64, device=dev), parts[3], parts[4].view(G * beams, 3), parts[5], parts[6],
                           1 if shared else beams)
        else:
            for t, name, dt, shape in zip(out, PagePlan._fields, (I32, I32, I32, I64, I32, I32, I32, I32), ((n,), (G,), (G,), (rows,), (rows,), (G * beams, 3), (1,), (1,))):
                _check(t, "out." + name, dt, shape)
            out = out._replace(beams=1 if shared else beams)
        nat.paged_plan(q_lens, kv_lens, tables, owned, free_pages, free_top, out.q_start, out.q_lens, out.kv_lens, out.slots, out.positions, out.copies, out.free_top,
                       out.refused, beams, page_size, shared)
    return out


def write_pages(k, v, key_cache, value_cache, slots):
    """k, v [rows, kv_heads, head_dim] (contiguous head_dim; slices of a packed projection as they are) into the slots of their rows: slot = page * page_size +
    position, negative: the row is left out.  A slot that two rows name gets one of them.  The caches are bf16 or fp32, as k and v."""
    _pool(key_cache, "key_cache"); _pool(value_cache, "value_cache", key_cache.dtype)
    _need(value_cache.shape == key_cache.shape and value_cache.stride() == key_cache.stride(), "key_cache and value_cache must have one shape and one layout")
    _check(slots, "slots", I64, (None,))
    shape = (slots.numel(), key_cache.shape[1], key_cache.shape[3])
    for t, name in ((k, "k"), (v, "v")):
        _check(t, name, key_cache.dtype, shape, dense=False)
        _need(t.stride(2) == 1 or t.shape[2] == 1, "%s must have contiguous head_dim", name)
    with _on(k, v, key_cache, value_cache, slots):
        if slots.numel():
            nat.paged_write(k, v, key_cache, value_cache, slots)


def attend_pages(q, key_cache, value_cache, tables, kv_lens, q_start, q_lens, *, max_q, beams=1, causal=True, scale=None, out=None):
    """Attention of new tokens over the pages of their request: out[i] = softmax_j(scale * q[i] . k[j]) v[j].

    q [rows, heads, head_dim] (contiguous head_dim 64 or 128), bf16 or fp32 as the caches; heads a multiple of kv_heads, query head h reads key head
    h // (heads // kv_heads).  Request r has the token rows q_start[r] .. + q_lens[r // beams] and the keys of its first kv_lens[r // beams] tokens, of which the
    new tokens, written before, are the last.  causal: a new token sees the keys up to itself; else all of them.  tables int32 [requests, blocks]
    (contiguous rows); kv_lens, q_lens int32 [requests // beams], q_start int32 [requests].  max_q: no request has more new tokens.  scale: default
    head_dim ** -0.5.  A token that sees no key gives zeros; rows of `out` that no request names are left as they are (undefined where `out` is made here)."""
    _pool(key_cache, "key_cache"); _pool(value_cache, "value_cache", key_cache.dtype)
    _need(value_cache.shape == key_cache.shape and value_cache.stride() == key_cache.stride(), "key_cache and value_cache must have one shape and one layout")
    pages, kv_heads, page_size, dim = key_cache.shape
    _need(dim in (64, 128), "head_dim must be 64 or 128, got %s", dim)
    _beams(beams)
    _check(tables, "tables", I32, (None, None), dense=False)
    _need(tables.numel() > 0 and (tables.stride(1) == 1 or tables.shape[1] == 1), "tables must be [requests, blocks] with contiguous rows")
    R = tables.shape[0]
    _need(R % beams == 0, "%d table rows are no groups of %d beams", R, beams)
    _need(tables.shape[1] * page_size <= 1 << 30, "a table row names more than 2**30 tokens")
    _check(kv_lens, "kv_lens", I32, (R // beams,)); _check(q_lens, "q_lens", I32, (R // beams,)); _check(q_start, "q_start", I32, (R,))
    _check(q, "q", key_cache.dtype, (None, None, dim), dense=False)
    _need(q.stride(2) == 1 and q.shape[1] % kv_heads == 0 and q.shape[1] > 0, "q must be [rows, heads, head_dim], contiguous head_dim, heads a multiple of %d; got %s",
          kv_heads, list(q.shape))
    _need(isinstance(max_q, int) and max_q >= 1, "max_q must be at least 1, got %s", max_q)
    for t, name in ((q, "q"), (key_cache, "key_cache"), (value_cache, "value_cache")):
        _need(t.data_ptr() % 16 == 0 and all(s * t.element_size() % 16 == 0 or n == 1 for s, n in zip(t.stride()[:-1], t.shape)),
              "%s must start and stride on 16 bytes", name)
    with _on(q, key_cache, value_cache, tables, kv_lens, q_start, q_lens, out):
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        else:
            _check(out, "out", q.dtype, tuple(q.shape), dense=False)
            _need(out.stride(2) == 1 and out.data_ptr() % 16 == 0 and all(s * out.element_size() % 16 == 0 for s in out.stride()[:2]),
                  "out must have contiguous head_dim and start and stride on 16 bytes")
        if q.shape[0]:
            nat.paged_attention(q, key_cache, value_cache, tables, kv_lens, q_start, q_lens, out, beams, min(max_q, q.shape[0]), causal,
                                float(dim ** -0.5 if scale is None else scale))
    return out


def select_beams(logits, scores, finished, *, eos, history=None, step=0, out=None):
    """The best `beams` continuations of each group over beams x vocabulary.

    logits [groups * beams, vocab] bf16 or fp32 (contiguous rows); scores fp32 [groups, beams]: the sums of log-probabilities so far, -inf for a beam that is not
    live (all but one before the first token); finished bool [groups, beams].  A candidate is scores + log_softmax(logits); a finished beam has one, the token `eos` at its
    score.  Descending, among equals the lowest beam * vocab + token first.  NaN counts as -inf; a row that holds +inf is all -inf.  history int64
    [groups, beams, length]: the rows of the parents come back with the new tokens in column `step`.  `out`: a BeamStep whose tensors take the results; each may be the input
    of its kind."""
    _check(scores, "scores", torch.float32, (None, None))
    G, W = scores.shape
    _beams(W)
    _need(G > 0, "select_beams needs a group")
    _check(logits, "logits", FLOATS, (G * W, None), dense=False)
    V = logits.shape[1]
    _need(V > 0 and (logits.stride(1) == 1 or V == 1) and (logits.stride(0) >= V or G * W == 1), "logits must have contiguous rows that do not overlap")
    _check(finished, "finished", torch.bool, (G, W))
    _need(isinstance(eos, int) and 0 <= eos < V, "eos %s is not in the vocabulary of %d", eos, V)
    if history is not None:
        _check(history, "history", I64, (G, W, None))
        _need(isinstance(step, int) and 0 <= step < history.shape[2], "step %s is not a column of the history of length %d", step, history.shape[2])
    with _on(logits, scores, finished, history, *((t for t in out) if out is not None else ())):
        if out is None:
            dev = logits.device
            ids = torch.empty(2, G, W, dtype=I64, device=dev)
            out = BeamStep(torch.empty(G, W, dtype=torch.float32, device=dev), ids[0], ids[1], torch.empty(G, W, dtype=torch.bool, device=dev),
                           None if history is None else torch.empty(history.shape, dtype=I64, device=dev))
        else:
            for t, name, dt in zip(out, BeamStep._fields, (torch.float32, I64, I64, torch.bool)):
                _check(t, "out." + name, dt, (G, W))
            _need((out.history is None) == (history is None), "out.history goes with history")
            if history is not None:
                _check(out.history, "out.history", I64, tuple(history.shape))
        nat.beam_select(logits, scores, finished, history, out.scores, out.parents, out.tokens, out.finished, out.history, eos, step)
    return out


def reorder_pages(parents, kv_lens, tables, cache, *, out=None):
    """The block tables after a selection, with the copies it takes.

    parents int64 [groups, beams]; kv_lens int32 [groups]: tokens in the cache; tables int32 [groups * beams, blocks]; cache [..., pages, kv_heads, page_size,
    head_dim]: every pool the tables are for (keys and values of all layers), leading dimensions as one contiguous run of planes.  Full blocks are shared by the children
    of a beam.  The block that goes on being written stays with the first child; the other children take the pages of beams without children and get its
    tokens copied in.  Returns the new tables (`out` may be `tables`)."""
    _check(parents, "parents", I64, (None, None))
    G, W = parents.shape
    _beams(W)
    _need(G > 0, "reorder_pages needs a group")
    _check(kv_lens, "kv_lens", I32, (G,)); _check(tables, "tables", I32, (G * W, None))
    _need(tables.shape[1] > 0, "tables must not be empty")
    _planes(cache)
    with _on(parents, kv_lens, tables, cache, out):
        if out is None:
            out = torch.empty_like(tables)
        else:
            _check(out, "out", I32, tuple(tables.shape))
        copies = torch.empty(G * W, 3, dtype=I32, device=tables.device)
        nat.paged_reorder(parents, kv_lens, tables, out, copies, cache.shape[-2])
        nat.paged_copy(copies, cache)
    return out


def _planes(cache):
    _check(cache, "cache", FLOATS, dense=False)
    _need(cache.dim() >= 4 and cache.numel() > 0 and cache.stride(-1) == 1, "cache must be [..., pages, kv_heads, page_size, head_dim] with contiguous head_dim")
    for a in range(cache.dim() - 5):
        _need(cache.stride(a) == cache.stride(a + 1) * cache.shape[a + 1], "the leading dimensions of cache must be one run of planes")
    _page_size(cache.shape[-2])


def copy_pages(copies, cache):
    """copies int32 [n, 3]: (source page, destination page, tokens); that many tokens of the page, in every plane of cache [..., pages, kv_heads, page_size,
    head_dim].  A negative page: nothing to copy.  No page may be both a source and a destination (the plans and tables of this module keep to that)."""
    _check(copies, "copies", I32, (None, 3))
    _planes(cache)
    with _on(copies, cache):
        if copies.shape[0]:
            nat.paged_copy(copies, cache)


class PagedCache:
    """Pool, block tables, free list and lengths of a decoder with `layers` layers for `groups` requests of `beams` rows; every update is in place, so that a
    step can be captured once and replayed.

        cache = PagedCache(layers, groups, beams, max_len, kv_heads=12, head_dim=64)
        plan = cache.plan(prompt_lens, rows, shared=True)         # the prompts: once per group
        cache.write(l, k, v, plan); ctx = cache.attend(l, q, plan, max_q=..., causal=False)
        cache.reorder(parents); plan = cache.plan(ones, rows)     # a step: one token per beam"""

    def __init__(self, layers, groups, beams, max_len, *, kv_heads, head_dim, page_size=16, pages=None, dtype=torch.bfloat16, device="cuda"):
        _page_size(page_size); _beams(beams)
        _need(layers > 0 and groups > 0 and max_len > 0 and kv_heads > 0, "layers, groups, max_len and kv_heads must be positive")
        _need(head_dim in (64, 128) and dtype in FLOATS, "head_dim is 64 or 128, dtype bf16 or fp32")
        blocks = -(-max_len // page_size)
        pages = groups * beams * blocks if pages is None else pages
        _need(pages > 0, "pages must be positive")
        self.beams, self.page_size = beams, page_size
        self.data = torch.zeros(layers, 2, pages, kv_heads, page_size, head_dim, dtype=dtype, device=device)
        self.tables = torch.empty(groups * beams, blocks, dtype=I32, device=device)
        self.owned = torch.empty_like(self.tables)
        self.kv_lens = torch.empty(groups, dtype=I32, device=device)
        self.free_pages = torch.empty(pages, dtype=I32, device=device)
        self.free_top = torch.empty(1, dtype=I32, device=device)
        self.reset()

    def reset(self):
        """Every page free, every length 0."""
        self.tables.fill_(-1); self.owned.fill_(-1); self.kv_lens.zero_()
        n = self.free_pages.numel()
        torch.arange(n - 1, -1, -1, dtype=I32, device=self.free_pages.device, out=self.free_pages)
        self.free_top.fill_(n)

    def plan(self, q_lens, rows, shared=False):
        """`plan_pages` on this cache's state, lengths and free list in place; pages that rows shared so far are copied."""
        dev, G, W = self.tables.device, self.kv_lens.numel(), self.beams
        n = G if shared else G * W
        new = lambda *s, dt=I32: torch.empty(*s, dtype=dt, device=dev)
        out = PagePlan(new(n), new(G), self.kv_lens, new(rows, dt=I64), new(rows), new(G * W, 3), self.free_top, new(1), W)
        plan = plan_pages(q_lens, self.kv_lens, self.tables, self.owned, self.free_pages, self.free_top, page_size=self.page_size, rows=rows, beams=W, shared=shared,
                          out=out)
        if W > 1 and not shared:
            copy_pages(plan.copies, self.data)
        return plan

    def write(self, layer, k, v, plan):
        write_pages(k, v, self.data[layer, 0], self.data[layer, 1], plan.slots)

    def attend(self, layer, q, plan, *, max_q, causal=True, scale=None, out=None):
        shared = plan.beams == 1
        return attend_pages(q, self.data[layer, 0], self.data[layer, 1], self.tables[::self.beams] if shared else self.tables, plan.kv_lens, plan.q_start,
                            plan.q_lens, max_q=max_q, beams=plan.beams, causal=causal, scale=scale, out=out)

    def reorder(self, parents):
        reorder_pages(parents, self.kv_lens, self.tables, self.data, out=self.tables)
