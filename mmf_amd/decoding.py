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
call here waits for the GPU, and every call can be captured into a hipGraph (its numbers with it: a selection that is replayed takes its `step` from the device).  An
index outside its table (a page, a slot, a parent, a step) is left out and reported by `mmf_amd._native.take_index_error()`.  Forward only: tensors that require
gradients are refused while gradients are on, and so are those that carry a tangent of forward-mode differentiation.  The
operators have no form without data, so torch.compile does not trace through them: call them outside of what it compiles."""
import os
from collections import namedtuple

import torch

from mmf_amd import _native as nat

I32, I64 = torch.int32, torch.int64

PagePlan = namedtuple("PagePlan", "q_start q_lens kv_lens slots positions copies free_top refused beams")
PagePlan.__doc__ = """A step's plan.  q_start int32 [groups * beams] (shared: [groups]) first token row of each; q_lens [groups] planned new tokens (0: the group
waits); kv_lens [groups] new lengths; slots int64 [rows] and positions int32 [rows], -1 where a row holds no planned token; copies int32 [groups * beams, 3] for
`copy_pages`; free_top, refused int32 [1]; beams: rows per length in this plan (1 when shared)."""
BeamStep = namedtuple("BeamStep", "scores parents tokens finished history")
BeamStep.__doc__ = "scores fp32, parents int64, tokens int64, finished bool, each [groups, beams], best first; history int64 [groups, beams, length] or None."


_LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libmmf_amd_decode.so")
_ops = None


def _lib():
    """torch.ops.mmf_amd_decode (csrc/decode_binding.cpp: every argument check and the call of the C entry), loaded at the first call."""
    global _ops
    if _ops is None:
        nat.lib()                       # the kernels' C ABI first (raises when it is missing)
        if not os.path.exists(_LIB_PATH):
            raise nat.NativeLibraryError("mmf_amd decoding library not found at %s. Build it with `python -m mmf_amd.csrc.build`. There is no fallback path." % _LIB_PATH)
        torch.ops.load_library(_LIB_PATH)
        ns = torch.ops.mmf_amd_decode
        forms = dict({n: getattr(ns, n).default for n in ("plan_pages", "write_pages", "attend_pages", "select_beams", "reorder_pages", "copy_pages")},
                     **{n + "_out": getattr(ns, n).out for n in ("plan_pages", "attend_pages", "select_beams", "reorder_pages")})
        _ops = namedtuple("Ops", forms)(**forms)
    return _ops


def plan_pages(q_lens, kv_lens, tables, owned, free_pages, free_top, *, page_size, rows, beams=1, shared=False, out=None):
    """Pages and slots of a step, from lengths on the device.

    q_lens int32 [groups]: new tokens of each row of a group (`shared`: of the group, while its rows still have one table: all see them, as a prompt); negative: the group is done, the
    pages its rows own go back on the free list and its length becomes 0.  kv_lens int32 [groups]: tokens in the cache.  tables, owned int32 [groups * beams,
    blocks]: the block tables, and which page each row took itself (both written in place).  free_pages int32 [capacity], free_top int32 [1]: the free list, pages
    are taken from its top.  rows: rows of the step's token buffers; the tokens of a group (of each of its beams) follow those of the group before.

    A group is served whole or waits (no page, no slot, q_lens 0): when its tokens do not fit its table row or `rows`, or when it and the groups before it need
    more pages than are free.  Not shared, a row that still shares the block it goes on writing gets a page of its own and a line in `copies`: call
    `copy_pages(plan.copies, cache)` before the write.  Lengths change by plans alone (a length set back by hand loses the pages behind it).
    `out`: a PagePlan whose tensors take the results; its kv_lens and free_top may be the inputs."""
    if out is None:
        return PagePlan(*_lib().plan_pages(q_lens, kv_lens, tables, owned, free_pages, free_top, page_size, rows, beams, shared), 1 if shared else beams)
    if len(out) < 8:
        raise nat.NativeLibraryError("out must be a PagePlan, got %d tensors" % len(out))
    start, lens, kv, slots, positions, copies, top, refused = out[:8]
    _lib().plan_pages_out(q_lens, kv_lens, tables, owned, free_pages, free_top, page_size, rows, beams, shared, out_q_start=start, out_q_lens=lens, out_kv_lens=kv,
                          out_slots=slots, out_positions=positions, out_copies=copies, out_free_top=top, out_refused=refused)
    return PagePlan(start, lens, kv, slots, positions, copies, top, refused, 1 if shared else beams)


def write_pages(k, v, key_cache, value_cache, slots):
    """k, v [rows, kv_heads, head_dim] (contiguous head_dim; slices of a packed projection as they are) into the slots of their rows: slot = page * page_size +
    position, negative: the row is left out.  What a slot holds that two rows name is undefined.  The caches are bf16 or fp32, as k and v."""
    _lib().write_pages(k, v, key_cache, value_cache, slots)


def attend_pages(q, key_cache, value_cache, tables, kv_lens, q_start, q_lens, *, max_q, beams=1, causal=True, scale=None, out=None):
    """Attention of new tokens over the pages of their request: out[i] = softmax_j(scale * q[i] . k[j]) v[j].

    q [rows, heads, head_dim] (contiguous head_dim 64 or 128), bf16 or fp32 as the caches; heads a multiple of kv_heads, query head h reads key head
    h // (heads // kv_heads).  Request r has the token rows q_start[r] .. + q_lens[r // beams] and the keys of its first kv_lens[r // beams] tokens, of which the
    new tokens, written before, are the last.  causal: a new token sees the keys up to itself; else all of them.  tables int32 [requests, blocks]
    (contiguous rows); kv_lens, q_lens int32 [requests // beams], q_start int32 [requests].  max_q: no request has more new tokens (tokens beyond are left out and
    reported).  scale: default head_dim ** -0.5.  A token that sees no key gives zeros; rows of `out` that no request names are left as they are (undefined
    where `out` is made here).  `out` may be q.  A page outside the pool reads as zeros and is reported.

    Requests longer than 512 keys may be split over the chip.  A call whose tables have room for such ones takes a workspace from torch's allocator, whatever the lengths are: 9 MB
    at head_dim 64 and 17 at 128 for single tokens (up to 32 rows of query heads and new tokens per key head), 52 and 102 MB for chunks; a captured call keeps its own."""
    if out is None:
        return _lib().attend_pages(q, key_cache, value_cache, tables, kv_lens, q_start, q_lens, max_q, beams, causal, scale)
    _lib().attend_pages_out(q, key_cache, value_cache, tables, kv_lens, q_start, q_lens, max_q, beams, causal, scale, out=out)
    return out


def select_beams(logits, scores, finished, *, eos, history=None, step=0, out=None):
    """The best `beams` continuations of each group over beams x vocabulary.

    logits [groups * beams, vocab] bf16 or fp32 (contiguous rows; up to 2**22 tokens); scores fp32 [groups, beams]: the sums of log-probabilities so far, -inf for a beam that is not
    live (all but one before the first token); finished bool [groups, beams].  A candidate is scores + log_softmax(logits); a finished beam has one, the token `eos` at its
    score.  Descending, among equals the lowest beam * vocab + token first.  NaN counts as -inf; a row that holds +inf is all -inf.  history int64
    [groups, beams, length]: the rows of the parents come back with the new tokens in column `step`, a number or an int32 [1] tensor on the device; a number is
    part of a captured call and stays what it was at capture, so a step that is replayed takes a tensor and advances it (`step += 1`).  `out`: a BeamStep whose tensors take the results; each may be the input
    of its kind."""
    at = step if torch.is_tensor(step) else None
    step = 0 if at is not None else step
    if out is None:
        r = _lib().select_beams(logits, scores, finished, eos, history, step, at)
        return BeamStep(*r) if history is not None else BeamStep(*r[:4], None)
    if not 4 <= len(out) <= 5:
        raise nat.NativeLibraryError("out must be a BeamStep, got %d tensors" % len(out))
    out = BeamStep(*out[:4], out[4] if len(out) == 5 else None)
    _lib().select_beams_out(logits, scores, finished, eos, history, step, at, out_scores=out.scores, out_parents=out.parents, out_tokens=out.tokens,
                            out_finished=out.finished, out_history=out.history)
    return out


def reorder_pages(parents, kv_lens, tables, cache, *, out=None):
    """The block tables after a selection, with the copies it takes.

    parents int64 [groups, beams]; kv_lens int32 [groups]: tokens in the cache; tables int32 [groups * beams, blocks]; cache [..., pages, kv_heads, page_size,
    head_dim]: every pool the tables are for (keys and values of all layers), leading dimensions as one contiguous run of planes.  Full blocks are shared by the children
    of a beam.  The block that goes on being written stays with the first child; the other children take the pages of beams without children and get its
    tokens copied in.  Returns the new tables (`out` may be `tables`).

    Pages stay with the row that took them until their group is done, also full ones that no table names any more: a pool has to hold, for each group, the blocks of its
    prompt and `beams` times the blocks written since, not just the pages that are still read."""
    if out is None:
        return _lib().reorder_pages(parents, kv_lens, tables, cache)
    _lib().reorder_pages_out(parents, kv_lens, tables, cache, out=out)
    return out


def copy_pages(copies, cache):
    """copies int32 [n, 3]: (source page, destination page, tokens); that many tokens of the page, in every plane of cache [..., pages, kv_heads, page_size,
    head_dim].  A negative page: nothing to copy.  No page may be both a source and a destination (the plans and tables of this module keep to that)."""
    _lib().copy_pages(copies, cache)


class PagedCache:
    """Pool, block tables, free list and lengths of a decoder with `layers` layers for `groups` requests of `beams` rows of up to `max_len` tokens.  `pages`: those that any
    course of decoding can take (groups * beams * blocks); with fewer, groups may have to wait (`plan.refused`).  Every update is in place, so that a
    step can be captured once and replayed (with `select_beams(..., step=at)`, `at` an int32 [1] tensor that the step advances).

        cache = PagedCache(layers, groups, beams, max_len, kv_heads=12, head_dim=64)
        plan = cache.plan(prompt_lens, rows, shared=True)         # the prompts: once per group
        cache.write(l, k, v, plan); ctx = cache.attend(l, q, plan, max_q=..., causal=False)
        cache.reorder(parents); plan = cache.plan(ones, rows)     # a step: one token per beam"""

    def __init__(self, layers, groups, beams, max_len, *, kv_heads, head_dim, page_size=16, pages=None, dtype=torch.bfloat16, device="cuda"):
        def need(ok, what):
            if not ok:
                raise nat.NativeLibraryError(what)

        need(1 <= page_size <= 1024 and page_size & (page_size - 1) == 0, "page_size must be a power of two up to 1024")
        need(1 <= beams <= 32, "beams must be 1 .. 32")
        need(layers > 0 and groups > 0 and max_len > 0 and kv_heads > 0, "layers, groups, max_len and kv_heads must be positive")
        need(head_dim in (64, 128) and dtype in (torch.bfloat16, torch.float32), "head_dim must be 64 or 128, dtype bf16 or fp32")
        blocks = -(-max_len // page_size)
        pages = groups * beams * blocks if pages is None else pages
        need(pages > 0, "pages must be positive")
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
