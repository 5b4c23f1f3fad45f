"""The operators of cached decoding: what is measured.

Five operators make up one step of decoding with a paged key / value cache, several beams per request:

  plan      pages for the new tokens of every request, taken from a free list on the GPU, and the slot of each new token
  write     the new tokens' keys and values into their slots
  attend    attention of the new tokens (one each, or a whole chunk) over the pages of their request
  select    the best continuations of every group of beams over beams x vocabulary, with the token histories
  reorder   the block tables after the beams' parents, with copies of the pages that two beams would go on writing

`run` computes them in plain torch operations, or, with `own` set, through mmf_amd.decoding."""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EOS = 2


def listed():
    return [
        # every decoding step of 32 images with 5 beams: one token per beam, 16-token pages
        _plan("plan_step", groups=32, beams=5, page=16, shared=False, ctx=(30, 181), new=(1, 1), tail=12, released=0.0, short=False),
        # a serving batch that admits prompts and chunks while finished requests give their pages back
        _plan("plan_prompts", groups=512, beams=1, page=16, shared=True, ctx=(0, 4096), new=(1, 2048), tail=0, released=0.1, short=False),
        # the K and V thirds of a packed projection, one token per beam of 32 images
        _write("write_step", tokens=160, kv_heads=12, dim=64, page=16, dtype="bf16", skipped=0.0),
        # prompts of a batch with grouped heads, some rows padding
        _write("write_prompts", tokens=16384, kv_heads=8, dim=128, page=32, dtype="bf16", skipped=0.1),
        # one decoding step over text, objects and OCR tokens: 5 beams share their image's pages
        _attend("attend_step", groups=32, beams=5, heads=12, kv_heads=12, dim=64, page=16, dtype="bf16", causal=True, ctx=(120, 181), new=(1, 1), tail=8),
        # few long conversations, grouped heads: one token over a long cache
        _attend("attend_long", groups=8, beams=1, heads=32, kv_heads=8, dim=128, page=16, dtype="bf16", causal=True, ctx=(16384, 65536), new=(1, 1), tail=0),
        # chunks of prompts of different lengths over what is cached of them
        _attend("attend_chunks", groups=6, beams=1, heads=32, kv_heads=8, dim=128, page=16, dtype="bf16", causal=True, ctx=(256, 16384), new=(256, 2048), tail=0),
        # the encoder positions of 32 images, all of which see each other, in the accurate mode
        _attend("attend_prompt_fp32", groups=32, beams=1, heads=12, kv_heads=12, dim=64, page=16, dtype="fp32", causal=False, ctx=(0, 0), new=(70, 170), tail=0),
        # the scores of 32 images with 5 beams over the answer vocabulary and the OCR tokens
        _select("select_step", groups=32, beams=5, vocab=5050, dtype="fp32", masked=45, done=0.2, first=False, length=12),
        # a large vocabulary
        _select("select_large", groups=16, beams=8, vocab=128000, dtype="bf16", masked=0, done=0.1, first=False, length=256),
        # the caches of a four-layer decoder after a selection of 5 beams for 32 images
        _reorder("reorder_step", groups=32, beams=5, layers=4, kv_heads=12, dim=64, page=16, dtype="bf16", ctx=(40, 181), tail=12),
        # long shared prompts, a deeper decoder
        _reorder("reorder_long", groups=8, beams=8, layers=16, kv_heads=8, dim=128, page=32, dtype="bf16", ctx=(2000, 4096), tail=100),
    ]


def draw(rng):
    shape = rng.randrange(1 << 30)
    op = rng.choice(["plan", "write", "attend", "attend", "select", "reorder"])
    if op == "plan":
        beams = rng.choice([1, 1, 2, 5, 8])
        shared = rng.random() < 0.5
        hi = _log(rng, 1, 2048) if shared or beams == 1 else rng.choice([1, 1, 3])
        return _plan(None, groups=_log(rng, 1, 512), beams=beams, page=rng.choice([8, 16, 32, 64]), shared=shared, ctx=(0, _log(rng, 1, 4096)), new=(rng.choice([0, 1]), hi),
                     tail=_log(rng, 1, 64), released=rng.choice([0.0, 0.1, 0.5]), short=rng.random() < 0.25, shape=shape)
    if op == "write":
        return _write(None, tokens=_log(rng, 1, 16384), kv_heads=rng.choice([1, 2, 5, 8, 12]), dim=rng.choice([64, 128]), page=rng.choice([8, 16, 32, 64]),
                      dtype=rng.choice(["bf16", "bf16", "fp32"]), skipped=rng.choice([0.0, 0.1, 0.5]), shape=shape)
    if op == "attend":
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        kv_heads = rng.choice([1, 2, 4, 8, 12])
        heads = kv_heads * rng.choice([1, 1, 2, 4, 8] if kv_heads <= 4 else [1, 1, 2, 4] if kv_heads == 8 else [1, 2])
        dim, page = rng.choice([64, 128]), rng.choice([8, 16, 32, 64])
        if rng.random() < 0.5:         # single tokens, or a few
            beams = rng.choice([1, 1, 2, 5, 8])
            ctx = _log(rng, 1, 8192 if dtype == "fp32" or beams > 1 else 65536)
            groups = _log(rng, 1, max(1, min(256 // beams, (1 << 19) // ctx)))
            return _attend(None, groups=groups, beams=beams, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, causal=True,
                           ctx=(max(0, ctx // 3), ctx), new=(1, rng.choice([1, 1, 2, 5])), tail=_log(rng, 1, 40), shape=shape)
        new = _log(rng, 8, 256 if dtype == "fp32" else 2048)
        ctx = rng.choice([0, _log(rng, 1, 2048 if dtype == "fp32" else 16384)])
        groups = _log(rng, 1, max(1, min(64, int(3e8 / (heads * new * (new + ctx))))))
        return _attend(None, groups=groups, beams=1, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, causal=rng.random() < 0.7,
                       ctx=(0, ctx), new=(rng.choice([1, new]), new), tail=0, shape=shape)
    if op == "select":
        beams = rng.choice([1, 2, 3, 5, 8, 16])
        vocab = _log(rng, 100, 128000)
        return _select(None, groups=_log(rng, 1, max(1, min(256, 16384000 // (beams * vocab)))), beams=beams, vocab=vocab, dtype=rng.choice(["bf16", "fp32"]),
                       masked=rng.choice([0, vocab // 100, vocab // 3]), done=rng.choice([0.0, 0.2, 0.7]), first=rng.random() < 0.2, length=_log(rng, 1, 512), shape=shape)
    beams = rng.choice([2, 3, 5, 8, 16])
    layers = rng.choice([1, 4, 6, 12])
    return _reorder(None, groups=_log(rng, 1, 32), beams=beams, layers=layers, kv_heads=rng.choice([1, 4, 8, 12]), dim=rng.choice([64, 128]),
                    page=rng.choice([8, 16, 32]), dtype=rng.choice(["bf16", "bf16", "fp32"]), ctx=(1, _log(rng, 2, 1024)), tail=_log(rng, 1, 40), shape=shape)


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _case(op, name, shape, **kw):
    c = {"op": op, "shape": shape}
    for k, v in kw.items():
        if isinstance(v, tuple):
            c[k + "_lo"], c[k + "_hi"] = min(v), max(v)
        else:
            c[k] = v
    if name is not None:
        c["name"] = name
    return c


def _plan(name, shape=1, **kw):
    return _case("plan", name, shape, **kw)


def _write(name, shape=2, **kw):
    return _case("write", name, shape, **kw)


def _attend(name, shape=3, **kw):
    return _case("attend", name, shape, **kw)


def _select(name, shape=4, **kw):
    return _case("select", name, shape, **kw)


def _reorder(name, shape=5, **kw):
    return _case("reorder", name, shape, **kw)


# ---------------------------------------------------------------------------------------------
# lengths, tables and pools: what the case alone says, before any seed
# ---------------------------------------------------------------------------------------------
def _lengths(c):
    """Cached and new tokens of each group, spread evenly over the logarithm of their range."""
    rng = random.Random(c["shape"])
    ctx, new = [], []
    for _ in range(c["groups"]):
        ctx.append(_spread(rng, c["ctx_lo"], c["ctx_hi"]))
        new.append(_spread(rng, c["new_lo"], c["new_hi"]) if "new_lo" in c else 0)
    return ctx, new


def _spread(rng, lo, hi):
    return lo if lo == hi else min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1)))) - 1)))


def _up(a, b):
    return -(-a // b)


def _owners(length, prompt, beams, page):
    """Blocks of a group, and how many of them its beams share: the full ones of the prompt, or all where there is one beam."""
    blocks = _up(length, page)
    return blocks, blocks if beams == 1 else min(blocks, prompt // page)


def _tables(c, lengths, prompts, blocks_per_row, gen):
    """Block tables [groups * beams, blocks], who owns which page, and the pages that are left, in a shuffled pool."""
    W, page = c["beams"], c["page"]
    counts = [_owners(n, p, W, page) for n, p in zip(lengths, prompts)]
    used = sum(s + W * (b - s) for b, s in counts)
    G = len(lengths)
    tables = torch.full((G, W, blocks_per_row), -1, dtype=torch.int32)
    owned = torch.full((G, W, blocks_per_row), -1, dtype=torch.int32)
    spare = c.get("_spare", 0)
    pages = torch.randperm(used + spare, generator=gen, dtype=torch.int32)
    at = 0
    for g, (b, s) in enumerate(counts):
        tables[g, :, :s] = pages[at:at + s]
        owned[g, 0, :s] = pages[at:at + s]
        at += s
        tables[g, :, s:b] = pages[at:at + W * (b - s)].view(W, b - s)
        owned[g, :, s:b] = tables[g, :, s:b]
        at += W * (b - s)
    return tables.view(G * W, -1), owned.view(G * W, -1), pages[at:]


def _normal(shape, dtype, gen, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32) * scale).to(dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    host = torch.Generator()
    host.manual_seed(seed)
    return {"plan": _prepare_plan, "write": _prepare_write, "attend": _prepare_attend, "select": _prepare_select,
            "reorder": _prepare_reorder}[case["op"]](case, gen, host)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"plan": _own_plan, "write": _own_write, "attend": _own_attend, "select": _own_select, "reorder": _own_reorder}[op](state)
    return {"plan": _plain_plan, "write": _plain_write, "attend": _plain_attend, "select": _plain_select, "reorder": _plain_reorder}[op](state)


# ---------------------------------------------------------------------------------------------
# plan: pages and slots
# ---------------------------------------------------------------------------------------------
def _plan_numbers(c):
    ctx, new = _lengths(c)
    rng = random.Random(c["shape"] + 1)
    new = [-1 if n > 0 and rng.random() < c["released"] else m for n, m in zip(ctx, new)]      # -1: finished, its pages go back
    prompts = [n if c["shared"] else max(0, n - c["tail"]) for n in ctx]
    W = 1 if c["shared"] else c["beams"]
    rows = sum(W * max(0, m) for m in new)
    need = sum(W * (_up(n + m, c["page"]) - _up(n, c["page"])) for n, m in zip(ctx, new) if m > 0)
    return ctx, new, prompts, rows, need


def _prepare_plan(c, gen, host):
    ctx, new, prompts, rows, need = _plan_numbers(c)
    blocks = _up(max([n + max(0, m) for n, m in zip(ctx, new)] + [1]), c["page"]) + 1
    if c["short"]:
        need = need // 3               # fewer pages than asked for: the requests behind the last page wait
    t, o, free = _tables(dict(c, _spare=need + 7), ctx, [c["page"] * _up(p, c["page"]) if c["shared"] else p for p in prompts], blocks, host)
    stack = torch.full((t.max().item() + 1 if free.numel() == 0 else max(int(t.max()), int(free.max())) + 1,), -1, dtype=torch.int32)
    stack[:free.numel()] = free
    return {"case": c, "rows": max(rows, 1), "q_lens": _i32(new), "kv_lens": _i32(ctx), "tables": t.to(DEV), "owned": o.to(DEV), "free": stack.to(DEV),
            "top": _i32([free.numel()])}


def _own_plan(s):
    from mmf_amd import decoding
    c = s["case"]
    p = decoding.plan_pages(s["q_lens"], s["kv_lens"], s["tables"], s["owned"], s["free"], s["top"], page_size=c["page"], rows=s["rows"], beams=c["beams"],
                            shared=c["shared"])
    return [p.q_start, p.q_lens, p.kv_lens, p.slots, p.positions, p.copies, p.free_top, p.refused, s["tables"], s["owned"], s["free"]]


def _plain_plan(s):
    c = s["case"]
    W, ps, T = c["beams"], c["page"], s["rows"]
    shared = c["shared"] or W == 1
    tables, owned, free = s["tables"], s["owned"], s["free"]
    G, P = s["q_lens"].numel(), tables.shape[1]
    q, kv, top = s["q_lens"].long(), s["kv_lens"].long(), s["top"].long()
    j = torch.arange(P, device=DEV)
    row_kv = kv.repeat_interleave(W)
    # pages of the finished requests go back on the stack, in the order of their rows
    back = (q < 0).repeat_interleave(W)[:, None] & (j < ((row_kv + ps - 1) // ps)[:, None]) & (owned >= 0)
    rank = back.flatten().long().cumsum(0) - 1
    stack = torch.cat([free, free.new_zeros(1)])
    stack[torch.where(back.flatten(), top + rank, free.numel())] = torch.where(back, owned, 0).flatten()
    free.copy_(stack[:-1])
    top = top + back.sum()
    # what each row needs: its new blocks, and a page of its own for the block it shares so far and goes on writing
    n = q.clamp(min=0)
    row_n = n.repeat_interleave(W)
    have, want = (row_kv + ps - 1) // ps, (row_kv + row_n + ps - 1) // ps
    part = row_kv // ps
    own_at = owned.gather(1, part.clamp(max=P - 1)[:, None])[:, 0]
    first = torch.arange(G * W, device=DEV) % W == 0
    forks = ~first & (row_kv % ps != 0) & (row_n > 0) & (own_at < 0) if not shared else torch.zeros(G * W, dtype=torch.bool, device=DEV)
    needs = torch.where(first | torch.full_like(first, not shared), want - have + forks.long(), 0)
    needs = torch.where(row_n > 0, needs, 0)
    per = 1 if shared else W
    start = per * (n.cumsum(0) - n)
    fits_table = (kv + n <= P * ps) & (start + per * n <= T)
    need = torch.where(fits_table, needs.view(G, W).sum(1), 0)
    served = (q >= 0) & fits_table & ((need == 0) | (need.cumsum(0) <= top))
    row_served = served.repeat_interleave(W)
    taken = torch.where(served, need, 0).sum()
    # the k-th page taken is the k-th from the top, blocks ascending within a row
    lo = torch.where(forks, part, have)
    fresh = row_served[:, None] & (row_n > 0)[:, None] & (j >= lo[:, None]) & (j < want[:, None])
    takes = fresh & (first | torch.full_like(first, not shared))[:, None]
    rank = takes.flatten().long().cumsum(0) - 1
    page = free[(top - 1 - rank).clamp(0, free.numel() - 1)].view(G * W, P)
    old = tables.gather(1, part.clamp(max=P - 1)[:, None])[:, 0]
    if shared:
        page = page.view(G, W, P)[:, :1].expand(G, W, P).reshape(G * W, P)
    tables.copy_(torch.where(fresh, page, tables))
    owned.copy_(torch.where(takes, page, torch.where(fresh, -1, owned)))
    forks = forks & row_served
    got = page.gather(1, part.clamp(max=P - 1)[:, None])[:, 0]
    copies = torch.where(forks[:, None], torch.stack([old, got, row_kv % ps], 1), -1)
    # rows: the tokens of a group (of each of its beams), one after another
    granted = torch.where(served, n, 0)
    starts = start if shared else (start[:, None] + n[:, None] * torch.arange(W, device=DEV)).flatten()
    row_q = n if shared else row_n
    t = torch.arange(T, device=DEV)
    r = torch.searchsorted(starts + row_q, t, right=True)
    inside = r < starts.numel()
    r = r.clamp(max=starts.numel() - 1)
    g = r if shared else r // W
    pos = kv[g] + t - starts[r]
    ok = inside & served[g]
    slot = tables[r * W if shared else r, (pos // ps).clamp(max=P - 1)].long() * ps + pos % ps
    i32 = torch.int32
    return [starts.to(i32), granted.to(i32), torch.where(q < 0, 0, kv + granted).to(i32), torch.where(ok, slot, -1), torch.where(ok, pos, -1).to(i32),
            copies.to(i32), (top - taken).to(i32), ((q >= 0) & ~served).sum(0, keepdim=True).to(i32), tables, owned, free]


# ---------------------------------------------------------------------------------------------
# write: keys and values into their slots
# ---------------------------------------------------------------------------------------------
def _prepare_write(c, gen, host):
    T, H, D, ps, dt = c["tokens"], c["kv_heads"], c["dim"], c["page"], DTYPES[c["dtype"]]
    pages = _up(T, ps) + 3
    qkv = _normal((T, 3, H, D), dt, gen)
    slots = torch.randperm(pages, generator=host)[:, None] * ps + torch.arange(ps)      # pages in any order, the tokens of a page one after another
    slots = slots.flatten()[:T].clone()
    slots[torch.rand(T, generator=host) < c["skipped"]] = -1
    cache = torch.zeros(2, pages, H, ps, D, dtype=dt, device=DEV)
    return {"case": c, "k": qkv[:, 1], "v": qkv[:, 2], "key_cache": cache[0], "value_cache": cache[1], "slots": slots.to(DEV)}


def _own_write(s):
    from mmf_amd import decoding
    decoding.write_pages(s["k"], s["v"], s["key_cache"], s["value_cache"], s["slots"])
    return [s["key_cache"], s["value_cache"]]


def _plain_write(s):
    kc, vc, slots = s["key_cache"], s["value_cache"], s["slots"]
    pages, H, ps, D = kc.shape
    # the token of each slot, if any: rows that are left out meet in a cell behind the last
    token = torch.full((pages * ps + 1,), -1, dtype=torch.int64, device=DEV)
    token[torch.where(slots >= 0, slots, pages * ps)] = torch.arange(slots.numel(), device=DEV)
    token = token[:-1].view(pages, 1, ps, 1)
    for x, cache in ((s["k"], kc), (s["v"], vc)):
        new = x[token.clamp(min=0).view(pages, ps)].transpose(1, 2)
        cache.copy_(torch.where(token >= 0, new, cache))
    return [kc, vc]


# ---------------------------------------------------------------------------------------------
# attend: new tokens over the pages of their request
# ---------------------------------------------------------------------------------------------
def _prepare_attend(c, gen, host):
    ctx, new = _lengths(c)
    W, ps, dt, D = c["beams"], c["page"], DTYPES[c["dtype"]], c["dim"]
    kv = [n + m for n, m in zip(ctx, new)]
    blocks = _up(max(kv), ps) + 1
    t, _, _ = _tables(dict(c, _spare=5), kv, [max(0, n - c["tail"]) for n in ctx], blocks, host)
    pages = int(t.max()) + 6
    t = t.to(DEV)
    cache = [_normal((pages, c["kv_heads"], ps, D), dt, gen) for _ in range(2)]
    # what no token has written yet holds anything
    row_kv = _i32(kv).repeat_interleave(W)
    written = torch.zeros(pages, ps, dtype=torch.bool, device=DEV)
    at = torch.arange(blocks * ps, device=DEV).view(blocks, ps)
    live = at[None] < row_kv[:, None, None]
    written[t.clamp(min=0)[:, :, None].expand_as(live)[live].long(), (at % ps).expand_as(live)[live]] = True
    for x in cache:
        x.masked_fill_(~written[:, None, :, None], float("nan"))
    T = W * sum(new)
    qkv = _normal((T, c["heads"] + 2 * c["kv_heads"], D), dt, gen, 1.5)
    row_new = [m for m in new for _ in range(W)]
    start = [0]
    for m in row_new:
        start.append(start[-1] + m)
    return {"case": c, "q": qkv[:, :c["heads"]], "key_cache": cache[0], "value_cache": cache[1], "tables": t, "kv_lens": _i32(kv), "q_start": _i32(start[:-1]),
            "q_lens": _i32(new), "host": (start, row_new, [n for n in kv for _ in range(W)]), "max_q": max(new)}


def _own_attend(s):
    from mmf_amd import decoding
    c = s["case"]
    return decoding.attend_pages(s["q"], s["key_cache"], s["value_cache"], s["tables"], s["kv_lens"], s["q_start"], s["q_lens"], max_q=s["max_q"],
                                 beams=c["beams"], causal=c["causal"])


def _plain_attend(s):
    c = s["case"]
    Hq, Hk, D, ps = c["heads"], c["kv_heads"], c["dim"], c["page"]
    start, row_new, row_kv = s["host"]
    out = torch.empty(s["q"].shape, dtype=s["q"].dtype, device=DEV)
    r0 = 0
    while r0 < len(row_new):           # as many rows at once as their scores fit 2 GiB
        r1, Q, L = r0 + 1, row_new[r0], row_kv[r0]
        while r1 < len(row_new):
            q1, l1 = max(Q, row_new[r1]), max(L, row_kv[r1])
            if (r1 + 1 - r0) * l1 * max(Hq * q1, Hk * D) > 1 << 29:
                break
            r1, Q, L = r1 + 1, q1, l1
        n, a, b = r1 - r0, start[r0], start[r1]
        if b > a:
            B = _up(L, ps)
            lens = s["kv_lens"].repeat_interleave(c["beams"])[r0:r1]
            news = s["q_lens"].repeat_interleave(c["beams"])[r0:r1]
            pages = s["tables"][r0:r1, :B].clamp(min=0).long()
            at = torch.arange(B * ps, device=DEV)
            seen = at < lens[:, None]
            k = s["key_cache"][pages].transpose(2, 3).reshape(n, B * ps, Hk, D).float().masked_fill(~seen[:, :, None, None], 0).transpose(1, 2).contiguous()
            v = s["value_cache"][pages].transpose(2, 3).reshape(n, B * ps, Hk, D).float().masked_fill(~seen[:, :, None, None], 0).transpose(1, 2).contiguous()
            i = torch.arange(Q, device=DEV)
            idx = (s["q_start"][r0:r1, None] + i).clamp(max=b - 1).long()
            q = s["q"][idx].float().view(n, Q, Hk, Hq // Hk, D).permute(0, 2, 3, 1, 4).reshape(n, Hk, -1, D)
            sc = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(D ** -0.5).view(n, Hk, Hq // Hk, Q, B * ps)
            see = seen[:, None, :].expand(n, Q, B * ps)
            if c["causal"]:
                see = see & (at[None, None] <= (lens - news)[:, None, None] + i[None, :, None])
            sc.masked_fill_(~see[:, None, None], float("-inf"))
            sc -= sc.amax(-1, keepdim=True).clamp(min=-1e30)
            sc.exp_()
            den = sc.sum(-1, keepdim=True)
            o = torch.matmul(sc.view(n, Hk, -1, B * ps), v).view(n, Hk, Hq // Hk, Q, D) / den.clamp(min=1e-30)
            o = o.permute(0, 3, 1, 2, 4).reshape(n, Q, Hq, D)
            live = i < news[:, None]
            out[a:b] = _packed(o, live, row_new[r0:r1], b - a).to(out.dtype)
        r0 = r1
    return out


def _packed(o, live, counts, total):
    """The live rows of [n, Q, ...] one after another, their number known on the host."""
    n, Q = live.shape
    if n * Q == total:
        return o.reshape(total, *o.shape[2:])
    order = torch.sort(torch.where(live, 0, 1).flatten(), stable=True).indices[:total]
    return o.reshape(n * Q, *o.shape[2:])[order]


def _exact_attend(s):
    c = s["case"]
    ps, group = c["page"], c["heads"] // c["kv_heads"]
    start, row_new, row_kv = s["host"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for r, (m, n) in enumerate(zip(row_new, row_kv)):
        if m == 0:
            continue
        slot = torch.arange(n, device=DEV)
        page = s["tables"][r].long()[slot // ps]
        keys, values = s["key_cache"][page, :, slot % ps], s["value_cache"][page, :, slot % ps]       # [n, kv heads, dim]
        hidden = slot[None, :] > (n - m) + torch.arange(m, device=DEV)[:, None]
        for h in range(c["heads"]):
            z = s["q"][start[r]:start[r] + m, h].double() @ keys[:, h // group].double().t() / math.sqrt(c["dim"])
            if c["causal"]:
                z[hidden] = -math.inf
            out[start[r]:start[r] + m, h] = torch.softmax(z, 1) @ values[:, h // group].double()
    return out


# ---------------------------------------------------------------------------------------------
# select: the best continuations of each group
# ---------------------------------------------------------------------------------------------
def _prepare_select(c, gen, host):
    G, W, V = c["groups"], c["beams"], c["vocab"]
    logits = _normal((G * W, V), torch.float32, gen, 2.5)
    if c["masked"]:                    # padding of the copied tokens: an additive mask, as the scores carry it
        cut = V - (torch.rand(G, generator=gen, device=DEV) * c["masked"]).long()
        logits += torch.where(torch.arange(V, device=DEV) >= cut.repeat_interleave(W)[:, None], -10000.0, 0.0)
    at = c["length"] // 2
    done = torch.rand(G, W, generator=gen, device=DEV) < c["done"]
    scores = -5.0 * torch.rand(G, W, generator=gen, device=DEV).cumsum(1)
    if c["first"]:                     # one live beam so far
        done = torch.zeros_like(done)
        scores = torch.where(torch.arange(W, device=DEV) == 0, 0.0, float("-inf")).expand(G, W).contiguous()
    history = torch.randint(0, V, (G, W, c["length"]), generator=gen, device=DEV)
    return {"case": c, "logits": logits.to(DTYPES[c["dtype"]]), "scores": scores, "done": done, "history": history, "step": at}


def _own_select(s):
    from mmf_amd import decoding
    b = decoding.select_beams(s["logits"], s["scores"], s["done"], eos=EOS, history=s["history"], step=s["step"])
    return [b.scores, b.parents, b.tokens, b.finished, b.history]


def _plain_select(s):
    G, W = s["scores"].shape
    x = s["logits"].double()           # candidates of different beams lie as near to each other as chance will have it
    V = x.shape[1]
    top = x.amax(1, keepdim=True)
    lse = (x - top).exp_().sum(1, keepdim=True).log_() + top
    x -= lse
    cand = s["scores"].double().view(G, W, 1) + x.view(G, W, V)
    only = torch.where(torch.arange(V, device=DEV) == EOS, s["scores"].double()[:, :, None], float("-inf"))
    cand = torch.where(s["done"][:, :, None], only, cand).view(G, W * V)
    score, at = torch.sort(cand, dim=1, descending=True, stable=True)
    score, at = score[:, :W], at[:, :W]
    parents, tokens = at // V, at % V
    finished = s["done"].gather(1, parents) | (tokens == EOS)
    history = s["history"].gather(1, parents[:, :, None].expand_as(s["history"]))
    history[:, :, s["step"]] = tokens
    return [score.float(), parents, tokens, finished, history]


def _exact_select(s):
    G, W = s["scores"].shape
    out = torch.empty(G, W, dtype=torch.float64)
    done, prior = s["done"].tolist(), s["scores"].double().tolist()
    for g in range(G):
        best = []
        for w in range(W):
            if done[g][w]:
                best.append(prior[g][w])
            elif prior[g][w] > -math.inf:
                best += (prior[g][w] + torch.topk(torch.log_softmax(s["logits"][g * W + w].double(), 0), min(W, s["logits"].shape[1])).values).tolist()
        out[g] = torch.tensor(sorted(best, reverse=True)[:W], dtype=torch.float64)
    return [out, None, None, None, None]


# ---------------------------------------------------------------------------------------------
# reorder: tables and shared pages after a selection
# ---------------------------------------------------------------------------------------------
def _parents(c):
    rng = random.Random(c["shape"] + 2)
    return [[min(c["beams"] - 1, int(rng.expovariate(1.0))) if rng.random() < 0.7 else w for w in range(c["beams"])] for _ in range(c["groups"])]


def _prepare_reorder(c, gen, host):
    ctx, _ = _lengths(c)
    blocks = _up(max(ctx), c["page"]) + 2
    t, _, _ = _tables(dict(c, _spare=3), ctx, [max(0, n - c["tail"]) for n in ctx], blocks, host)
    pages = int(t.max()) + 4
    cache = _normal((c["layers"], 2, pages, c["kv_heads"], c["page"], c["dim"]), DTYPES[c["dtype"]], gen)
    return {"case": c, "parents": torch.tensor(_parents(c), device=DEV), "kv_lens": _i32(ctx), "tables": t.to(DEV), "cache": cache}


def _own_reorder(s):
    from mmf_amd import decoding
    tables = decoding.reorder_pages(s["parents"], s["kv_lens"], s["tables"], s["cache"])
    return [tables, s["cache"]]


def _plain_reorder(s):
    c = s["case"]
    W, ps = c["beams"], c["page"]
    parents, cache = s["parents"], s["cache"]
    G = parents.shape[0]
    t = s["tables"].view(G, W, -1)
    w = torch.arange(W, device=DEV)
    new = t.gather(1, parents[:, :, None].expand_as(t))
    # the first child of a beam goes on in its page; the others take, in order, the pages of the beams without children
    same = parents[:, :, None] == parents[:, None, :]
    extra = (same & (w[None, :] < w[:, None])).any(2)
    childless = ~(parents[:, None, :] == w[:, None]).any(2)
    give = torch.sort((~childless).long(), dim=1, stable=True).indices         # beams without children first
    take = (extra.long().cumsum(1) - 1).clamp(min=0)
    part, rest = s["kv_lens"].long() // ps, s["kv_lens"].long() % ps
    at = part.clamp(max=t.shape[2] - 1)[:, None, None].expand(G, W, 1)
    last = t.gather(2, at)[:, :, 0]
    src = last.gather(1, parents)
    dst = torch.where(extra & (rest > 0)[:, None], last.gather(1, give.gather(1, take)), src)
    new.scatter_(2, at, torch.where((rest > 0)[:, None], dst, new.gather(2, at)[:, :, 0])[:, :, None])
    src = torch.where((rest > 0)[:, None], src, 0).flatten().long()
    dst = torch.where((rest > 0)[:, None], dst, 0).flatten().long()
    fresh = torch.arange(ps, device=DEV) < rest.repeat_interleave(W)[:, None]
    moved = torch.where(fresh[None, None, :, None, :, None], cache[:, :, src], cache[:, :, dst])
    cache[:, :, dst] = moved
    return [new.reshape(s["tables"].shape), cache]


# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "attend":
        return _exact_attend(prepare(case, seed))
    if case["op"] == "select":
        return _exact_select(prepare(case, seed))
    return None                        # whole numbers and moved values: nothing is computed that could be off


def work(case):
    c, op = case, case["op"]
    if op == "plan":
        ctx, new, _, rows, need = _plan_numbers(c)
        W = c["beams"]
        fresh = sum(W * (_up(n + max(0, m), c["page"]) - _up(n, c["page"])) for n, m in zip(ctx, new))
        return {"bytes": 16 * c["groups"] + 16 * c["groups"] * W + 12 * rows + 4 * need + 8 * fresh, "flops": 0}
    if op == "write":
        size = DTYPES[c["dtype"]].itemsize
        return {"bytes": 8 * c["tokens"] + 4 * size * int(c["tokens"] * (1 - c["skipped"])) * c["kv_heads"] * c["dim"], "flops": 0}
    if op == "attend":
        size = DTYPES[c["dtype"]].itemsize
        ctx, new = _lengths(c)
        tokens = pairs = queries = 0
        for n, m in zip(ctx, new):
            b, shared = _owners(n + m, max(0, n - c["tail"]), c["beams"], c["page"])
            tokens += shared * c["page"] + c["beams"] * (n + m - shared * c["page"]) if b > shared else n + m
            pairs += c["beams"] * (m * n + (m * (m + 1) // 2 if c["causal"] else m * m))
            queries += c["beams"] * m
        return {"bytes": size * (2 * tokens * c["kv_heads"] * c["dim"] + 2 * queries * c["heads"] * c["dim"]), "flops": 4 * pairs * c["heads"] * c["dim"]}
    if op == "select":
        n = c["groups"] * c["beams"]
        return {"bytes": DTYPES[c["dtype"]].itemsize * n * c["vocab"] + n * (16 * c["length"] + 40), "flops": 3 * n * c["vocab"]}
    ctx, _ = _lengths(c)
    size = DTYPES[c["dtype"]].itemsize
    moved = sum((c["beams"] - len(set(p))) * (n % c["page"]) for n, p in zip(ctx, _parents(c)))
    return {"bytes": 8 * c["beams"] * sum(_up(n, c["page"]) for n in ctx) + 4 * size * moved * c["layers"] * c["kv_heads"] * c["dim"], "flops": 0}
