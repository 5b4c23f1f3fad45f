"""The operators of cached decoding (mmf_amd/decoding.py) against their plain restatements in 64 bits (tests/decoding_oracle.py): whole numbers have to be equal,
computed values lie within bounds derived from the roundings the kernels make."""
import random

import pytest
import torch

from tests import decoding_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = torch.int32


def D():
    from mmf_amd import decoding
    return decoding


def i32(x):
    return torch.tensor(x, dtype=I32, device=DEV)


@pytest.fixture(autouse=True)
def no_index_error():
    from mmf_amd import _native as nat
    nat.take_index_error()
    yield
    assert not nat.take_index_error()


# ---------------------------------------------------------------------------------------------
# plan
# ---------------------------------------------------------------------------------------------
def plan_both(q_lens, kv_lens, tables, owned, free, top, page, rows, beams, shared):
    t, o, f = i32(tables), i32(owned), i32(free)
    p = D().plan_pages(i32(q_lens), i32(kv_lens), t, o, f, i32([top]), page_size=page, rows=rows, beams=beams, shared=shared)
    tables, owned, free = [list(r) for r in tables], [list(r) for r in owned], list(free)
    want = O.plan(q_lens, kv_lens, tables, owned, free, top, page, rows, beams, shared)
    got = [p.q_start, p.q_lens, p.kv_lens, p.slots, p.positions, p.copies, p.free_top, p.refused]
    for name, g, w in zip(p._fields, got, want):
        w = [w] if isinstance(w, int) else w
        if name == "q_start":
            w = [min(x, rows) for x in w]
        assert g.tolist() == w, name
    assert t.tolist() == tables and o.tolist() == owned and f.tolist() == free
    return want, tables, owned, free


@pytest.mark.parametrize("page,beams,shared,groups", [(1, 1, False, 1), (16, 1, True, 7), (16, 5, False, 9), (16, 5, True, 9), (8, 32, False, 3), (64, 2, True, 1500), (1024, 3, False, 40), (64, 1, True, 2), (64, 5, True, 2), (64, 2, False, 2),
                                                      (64, 32, True, 100),
                                                      (32, 1, False, 2100)])
def test_plan_grows_releases_and_waits_like_the_plain_form(page, beams, shared, groups):
    """Five steps of one pool: prompts, single tokens, chunks, finished groups, more tokens than pages, tables or rows hold."""
    rng = random.Random(page * 100 + beams)
    P = 6
    pages = groups * beams * 3 + 1
    tables, owned = [[-1] * P for _ in range(groups * beams)], [[-1] * P for _ in range(groups * beams)]
    free = rng.sample(range(pages), pages)
    top, kv = pages, [0] * groups
    for step in range(5):
        sh = shared if step else True                      # the first step is a prompt: with beams, the next one gives rows pages of their own
        q = [rng.choice([0, 1, 1, 2, page, page * 2 + 1, rng.randrange(page * P + 2)]) for _ in range(groups)]
        q = [-1 if step > 1 and rng.random() < 0.2 else n for n in q]
        per = 1 if sh else beams
        rows = max(1, sum(per * max(n, 0) for n in q) - rng.choice([0, 0, 3])) + rng.choice([0, 5])
        want, tables, owned, free = plan_both(q, kv, tables, owned, free, top, page, rows, beams, sh)
        kv, top = want[2], want[6]


def test_plan_results_in_place_and_no_pages_at_all():
    free_top, kv = i32([2]), i32([3, 8, 0])
    t, o = torch.full((3, 4), -1, dtype=I32, device=DEV), torch.full((3, 4), -1, dtype=I32, device=DEV)
    t[0, 0], t[1, :2] = 9, i32([7, 8]); o.copy_(t)
    plan = D().plan_pages(i32([1, 1, 0]), kv, t, o, i32([4, 5, 6]), free_top, page_size=4, rows=4)
    same = plan._replace(kv_lens=kv, free_top=free_top)
    D().plan_pages(i32([1, 1, 0]), kv, t, o, i32([4, 5, 6]), free_top, page_size=4, rows=4, out=same)
    assert kv.tolist() == [4, 9, 0] and free_top.tolist() == [1] and plan.slots.tolist() == [39, 20, -1, -1]
    # nothing is free: the token inside its page is planned, the others wait
    plan = D().plan_pages(i32([1, 4, 1]), i32([2, 8, 0]), t, o, i32([4, 5, 6]), i32([0]), page_size=4, rows=9)
    assert plan.q_lens.tolist() == [1, 0, 0] and plan.refused.tolist() == [2] and plan.slots.tolist() == [38] + [-1] * 8


# ---------------------------------------------------------------------------------------------
# write
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,heads,dim,page,offset", [(1, 1, 64, 16, 0), (77, 12, 64, 16, 0), (300, 5, 128, 1, 0), (33, 2, 64, 8, 1), (40, 3, 128, 64, 0)])
def test_write_moves_every_row_to_its_slot(dtype, tokens, heads, dim, page, offset):
    g = torch.Generator().manual_seed(tokens)
    pages = -(-tokens // page) + 2
    flat = torch.randn(tokens * 3 * heads * dim + offset, generator=g).to(dtype).to(DEV)
    qkv = flat[offset:].view(tokens, 3, heads, dim)             # offset 1: rows that start on no 16 bytes
    caches = torch.randn(2, pages, heads, page, dim, generator=g).to(dtype).to(DEV)
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots[torch.rand(tokens, generator=g) < 0.2] = -1
    want = caches.clone().cpu()
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            want[0, s // page, :, s % page], want[1, s // page, :, s % page] = qkv[t, 1].cpu(), qkv[t, 2].cpu()
    D().write_pages(qkv[:, 1], qkv[:, 2], caches[0], caches[1], slots.to(DEV))
    assert torch.equal(caches.cpu(), want)


def test_write_into_a_token_major_pool_and_nothing_to_write():
    x = torch.randn(6, 2, 64, device=DEV)
    pool = torch.zeros(2, 3, 4, 2, 64, device=DEV).transpose(2, 3)            # [pages, page_size, heads, dim] memory seen as [pages, heads, page_size, dim]
    D().write_pages(x, -x, pool[0], pool[1], torch.tensor([0, 11, 5, -1, 6, -7], device=DEV))
    for t, s in ((0, 0), (1, 11), (2, 5), (4, 6)):
        assert torch.equal(pool[0, s // 4, :, s % 4], x[t]) and torch.equal(pool[1, s // 4, :, s % 4], -x[t])
    assert int((pool[0] != 0).any(-1).sum()) == 8
    D().write_pages(x[:0], x[:0], pool[0], pool[1], torch.empty(0, dtype=torch.int64, device=DEV))


# ---------------------------------------------------------------------------------------------
# attend
# ---------------------------------------------------------------------------------------------
def attend_case(kv, new, *, beams=1, heads=4, kv_heads=4, dim=64, page=16, dtype=torch.bfloat16, shared=0, seed=0, spread=1.5, token_major=False, gaps=0):
    """Caches with NaN where no token lives, tables with -1 behind the last block, `gaps` rows between the requests' tokens."""
    g = torch.Generator().manual_seed(seed + 7 * sum(kv))
    R = len(kv) * beams
    blocks = max(1, max(-(-n // page) for n in kv)) + 1
    tables = torch.full((R, blocks), -1, dtype=I32)
    need = R * blocks + 3
    pages = torch.randperm(need, generator=g, dtype=I32)
    at = 0
    for r in range(R):
        b = -(-kv[r // beams] // page)
        s = shared // page if r % beams else 0
        s = min(s, b)
        if s:
            tables[r, :s] = tables[r - r % beams, :s]
        tables[r, s:b] = pages[at:at + b - s]
        at += b - s
    shape = (need, page, kv_heads, dim) if token_major else (need, kv_heads, page, dim)
    caches = torch.full((2,) + shape, float("nan"))
    view = caches.transpose(2, 3) if token_major else caches
    for r in range(R):
        for j in range(-(-kv[r // beams] // page)):
            n = min(page, kv[r // beams] - j * page)
            view[:, int(tables[r, j]), :, :n] = torch.randn(2, kv_heads, n, dim, generator=g)
    row_new = [n for n in new for _ in range(beams)]
    start, t = [], 0
    for n in row_new:
        start.append(t)
        t += n + gaps
    q = (torch.randn(t + 2, heads + 2, dim, generator=g) * spread).to(dtype).to(DEV)[:, :heads]
    caches = caches.to(dtype).to(DEV)
    view = caches.transpose(2, 3) if token_major else caches
    return dict(q=q, key_cache=view[0], value_cache=view[1], tables=tables.to(DEV), kv_lens=i32(kv), q_start=i32(start), q_lens=i32(new))


def attend_check(c, beams=1, causal=True, scale=None, max_q=None, out=None):
    dt, dim = c["q"].dtype, c["q"].shape[2]
    sc = dim ** -0.5 if scale is None else scale
    fill = out if out is not None else torch.full(c["q"].shape, 7.0, dtype=dt, device=DEV)
    before = fill.clone()
    got = D().attend_pages(*(c[k] for k in ("q", "key_cache", "value_cache", "tables", "kv_lens", "q_start", "q_lens")), max_q=max_q or max(1, int(c["q_lens"].max())),
                           beams=beams, causal=causal, scale=scale, out=fill)
    want, mag, reach, named = O.attend(*(c[k] for k in ("q", "key_cache", "value_cache", "tables", "kv_lens", "q_start", "q_lens")), beams, causal, sc)
    # A score s = scale * sum_e q_e k_e in 32 bits is off by at most (dim + 4) 2^-24 scale sum |q_e k_e| (dim products and sums, the scale, the difference to the maximum,
    # the factor log2 e), its exponential by another 4 units; `reach` bounds scale sum |q k| + |s - max|.  Sums of n terms add n 2^-24 at most, twice (numerator and
    # denominator).  Relative errors of the probabilities reach the output through mag = sum p |v|.
    n = int(c["kv_lens"].max())
    rel = 2.0 ** -24 * ((dim + 4) * reach + 2 * n + 16)
    tol = 2.2 * rel[..., None] * mag
    if dt == torch.bfloat16:
        tol = 1.01 * (tol + 2.0 ** -8 * mag + 2.0 ** -8 * want.abs())         # each probability rounded to bf16 once, the output once
    else:
        tol = tol + 2.0 ** -23 * want.abs()
    err = (got.double().cpu() - want).abs()
    assert bool(torch.isfinite(got[named.to(DEV)].float()).all())
    worst = float((err - tol - 1e-30)[named].max()) if bool(named.any()) else 0.0
    assert worst <= 0, "off by %g beyond its bound (largest error %g)" % (worst, float(err[named].max()))
    assert torch.equal(got[~named.to(DEV)], before[~named.to(DEV)])          # rows no request names
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(1, 1, 64, 1), (12, 12, 64, 16), (8, 2, 128, 8), (8, 1, 64, 64), (6, 2, 128, 1024), (40, 2, 64, 32)])
def test_single_tokens(dtype, heads, kv_heads, dim, page):
    """One new token each, from the first of a sequence to lengths around the ends of pages and tiles."""
    kv = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 300]
    attend_check(attend_case(kv, [1] * len(kv), heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(3, 3, 64, 16), (4, 1, 128, 8), (4, 2, 64, 128)])
def test_chunks(dtype, causal, heads, kv_heads, dim, page):
    """Chunks of every kind of length, behind nothing and behind a cache, and requests without a new token."""
    kv = [5, 1, 33, 64, 97, 130, 200, 40, 161]
    new = [5, 1, 2, 64, 33, 65, 100, 0, 31]
    attend_check(attend_case(kv, new, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype), causal=causal)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("beams,shared,new", [(5, 96, 1), (2, 16, 1), (8, 0, 1), (32, 64, 1), (3, 80, 4)])
def test_beams_share_pages(dtype, beams, shared, new):
    attend_check(attend_case([130, 97, 16, new], [new] * 4, beams=beams, heads=4, kv_heads=2, dtype=dtype, shared=shared), beams=beams)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_long_cache_few_rows(dtype):
    attend_check(attend_case([4097, 9000], [1, 2], heads=4, kv_heads=2, dim=128, dtype=dtype))
    attend_check(attend_case([5000], [1], heads=1, kv_heads=1, dim=64, page=64, dtype=dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("beams,kv,new", [(1, [150, 1, 512], 1), (4, [150, 40], 1), (1, [150, 511, 70], 40), (1, [150, 513, 70], 1), (1, [100, 900, 70], 40), (4, [150, 700], 1)])
def test_requests_in_tables_with_room_for_long_ones(dtype, beams, kv, new):
    """Nothing is split where no request is long, whatever the tables have room for; one long request among short ones is."""
    c = attend_case(kv, [new if n >= new else n for n in kv], beams=beams, heads=4, kv_heads=2, dim=64, dtype=dtype)
    c["tables"] = torch.cat([c["tables"], torch.full((len(kv) * beams, 200), -1, dtype=I32, device=DEV)], 1)
    attend_check(c, beams=beams)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_between_the_requests_and_a_token_major_pool(dtype):
    attend_check(attend_case([40, 3, 70], [7, 3, 40], heads=4, kv_heads=2, dim=64, dtype=dtype, token_major=True, gaps=3))
    attend_check(attend_case([40, 3, 70], [1, 1, 1], heads=4, kv_heads=2, dim=128, dtype=dtype, token_major=True, gaps=2))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tokens_that_see_no_key_give_zeros(dtype):
    """More new tokens than keys (a group that had to wait): the first of them see nothing; no key at all: none does."""
    c = attend_case([4, 0, 20], [6, 3, 2], heads=2, kv_heads=2, dtype=dtype)
    out = attend_check(c)
    assert float(out[:2].abs().max()) == 0 and float(out[6:9].abs().max()) == 0
    out = attend_check(c, causal=False)
    assert float(out[6:9].abs().max()) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 40])
def test_large_scores_and_values(dtype, new):
    """Scores in the hundreds (a softmax of one key), keys and values near the ends of the range, scale 0 and a negative scale."""
    c = attend_case([200, 77], [new, new], heads=4, kv_heads=4, dtype=dtype, spread=60.0)
    attend_check(c)
    attend_check(c, scale=0.0)
    attend_check(c, scale=-0.125)
    for x in ("key_cache", "value_cache"):
        c[x] = c[x] * 1e30
    c["q"] = c["q"] * 1e-30
    attend_check(c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kv,new,beams,shared,heads,dim", [([70, 33, 90], [40, 33, 7], 1, 0, 4, 64), ([70, 200], [64, 130], 1, 0, 8, 128), ([40, 70, 64], [4, 2, 1], 1, 0, 4, 128),
                                                          ([70, 50], [1, 1], 4, 48, 2, 64), ([100], [3], 2, 32, 4, 64), ([3000], [50], 1, 0, 2, 64), ([3000], [2], 1, 0, 2, 128)])
def test_infinities_and_nan_stay_with_the_rows_that_see_them(dtype, kv, new, beams, shared, heads, dim):
    """Values (of later tokens in the chunk, of another beam, of an early key) that are infinite or no number: a row that sees one has it in its column, every other output
    is what it was, bit for bit.  A key that is no number: all of a row that sees it, nothing of the others."""
    c = attend_case(kv, new, beams=beams, heads=heads, kv_heads=2, dim=dim, dtype=dtype, shared=shared)
    good = attend_check(c, beams=beams)

    def spot(r, key):
        return int(c["tables"][r, key // 16]), key % 16
    for cache in ("value_cache", "key_cache"):
        bad = dict(c, **{cache: c[cache].clone()})
        for r in range(len(kv) * beams):
            n, m = kv[r // beams], new[r // beams]
            for k, (key, col, x) in enumerate([(n - 1, 5, float("nan")), (n - 1, 37, float("inf")), (n - 1 - m // 2, 6, float("-inf")), (n - 1 - m // 2, 37, float("-inf")),
                                               (max(0, n - m) // 2 + 1, 60, float("inf")), (n - 1 - m // 3, 5, float("inf"))]):
                if cache == "key_cache" and k > 2:
                    continue
                page, pos = spot(r, key)
                bad[cache][page, r % 2, pos, col] = float("nan") if cache == "key_cache" else x
        names = ("q", "key_cache", "value_cache", "tables", "kv_lens", "q_start", "q_lens")
        out = torch.full_like(good, 7.0)
        got = D().attend_pages(*(bad[k] for k in names), max_q=max(new), beams=beams, out=out)
        want, _, _, named = O.attend(*(bad[k] for k in names), beams, True, dim ** -0.5)
        g = got.double().cpu()
        fine = torch.isfinite(want) & named[:, None, None]
        assert bool(fine.any()) and not bool(torch.isfinite(want[named]).all())
        assert torch.equal(g[fine], good.double().cpu()[fine])
        odd = ~torch.isfinite(want) & named[:, None, None]
        assert torch.equal(torch.nan_to_num(g[odd], 9.0, 10.0, -10.0), torch.nan_to_num(want[odd], 9.0, 10.0, -10.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_max_q_larger_than_any_request_and_out_in_place_of_q(dtype):
    c = attend_case([90, 40], [9, 20], heads=4, kv_heads=2, dtype=dtype)
    a = attend_check(c, max_q=500)
    q = c["q"].clone()
    out = D().attend_pages(q, c["key_cache"], c["value_cache"], c["tables"], c["kv_lens"], c["q_start"], c["q_lens"], max_q=20, out=q)
    assert torch.equal(out[:29], a[:29])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page", [4, 16, 64])
@pytest.mark.parametrize("new", [1, 40])
def test_pages_outside_the_pool_read_as_zeros(dtype, page, new):
    from mmf_amd import _native as nat
    c = attend_case([150, 90], [new, new], heads=4, kv_heads=2, page=page, dtype=dtype)
    empty = torch.cat([torch.zeros_like(c["key_cache"][:1]), c["key_cache"]]), torch.cat([torch.zeros_like(c["value_cache"][:1]), c["value_cache"]])
    want_t, t = c["tables"] + 1, c["tables"] + 1
    for block in (0, 40 // page, 149 // page):
        want_t[0, block] = 0
    rest = dict(kv_lens=c["kv_lens"], q_start=c["q_start"], q_lens=c["q_lens"], max_q=new)
    want = D().attend_pages(c["q"], *empty, want_t, **rest)
    for bad in (-1, -2 ** 31, empty[0].shape[0], 2 ** 31 - 1):
        for block in (0, 40 // page, 149 // page):
            t[0, block] = bad
        nat.take_index_error()
        got = D().attend_pages(c["q"], *empty, t, **rest)
        assert nat.take_index_error()
        assert torch.equal(got[:2 * new], want[:2 * new])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_more_query_heads_on_a_key_head_than_a_step_has_rows(dtype):
    attend_check(attend_case([70, 1, 33], [1, 1, 1], heads=64, kv_heads=1, dim=64, dtype=dtype))
    attend_check(attend_case([70, 40], [3, 2], heads=66, kv_heads=2, dim=128, dtype=dtype))


def test_pages_outside_the_pool_are_reported_and_other_requests_do_not_notice():
    from mmf_amd import _native as nat
    for new, dtype in ((1, torch.bfloat16), (40, torch.bfloat16), (1, torch.float32), (40, torch.float32)):
        c = attend_case([64, 90], [new, new], heads=2, kv_heads=2, page=16, dtype=dtype)
        good = attend_check(c)
        for bad in (-3, 10 ** 6):
            t = c["tables"].clone()
            t[0, 3] = bad
            got = D().attend_pages(c["q"], c["key_cache"], c["value_cache"], t, c["kv_lens"], c["q_start"], c["q_lens"], max_q=new)
            assert nat.take_index_error()
            assert torch.equal(got[new:2 * new], good[new:2 * new])
        # rows outside the token buffer, more new tokens than max_q: reported, nothing is read or written out of range
        D().attend_pages(c["q"], c["key_cache"], c["value_cache"], c["tables"], c["kv_lens"], i32([10 ** 7, 0]), c["q_lens"], max_q=new)
        assert nat.take_index_error()
        if new > 1:
            D().attend_pages(c["q"], c["key_cache"], c["value_cache"], c["tables"], c["kv_lens"], c["q_start"], c["q_lens"], max_q=1)
            assert nat.take_index_error()


# ---------------------------------------------------------------------------------------------
# select
# ---------------------------------------------------------------------------------------------
def select_check(logits, scores, finished, eos, history=None, step=0, gap=1e-4):
    want = O.select(logits, scores, finished, eos)
    assert want[4] > gap, "the case does not decide its order: %g" % want[4]
    got = D().select_beams(logits, scores, finished, eos=eos, history=history, step=step)
    assert torch.equal(got.parents.cpu(), want[1]) and torch.equal(got.tokens.cpu(), want[2]) and torch.equal(got.finished.cpu(), want[3])
    live = torch.isfinite(want[0])
    assert torch.equal(got.scores.cpu()[~live].double(), want[0][~live])
    # the sum of the exponentials is off by 2^-22 of itself (each by two units of 2^-24, twice), its logarithm by as much; then one rounding to 32 bits
    assert bool(((got.scores.double().cpu() - want[0]).abs() <= 2.0 ** -22 + 2.0 ** -24 * want[0].abs() + 2.0 ** -40)[live].all())
    if history is not None:
        h = history.cpu().gather(1, want[1][:, :, None].expand(*want[1].shape, history.shape[2])).clone()
        h[:, :, step] = want[2]
        assert torch.equal(got.history.cpu(), h)
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("groups,beams,vocab", [(1, 1, 1), (3, 1, 5050), (7, 5, 5050), (2, 8, 33333), (1, 32, 700), (5, 3, 2), (2, 4, 8192), (1, 2, 8193), (40, 2, 100), (1, 16, 70001)])
def test_select_over_beams_and_vocabulary(dtype, groups, beams, vocab):
    g = torch.Generator().manual_seed(vocab + beams)
    logits = (torch.randn(groups * beams, vocab + 3, generator=g) * 3).to(dtype).to(DEV)[:, :vocab]
    scores = -torch.rand(groups, beams, generator=g).cumsum(1).to(DEV)
    finished = (torch.rand(groups, beams, generator=g) < 0.3).to(DEV)
    history = torch.randint(0, vocab, (groups, beams, 9), generator=g).to(DEV)
    select_check(logits, scores, finished, min(2, vocab - 1), history, 4)


def test_select_first_step_masked_vocabulary_and_rows_that_offer_nothing():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(12, 500, generator=g) * 2
    x[:, 200:] = float("-inf")                       # a masked vocabulary
    x[1, 3:] = float("-inf")                         # fewer live tokens than beams
    x[2] = float("-inf")                             # none
    x[5, 7], x[6, 0], x[7, 5] = float("nan"), float("inf"), float("-inf")
    x[8:12] = x[8]                                   # equal rows at equal scores: ties between beams
    s = torch.tensor([[0.0, -0.5, -0.25, float("-inf")], [float("nan"), -1.0, -0.1, -0.2], [-1.0, -1.0, -1.0, -1.0]])
    f = torch.zeros(3, 4, dtype=torch.bool)
    select_check(x.to(DEV), s.to(DEV), f.to(DEV), 2)
    s = torch.tensor([[0.0] + [float("-inf")] * 3] * 3)
    select_check(x.to(DEV), s.to(DEV), f.to(DEV), 2)
    f[0] = True                                      # all finished: the order of the scores, the end token again
    f[1, 1:3] = True
    select_check(x.to(DEV), torch.tensor([[-3.0, -1.0, -2.0, -1.0], [-1.0, -0.5, -9.0, -2.0], [0.0, 0.0, 0.0, 0.0]]).to(DEV), f.to(DEV), 499)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("beams,vocab", [(1, 9000), (5, 9000), (32, 600)])
def test_select_among_equal_logits_takes_the_lowest_index(dtype, beams, vocab):
    for fill in (0.0, float("-inf"), -10000.0):
        x = torch.full((2 * beams, vocab), fill, dtype=dtype, device=DEV)
        s = torch.zeros(2, beams, device=DEV)
        select_check(x, s, torch.zeros(2, beams, dtype=torch.bool, device=DEV), 0)
        x[:, vocab - 3] = 1.0                        # one above a plateau
        select_check(x, s, torch.zeros(2, beams, dtype=torch.bool, device=DEV), 0)
    x = torch.arange(vocab, device=DEV, dtype=torch.float32).div(100, rounding_mode="floor").expand(2 * beams, vocab).to(dtype).contiguous()      # plateaus of 100
    select_check(x, -torch.arange(2.0 * beams, device=DEV).view(2, beams) * 0.3, torch.zeros(2, beams, dtype=torch.bool, device=DEV), 1)


def test_select_in_place():
    g = torch.Generator().manual_seed(5)
    x = torch.randn(15, 800, generator=g).to(DEV)
    s, f = -torch.rand(3, 5, generator=g).to(DEV), (torch.rand(3, 5, generator=g) < 0.4).to(DEV)
    h = torch.randint(0, 800, (3, 5, 300), generator=g).to(DEV)
    want = D().select_beams(x, s, f, eos=2, history=h, step=299)
    out = want._replace(scores=s, finished=f, history=h, parents=torch.empty_like(want.parents), tokens=torch.empty_like(want.tokens))
    D().select_beams(x, s, f, eos=2, history=h, step=299, out=out)
    for a, b in zip(out, want):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------
# reorder
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("beams,page,layers,in_place", [(1, 16, 1, False), (5, 16, 2, True), (2, 1, 1, False), (8, 32, 3, True), (32, 8, 1, True)])
def test_reorder_tables_and_shared_pages(dtype, beams, page, layers, in_place):
    rng = random.Random(beams)
    kv = [0, 1, page, page + 1, 3 * page - 1, 2 * page]
    G, P = len(kv), 5
    for kind in ("random", "one", "reverse", "same"):
        parents = [[{"random": rng.randrange(beams), "one": beams - 1, "reverse": beams - 1 - w, "same": w}[kind] for w in range(beams)] for _ in range(G)]
        pool = rng.sample(range(G * beams * P), G * beams * P)
        tables = [[pool[r * P + j] for j in range(P)] for r in range(G * beams)]
        for g in range(G):                                     # full blocks are shared
            for w in range(beams):
                for j in range(kv[g] // page):
                    tables[g * beams + w][j] = tables[g * beams + rng.randrange(w + 1)][j]
        cache = torch.randn(layers, 2, G * beams * P, 3, page, 64, device=DEV).to(dtype)
        t, want_cache = i32(tables), cache.clone()
        want, copies = O.reorder(parents, kv, tables, page)
        for s, d, n in copies:
            if s >= 0:
                want_cache[:, :, d, :, :n] = cache[:, :, s, :, :n]
        got = D().reorder_pages(torch.tensor(parents, device=DEV), i32(kv), t, cache, out=t if in_place else None)
        assert got.tolist() == want and torch.equal(cache, want_cache)


def test_reorder_parents_outside_the_group_stay_and_are_reported():
    from mmf_amd import _native as nat
    t = i32([[0, 1], [2, 3], [4, 5]])
    got = D().reorder_pages(torch.tensor([[0, 7, -1]], device=DEV), i32([8]), t, torch.zeros(1, 6, 1, 4, 64, device=DEV))
    assert nat.take_index_error() and got.tolist() == t.tolist()


# ---------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------
class Decoder:
    """Two attention layers over random projections, and a vocabulary; `history` decides everything, so a plain run can be made from the tokens alone."""

    def __init__(self, heads=4, kv_heads=2, dim=64, vocab=300, layers=2, dtype=torch.float32, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.shape, self.layers, self.vocab, self.dtype = (heads, kv_heads, dim), layers, vocab, dtype
        H = heads * dim
        self.emb = torch.randn(vocab, H, generator=g).to(DEV)
        self.pos = (torch.randn(400, H, generator=g) * 0.5).to(DEV)
        self.w = [(torch.randn(H, (heads + 2 * kv_heads) * dim, generator=g) / H ** 0.5).to(DEV) for _ in range(layers)]
        self.o = [(torch.randn(H, H, generator=g) / H ** 0.5).to(DEV) for _ in range(layers)]
        self.head = (torch.randn(H, vocab, generator=g) * 3 / H ** 0.5).to(DEV)

    def step(self, cache, plan, tokens, max_q):
        heads, kv_heads, dim = self.shape
        x = self.emb[tokens] + self.pos[plan.positions.clamp(min=0).long()]
        for l in range(self.layers):
            qkv = (x @ self.w[l]).to(self.dtype).view(-1, heads + 2 * kv_heads, dim)
            cache.write(l, qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:], plan)
            ctx = cache.attend(l, qkv[:, :heads], plan, max_q=max_q)
            x = x + ctx.float().reshape(x.shape[0], -1) @ self.o[l]
        return x @ self.head

    def plain(self, tokens):
        """Logits behind the last of `tokens`, in 64 bits, without a cache."""
        heads, kv_heads, dim = self.shape
        n = len(tokens)
        x = self.emb.double()[tokens] + self.pos.double()[:n]
        for l in range(self.layers):
            qkv = (x @ self.w[l].double()).view(n, heads + 2 * kv_heads, dim).transpose(0, 1)
            q, k, v = qkv[:heads], qkv[heads:heads + kv_heads].repeat_interleave(heads // kv_heads, 0), qkv[heads + kv_heads:].repeat_interleave(heads // kv_heads, 0)
            s = (q @ k.transpose(1, 2).contiguous()) * dim ** -0.5
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1), float("-inf"))
            x = x + (torch.softmax(s, -1) @ v).transpose(0, 1).reshape(n, -1) @ self.o[l].double()
        return x[-1] @ self.head.double()


@pytest.mark.parametrize("beams,page", [(4, 8), (3, 4), (1, 16)])
def test_a_beam_search_over_the_paged_cache_is_the_search_without_one(beams, page):
    """Prompts of different lengths, nine steps of write, attend, select and reorder: every step's logits are those of a plain run over the tokens each beam holds."""
    d = D()
    G, steps, eos = 3, 9, 2
    lens = [5, 13, 8]
    model = Decoder()
    g = torch.Generator().manual_seed(11)
    prompts = [torch.randint(3, model.vocab, (n,), generator=g).to(DEV) for n in lens]
    cache = d.PagedCache(model.layers, G, beams, max(lens) + steps, kv_heads=2, head_dim=64, page_size=page, dtype=torch.float32)
    plan = cache.plan(i32(lens), sum(lens), shared=True)
    logits = model.step(cache, plan, torch.cat(prompts), max(lens))
    last = torch.tensor([sum(lens[:i + 1]) - 1 for i in range(G)], device=DEV)
    logits = logits[last].repeat_interleave(beams, 0)
    scores = torch.full((G, beams), float("-inf"), device=DEV); scores[:, 0] = 0
    finished = torch.zeros(G, beams, dtype=torch.bool, device=DEV)
    history = torch.zeros(G, beams, steps, dtype=torch.int64, device=DEV)
    for t in range(steps):
        for r in range(G * beams):
            if float(scores.view(-1)[r]) > float("-inf"):
                tokens = torch.cat([prompts[r // beams], history.view(-1, steps)[r, :t]])
                want = model.plain(tokens)
                assert float((logits[r].double() - want).abs().max()) < 1e-3 * float(want.abs().max()), (t, r)
        b = d.select_beams(logits, scores, finished, eos=eos, history=history, step=t)
        scores, finished, history = b.scores, b.finished, b.history
        if t + 1 < steps:
            cache.reorder(b.parents)
            plan = cache.plan(torch.ones(G, dtype=I32, device=DEV), G * beams)
            assert int(plan.refused) == 0
            logits = model.step(cache, plan, b.tokens.view(-1), 1)
    assert cache.kv_lens.tolist() == [n + steps - 1 for n in lens]
    # finished: every page comes back
    cache.plan(torch.full((G,), -1, dtype=I32, device=DEV), 1)
    assert int(cache.free_top) == cache.free_pages.numel() and sorted(cache.free_pages.tolist()) == list(range(cache.free_pages.numel()))


def test_a_captured_step_replays_like_the_eager_one():
    """A step captured once (state in place) and replayed, with eager work between the replays, against the same steps made eagerly."""
    d = D()
    G, W, steps = 2, 3, 6
    model = Decoder(dtype=torch.bfloat16, seed=4)
    runs = []
    for graphed in (False, True):
        cache = d.PagedCache(model.layers, G, W, 64, kv_heads=2, head_dim=64, page_size=8)
        plan = cache.plan(i32([11, 6]), 17, shared=True)
        g = torch.Generator().manual_seed(1)
        logits = model.step(cache, plan, torch.randint(3, model.vocab, (17,), generator=g).to(DEV), 11)[torch.tensor([10, 16], device=DEV)].repeat_interleave(W, 0)
        scores = torch.full((G, W), float("-inf"), device=DEV); scores[:, 0] = 0
        b = d.select_beams(logits, scores, torch.zeros(G, W, dtype=torch.bool, device=DEV), eos=2, history=torch.zeros(G, W, steps, dtype=torch.int64, device=DEV), step=0)
        state = d.BeamStep(*(x.clone() for x in b))
        one = torch.ones(G, dtype=I32, device=DEV)

        def step():
            cache.reorder(state.parents)
            plan = cache.plan(one, G * W)
            logits = model.step(cache, plan, state.tokens.view(-1), 1)
            d.select_beams(logits, state.scores, state.finished, eos=2, history=state.history, step=3, out=state)

        seen = []
        step()                                              # warm: library handles, workspaces
        if graphed:
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                step()
        for i in range(steps):
            graph.replay() if graphed else step()
            junk = torch.randn(64, 64, device=DEV) @ torch.randn(64, 64, device=DEV)
            torch.cuda.synchronize()
            seen.append([x.clone() for x in state] + [cache.kv_lens.clone(), cache.tables.clone(), cache.free_top.clone()])
        runs.append(seen)
    for a, b in zip(*runs):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_calls_on_another_stream_than_the_tensors_own():
    c = attend_case([300, 500], [1, 40], heads=4, kv_heads=4)
    want = attend_check(c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = D().attend_pages(c["q"], c["key_cache"], c["value_cache"], c["tables"], c["kv_lens"], c["q_start"], c["q_lens"], max_q=40)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[:41], want[:41])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pages_beyond_32_bits_of_bytes_and_elements(dtype):
    """A pool whose last pages start behind 2^32 elements: written, read by single tokens and by chunks, copied, as the first pages of a small pool are."""
    page, heads, dim, near = 64, 8, 128, 40
    pages = 2 ** 32 // (page * heads * dim) + near
    pool = torch.empty(2, pages, heads, page, dim, dtype=dtype, device=DEV)
    small = torch.zeros(2, near, heads, page, dim, dtype=dtype, device=DEV)
    pool[:, -near:] = 0
    g = torch.Generator().manual_seed(5)
    kv = [64 * 9 + 5, 700]
    k, v = (torch.randn(sum(kv), heads, dim, generator=g).to(dtype).to(DEV) for _ in range(2))
    tables = torch.randperm(near, generator=g, dtype=I32)[:22].view(2, 11)
    pos = torch.cat([torch.arange(n) for n in kv])
    req = torch.repeat_interleave(torch.arange(2), torch.tensor(kv))
    slots = tables[req, pos // page].long() * page + pos % page
    far = pages - near
    D().write_pages(k, v, small[0], small[1], slots.to(DEV))
    D().write_pages(k, v, pool[0], pool[1], (slots + far * page).to(DEV))
    assert torch.equal(pool[:, far:], small)
    for new in ([1, 1], [100, 650]):
        q = torch.randn(sum(new), 2 * heads, dim, generator=g).to(dtype).to(DEV)
        rest = dict(kv_lens=i32(kv), q_start=i32([0, new[0]]), q_lens=i32(new), max_q=max(new))
        assert torch.equal(D().attend_pages(q, pool[0], pool[1], (tables + far).to(DEV), **rest), D().attend_pages(q, small[0], small[1], tables.to(DEV), **rest))
    D().copy_pages(i32([[int(tables[0, 0]), int(tables[1, 10]), 33]]), small)
    D().copy_pages(i32([[far + int(tables[0, 0]), far + int(tables[1, 10]), 33]]), pool)
    assert torch.equal(pool[:, far:], small)


@pytest.mark.parametrize("beams,groups,new", [(1, 1000, 1), (1, 1000, 40), (32, 33, 1), (2, 500, 17), (1, 70, 40)])
def test_more_requests_than_a_launch_takes(beams, groups, new):
    """Requests beyond what one launch plans for, and beyond those that are put in order of length; each alike: 7 different lengths, compared among themselves and once with the plain form."""
    kv = [new + (g % 7) * 9 for g in range(groups)]
    c = attend_case(kv[:7], [new] * 7, beams=beams, heads=2, kv_heads=1)
    few = attend_check(c, beams=beams)
    rows, per = new * beams, len(kv[:7])
    idx = torch.arange(groups, device=DEV) % per
    many = dict(c, q=c["q"][:rows * per].view(per, rows, 2, 64)[idx].reshape(groups * rows, 2, 64), kv_lens=c["kv_lens"][idx], q_lens=c["q_lens"][idx],
                tables=c["tables"].view(per, beams, -1)[idx].reshape(groups * beams, -1), q_start=torch.arange(groups * beams, dtype=I32, device=DEV) * new)
    got = D().attend_pages(many["q"], many["key_cache"], many["value_cache"], many["tables"], many["kv_lens"], many["q_start"], many["q_lens"], max_q=new, beams=beams)
    assert torch.equal(got.view(groups, rows, 2, 64), few[:rows * per].view(per, rows, 2, 64)[idx])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_select_from_the_largest_vocabulary(dtype):
    W, V = 32, 2 ** 22
    g = torch.Generator(device=DEV).manual_seed(3)
    x = (torch.randn(W, V, generator=g, device=DEV) * 2).to(dtype)
    chosen = torch.randperm(W * V, generator=g, device=DEV)[:W]
    x.view(-1)[chosen] = (14 + 0.125 * torch.arange(W, device=DEV)).to(dtype)          # (exact in bf16: these and no others are the best)
    s = torch.zeros(1, W, device=DEV)
    got = D().select_beams(x, s, torch.zeros(1, W, dtype=torch.bool, device=DEV), eos=0)
    lse = torch.stack([torch.logsumexp(x[w].double(), 0) for w in range(W)])
    want, order = (x.view(-1)[chosen].double() - lse[chosen // V]).sort(descending=True)
    assert float((want[:-1] - want[1:]).min()) > 1e-4
    assert torch.equal(got.parents[0] * V + got.tokens[0], chosen[order])
    assert bool(((got.scores[0].double() - want).abs() <= 2.0 ** -22 + 2.0 ** -24 * want.abs() + 2.0 ** -40).all())


def test_two_graphs_of_split_attention_replay_in_turn_with_eager_calls_between():
    """Long caches are split over workgroups and joined through a workspace: two captured calls, and eager ones between their replays, do not meet in it."""
    cases = [attend_case([3000, 700], [1, 1], heads=4, kv_heads=2, dim=64), attend_case([2500], [60], heads=4, kv_heads=2, dim=64, seed=1)]
    names = ("q", "key_cache", "value_cache", "tables", "kv_lens", "q_start", "q_lens")

    def call(c):
        return D().attend_pages(*(c[k] for k in names), max_q=max(1, int(c["q"].shape[0])))
    for c in cases:
        call(c)
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(c))
        graphs.append(g)
    for turn in range(4):
        for c in cases:
            c["q"].copy_(torch.randn(c["q"].shape, generator=torch.Generator().manual_seed(turn)))
        for i in ((0, 1), (1, 0))[turn & 1]:
            outs[i].zero_()
            graphs[i].replay()
            call(cases[1 - i])
        torch.cuda.synchronize()
        for c, o in zip(cases, outs):
            n = int(c["q_lens"].sum())
            assert torch.equal(o[:n], call(c)[:n])


def test_two_streams_at_once():
    """Calls that run beside each other: every one has a workspace of its own."""
    c = [attend_case([3000, 700], [1, 1], heads=4, kv_heads=2, dim=64), attend_case([2500], [60], heads=4, kv_heads=2, dim=64, seed=1)]
    names = ("q", "key_cache", "value_cache", "tables", "kv_lens", "q_start", "q_lens")
    x = [torch.randn(8, 5050, device=DEV) for _ in range(2)]
    s, f = torch.zeros(2, 4, device=DEV), torch.zeros(2, 4, dtype=torch.bool, device=DEV)
    n = [int(a["q_lens"].sum()) for a in c]

    def run(i):
        return D().attend_pages(*(c[i][k] for k in names), max_q=60)[:n[i]], *D().select_beams(x[i], s, f, eos=2)[:4]
    want = [run(0), run(1)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got.append((i, run(i)))
    torch.cuda.synchronize()
    for i, r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want[i]))
