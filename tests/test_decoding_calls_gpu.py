"""Calls of the decoding operators (mmf_amd/decoding.py) that the documentation allows: layouts of the cache's planes, indices outside their tables."""
import pytest
import torch

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
# planes: leading dimensions of the cache, some of size 1
# ---------------------------------------------------------------------------------------------
LEADING = [(), (1,), (4,), (4, 1), (1, 4), (4, 1, 2), (1, 1), (2, 1, 1), (1, 3, 1, 2)]


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 5)])
@pytest.mark.parametrize("lead", LEADING)
def test_copies_reach_every_plane(lead, dtype, dim):
    cache = torch.randn(*lead, 6, 2, 16, dim, device=DEV).to(dtype)
    copies = [[0, 3, 7], [5, 1, 16], [-1, -1, -1], [4, 4, 9]]
    want = cache.clone()
    for s, d, n in copies[:2]:
        want[..., d, :, :n, :] = cache[..., s, :, :n, :]
    D().copy_pages(i32(copies), cache)
    assert torch.equal(cache, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lead", LEADING)
def test_reorder_copies_in_every_plane(lead, dtype):
    cache = torch.randn(*lead, 6, 2, 16, 64, device=DEV).to(dtype)
    want = cache.clone()
    want[..., 2, :, :5, :] = cache[..., 3, :, :5, :]            # both children of beam 1: the second takes beam 0's page
    want[..., 4, :, :5, :] = cache[..., 3, :, :5, :]            # and the third beam 2's
    got = D().reorder_pages(torch.tensor([[1, 1, 1]], device=DEV), i32([21]), i32([[0, 2], [1, 3], [5, 4]]), cache)
    assert got.tolist() == [[1, 3], [1, 2], [1, 4]] and torch.equal(cache, want)


def test_planes_of_a_slice_of_the_layers():
    """One leading dimension may have any stride: keys only, of a pool that holds keys and values."""
    cache = torch.randn(3, 2, 6, 2, 16, 64, device=DEV)
    want = cache.clone()
    want[:, 0, 3, :, :7] = cache[:, 0, 0, :, :7]
    D().copy_pages(i32([[0, 3, 7]]), cache[:, 0])
    assert torch.equal(cache, want)


# ---------------------------------------------------------------------------------------------
# a step on the device
# ---------------------------------------------------------------------------------------------
def beam_state(G, W, V, length, seed=0):
    g = torch.Generator().manual_seed(seed)
    scores = -torch.rand(G, W, generator=g).cumsum(1)
    return (torch.randn(G * W, V, generator=g) * 2).to(DEV), scores.to(DEV), (torch.rand(G, W, generator=g) < 0.2).to(DEV), torch.randint(0, V, (G, W, length), generator=g).to(DEV)


@pytest.mark.parametrize("length,beams", [(1, 3), (7, 1), (300, 5), (40, 32)])
def test_a_step_on_the_device_is_the_same_number(length, beams):
    x, s, f, h = beam_state(3, beams, 700, length)
    for step in {0, length // 2, length - 1}:
        want = D().select_beams(x, s, f, eos=2, history=h, step=step)
        got = D().select_beams(x, s, f, eos=2, history=h, step=i32([step]))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(got.history[:, :, step], got.tokens)


@pytest.mark.parametrize("step", [-1, 9, -2 ** 31, 2 ** 31 - 1])
def test_a_step_outside_the_history_is_left_out_and_reported(step):
    from mmf_amd import _native as nat
    x, s, f, h = beam_state(2, 4, 500, 9)
    want = D().select_beams(x, s, f, eos=2, history=h, step=0)
    got = D().select_beams(x, s, f, eos=2, history=h, step=i32([step]))
    assert nat.take_index_error()
    assert all(torch.equal(a, b) for a, b in zip(got[:4], want[:4]))
    assert torch.equal(got.history, h.gather(1, got.parents[:, :, None].expand_as(h)))
    D().select_beams(x, s, f, eos=2, step=i32([step]))          # without a history there is no column to miss


@pytest.mark.parametrize("beams,dtype", [(1, torch.bfloat16), (3, torch.bfloat16), (5, torch.float32)])
def test_a_captured_search_keeps_its_tokens(beams, dtype):
    """A step captured once and replayed, the history's column advanced within it: every column is the eager search's, after each replay."""
    from tests.test_decoding_gpu import Decoder
    d = D()
    G, steps = 2, 9
    model = Decoder(dtype=dtype, seed=4)
    runs = []
    for graphed in (False, True):
        cache = d.PagedCache(model.layers, G, beams, 64, kv_heads=2, head_dim=64, page_size=8, dtype=dtype)
        plan = cache.plan(i32([11, 6]), 17, shared=True)
        g = torch.Generator().manual_seed(1)
        logits = model.step(cache, plan, torch.randint(3, model.vocab, (17,), generator=g).to(DEV), 11)[torch.tensor([10, 16], device=DEV)].repeat_interleave(beams, 0)
        scores = torch.full((G, beams), float("-inf"), device=DEV); scores[:, 0] = 0
        b = d.select_beams(logits, scores, torch.zeros(G, beams, dtype=torch.bool, device=DEV), eos=2, history=torch.full((G, beams, steps), -1, device=DEV), step=0)
        state, at, one = d.BeamStep(*(x.clone() for x in b)), i32([1]), torch.ones(G, dtype=I32, device=DEV)

        def step(column):
            cache.reorder(state.parents)
            plan = cache.plan(one, G * beams)
            logits = model.step(cache, plan, state.tokens.view(-1), 1)
            d.select_beams(logits, state.scores, state.finished, eos=2, history=state.history, step=column, out=state)

        step(at if graphed else 1)                             # warm: library handles, workspaces
        at += 1
        if graphed:
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                step(at)
                at += 1
        seen = []
        for i in range(2, steps):
            graph.replay() if graphed else step(i)
            junk = torch.randn(64, 64, device=DEV) @ torch.randn(64, 64, device=DEV)
            torch.cuda.synchronize()
            seen.append([x.clone() for x in state])
            assert bool((state.history[:, :, :i + 1] >= 0).all()) and bool((state.history[:, :, i + 1:] == -1).all())
        runs.append(seen)
    for a, b in zip(*runs):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


# ---------------------------------------------------------------------------------------------
# schemas
# ---------------------------------------------------------------------------------------------
def form_args():
    g = torch.Generator().manual_seed(2)
    kc, vc = (torch.randn(9, 2, 16, 64, generator=g).to(DEV) for _ in range(2))
    q, k, v = (torch.randn(4, n, 64, generator=g).to(DEV) for n in (4, 2, 2))
    x, s, f, h = beam_state(2, 2, 50, 6)
    tables, owned = i32([[0, 1, -1], [0, 2, -1], [3, -1, -1], [3, -1, -1]]), i32([[0, 1, -1], [-1, 2, -1], [3, -1, -1], [-1, -1, -1]])
    one = torch.ones(2, dtype=I32, device=DEV)
    plan = dict(q_lens=one, kv_lens=i32([20, 16]), tables=tables.clone(), owned=owned, free_pages=i32([4, 5, 6, 7, 8]), free_top=i32([5]), page_size=16, rows=4, beams=2, shared=False)
    attend = dict(q=q, key_cache=kc, value_cache=vc, tables=tables[:, :2].clamp(min=0).contiguous(), kv_lens=i32([20, 16]), q_start=i32([0, 1, 2, 3]), q_lens=one, max_q=1, beams=2,
                  causal=True, scale=None)
    select = dict(logits=x, scores=s, finished=f, eos=2, history=h, step=0, step_at=i32([3]))
    reorder = dict(parents=torch.tensor([[1, 1], [0, 0]], device=DEV), kv_lens=i32([20, 16]), tables=tables.clone(), cache=torch.stack([kc, vc]))
    return {"plan_pages": plan, "write_pages": dict(k=k, v=v, key_cache=kc, value_cache=vc, slots=torch.tensor([3, -1, 40, 100], device=DEV)), "attend_pages": attend, "select_beams": select,
            "reorder_pages": reorder, "copy_pages": dict(copies=i32([[0, 4, 5]]), cache=torch.stack([kc, vc]))}


FORMS = [(n, "default") for n in ("plan_pages", "write_pages", "attend_pages", "select_beams", "reorder_pages", "copy_pages")] + \
        [(n, "out") for n in ("plan_pages", "attend_pages", "select_beams", "reorder_pages")]


@pytest.mark.parametrize("name,form", FORMS)
def test_a_call_writes_what_its_schema_marks_and_nothing_else(name, form):
    D()._lib()
    packet = getattr(torch.ops.mmf_amd_decode, name)
    args, want = form_args()[name], None
    if form == "out":
        outs = [a.name for a in packet.out._schema.arguments if a.kwarg_only]
        want = packet.default(**form_args()[name])
        want = want if isinstance(want, (tuple, list)) else (want,)
        assert len(want) == len(outs)
        args.update({n: torch.full_like(w, True if w.dtype == torch.bool else 77) for n, w in zip(outs, want)})
    before = {n: t.clone() for n, t in args.items() if torch.is_tensor(t)}
    got = getattr(packet, form)(**args)
    written = {a.name for a in getattr(packet, form)._schema.arguments if a.alias_info is not None and a.alias_info.is_write}
    changed = {n for n, t in before.items() if not torch.equal(t, args[n])}
    assert changed <= written, changed - written
    if form == "out":
        assert got is None and all(torch.equal(args[n], w) for n, w in zip(outs, want))
    else:
        results = [] if got is None else list(got) if isinstance(got, (tuple, list)) else [got]
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in results if t.numel())
        assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))                       # results do not overlap
        held = {args[n].untyped_storage().data_ptr() for n in before}
        assert not any(t.untyped_storage().data_ptr() in held for t in results if t.numel())


# ---------------------------------------------------------------------------------------------
# pages that are none: reported by whoever leaves them out
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("groups", [1, 300])
@pytest.mark.parametrize("beams,shared,new", [(1, True, 1), (1, True, 40), (3, False, 1), (3, True, 2)])
def test_a_plan_reports_tokens_whose_block_has_no_page(beams, shared, new, groups):
    """Tokens that go on in a block whose table entry is -1 get no slot; those behind it have pages of their own.  In one launch and in two."""
    from mmf_amd import _native as nat
    page, P = 16, 6
    tables = torch.full((groups * beams, P), -1, dtype=I32, device=DEV)
    tables[:, 0] = torch.arange(groups * beams, dtype=I32, device=DEV)
    per = 1 if shared else beams
    free = torch.arange(1000, 1000 + 4 * groups * beams, dtype=I32, device=DEV)

    def plan(t):
        return D().plan_pages(torch.full((groups,), new, dtype=I32, device=DEV), torch.full((groups,), 5, dtype=I32, device=DEV), t, t.clone(), free.clone(), i32([free.numel()]),
                              page_size=page, rows=groups * per * new, beams=beams, shared=shared)
    good = plan(tables.clone())
    assert not nat.take_index_error() and bool((good.slots >= 0).all()) and int(good.refused) == 0
    bad = tables.clone()
    bad[0, 0] = -1
    p = plan(bad)
    assert nat.take_index_error()
    lost = min(new, page - 5)
    want = good.slots.clone()
    want[:lost] = -1
    assert torch.equal(p.slots, want) and torch.equal(p.positions, good.positions) and torch.equal(p.q_lens, good.q_lens)


def test_a_plan_reports_a_block_that_cannot_be_copied_and_free_pages_that_are_none():
    from mmf_amd import _native as nat
    t, o = i32([[-1, -1], [-1, -1]]), i32([[0, -1], [-1, -1]])          # the second beam shares the block and has to have a copy of it
    p = D().plan_pages(i32([1]), i32([3]), t, o, i32([7, 8]), i32([2]), page_size=16, rows=2, beams=2)
    assert nat.take_index_error()
    assert p.copies.tolist() == [[-1, -1, -1], [-1, 8, 3]] and p.slots.tolist() == [-1, 8 * 16 + 3]
    t = i32([[-1, -1]])
    p = D().plan_pages(i32([1]), i32([0]), t, t.clone(), i32([7, -4]), i32([2]), page_size=16, rows=1)
    assert nat.take_index_error() and p.slots.tolist() == [-1]


@pytest.mark.parametrize("case,reports", [("good", False), ("no source", True), ("no destination", True), ("no page, no copy", False), ("too long", True), ("negative", True),
                                          ("full", False)])
def test_a_reorder_reports_copies_without_a_page_and_lengths_without_a_block(case, reports):
    from mmf_amd import _native as nat
    cache = torch.randn(8, 2, 16, 64, device=DEV)
    tables = [[0, 1], [2, 3], [4, 5]]
    parents, kv = [[0, 0, 2]], 20                              # the second child of beam 0 takes beam 1's page
    if case == "no source":
        tables[0][1] = -1
    elif case == "no destination":
        tables[1][1] = -5
    elif case == "no page, no copy":
        parents, tables[2][1] = [[1, 0, 2]], -1
    elif case in ("too long", "negative", "full"):
        kv = {"too long": 33, "negative": -3, "full": 32}[case]
    before, want = cache.clone(), cache.clone()
    if case == "good":
        want[3, :, :4] = before[1, :, :4]
    got = D().reorder_pages(torch.tensor(parents, device=DEV), i32([kv]), i32(tables), cache)
    assert nat.take_index_error() == reports
    assert torch.equal(cache, want)
    last = 1 if case in ("good", "no source", "no destination") else None               # the block that goes on being written, if there is one
    for w, p in enumerate(parents[0]):
        source = [0, 1, 2][w] if last else p
        assert got[w].tolist() == [tables[p][0], tables[source][1]]


# ---------------------------------------------------------------------------------------------
# errors between steps
# ---------------------------------------------------------------------------------------------
def test_replays_report_as_often_as_they_meet_a_bad_page():
    from mmf_amd import _native as nat
    a = form_args()
    write, attend = a["write_pages"], a["attend_pages"]
    attend.pop("causal"), attend.pop("scale")
    D().write_pages(**write)
    D().attend_pages(**attend)
    assert not nat.take_index_error()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        D().write_pages(**write)
        D().attend_pages(**attend)
    good, table = write["slots"].clone(), attend["tables"].clone()
    for turn in range(6):
        write["slots"].copy_(good + (10 ** 6 if turn % 3 == 1 else 0))
        attend["tables"].copy_(table + (100 if turn % 3 == 2 else 0))
        torch.cuda.synchronize()
        assert not nat.take_index_error()
        graph.replay()
        torch.cuda.synchronize()
        assert nat.take_index_error() == (turn % 3 != 0), turn
        assert not nat.take_index_error()


# ---------------------------------------------------------------------------------------------
# groups of beams that do not fill a workgroup evenly, calls with nothing to do, lists of free pages that are not what they say
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("beams,heads,kv_heads,new,kv,shared", [(5, 16, 2, 1, [150, 33, 1], 32), (3, 16, 1, 1, [70, 200], 64), (7, 12, 2, 1, [700, 40], 512), (5, 6, 2, 2, [90, 17], 16),
                                                               (32, 24, 8, 1, [40], 16), (3, 32, 1, 1, [600, 100], 0)])
def test_beams_that_a_workgroup_takes_in_uneven_parts(dtype, beams, heads, kv_heads, new, kv, shared):
    from tests.test_decoding_gpu import attend_case, attend_check
    attend_check(attend_case(kv, [min(new, n) for n in kv], beams=beams, heads=heads, kv_heads=kv_heads, dtype=dtype, shared=shared), beams=beams)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("max_q", [1, 40])
@pytest.mark.parametrize("kv", [[70, 20], [3000, 700], [0, 0]])
def test_attention_without_a_new_token_leaves_its_result_alone(dtype, max_q, kv):
    from tests.test_decoding_gpu import attend_case
    c = attend_case(kv, [0, 0], heads=4, kv_heads=2, dtype=dtype, gaps=50)
    out = torch.full_like(c["q"], 7.0)
    D().attend_pages(c["q"], c["key_cache"], c["value_cache"], c["tables"], c["kv_lens"], c["q_start"], c["q_lens"], max_q=max_q, out=out)
    assert bool((out == 7.0).all())


@pytest.mark.parametrize("told,top", [(9, 5), (-3, 0)])
def test_a_plan_reports_a_stack_that_is_longer_than_its_list(told, top):
    from mmf_amd import _native as nat
    t = torch.full((1, 4), -1, dtype=I32, device=DEV)
    p = D().plan_pages(i32([20]), i32([0]), t, t.clone(), i32([10, 11, 12, 13, 14]), i32([told]), page_size=16, rows=20)
    assert nat.take_index_error()
    assert p.free_top.tolist() == [top - 2 if top else 0] and p.refused.tolist() == [0 if top else 1]
    assert t.tolist() == ([[14, 13, -1, -1]] if top else [[-1] * 4])


def test_a_plan_reports_pages_that_come_back_twice():
    from mmf_amd import _native as nat
    t = i32([[0, 1], [2, 3]])
    free = i32([7, 8, -1])
    p = D().plan_pages(i32([-1, -1]), i32([32, 32]), t, t.clone(), free, i32([2]), page_size=16, rows=1)      # four pages come back where one fits
    assert nat.take_index_error()
    assert p.free_top.tolist() == [3] and free.tolist() == [7, 8, 0] and p.kv_lens.tolist() == [0, 0]
