"""What the decoding operators (mmf_amd/decoding.py) say about calls before any kernel runs: layouts, tangents, what a call writes."""
import pytest
import torch

from mmf_amd import decoding as d

I32, I64 = torch.int32, torch.int64


def z(*s, dt=I32):
    return torch.zeros(*s, dtype=dt)


# ---------------------------------------------------------------------------------------------
# planes
# ---------------------------------------------------------------------------------------------
PAGE = (4, 2, 16, 64)
P = 4 * 2 * 16 * 64
INNER = (2 * 16 * 64, 16 * 64, 64, 1)


def planes(sizes, strides):
    room = sum((n - 1) * s for n, s in zip(sizes, strides)) + P
    return torch.zeros(room).as_strided((*sizes, *PAGE), (*strides, *INNER))


@pytest.mark.parametrize("sizes,strides", [
    ((3, 1, 2), (3 * P, 3 * P, P)),            # the middle one hides that the outer steps over more planes than the inner has
    ((3, 1, 1, 2), (3 * P, 3 * P, 2 * P, P)), ((3, 2), (3 * P, P)), ((2, 3, 1, 2), (6 * P, 3 * P, 3 * P, P))])
@pytest.mark.parametrize("call", ["copy", "reorder"])
def test_planes_that_are_no_run_are_refused(sizes, strides, call):
    cache = planes(sizes, strides)
    with pytest.raises(RuntimeError, match="run of planes"):
        d.copy_pages(z(4, 3), cache) if call == "copy" else d.reorder_pages(z(2, 3, dt=I64), z(2), z(6, 2), cache)


@pytest.mark.parametrize("sizes,strides", [
    ((3, 1), (P, P)), ((1, 3), (17, P)), ((3, 1, 2), (2 * P, 2 * P, P)), ((1, 1), (5, 7)), ((3,), (2 * P,)), ((), ()), ((1, 2, 1, 3), (9, 3 * P, 3 * P, P))])
def test_planes_that_are_a_run_reach_the_device_check(sizes, strides):
    with pytest.raises(RuntimeError, match="HBM"):
        d.copy_pages(z(4, 3), planes(sizes, strides))


# ---------------------------------------------------------------------------------------------
# a step on the device
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("step,says", [(z(1), "HBM"), (z(1, dt=I64), "step must be"), (z(2), "step must be"), (torch.tensor(3, dtype=I32), "step must be"), (z(1).float(), "step must be"),
                                       (5, "not a column"), (-1, "not a column")])
def test_steps_that_are_no_column_and_no_int32_tensor_are_refused(step, says):
    with pytest.raises(RuntimeError, match=says):
        d.select_beams(torch.zeros(6, 10), torch.zeros(2, 3), z(2, 3, dt=torch.bool), eos=2, history=z(2, 3, 5, dt=I64), step=step)


def test_the_c_entry_refuses_a_null_step():
    from mmf_amd import _native as nat
    L = nat.lib()
    assert L.mmf_beam_select_at(None, None, None) != 0 and b"null operand" in L.mmf_amd_last_error()


# ---------------------------------------------------------------------------------------------
# forward-mode tangents: no operator here has a derivative
# ---------------------------------------------------------------------------------------------
bf = torch.bfloat16


def calls():
    kc, vc = torch.zeros(4, 2, 16, 64, dtype=bf), torch.zeros(4, 2, 16, 64, dtype=bf)
    q, k = torch.zeros(9, 4, 64, dtype=bf), torch.zeros(5, 2, 64, dtype=bf)
    attend = dict(q=q, key_cache=kc, value_cache=vc, tables=z(6, 3), kv_lens=z(3), q_start=z(6), q_lens=z(3), max_q=2, beams=2, out=torch.zeros(9, 4, 64, dtype=bf))
    select = dict(logits=torch.zeros(6, 10), scores=torch.zeros(2, 3), finished=z(2, 3, dt=torch.bool), eos=2)
    return {"write": (d.write_pages, dict(k=k, v=k.clone(), key_cache=kc, value_cache=vc, slots=z(5, dt=I64)), ("k", "v", "key_cache", "value_cache")),
            "attend": (d.attend_pages, attend, ("q", "key_cache", "value_cache", "out")), "select": (d.select_beams, select, ("logits", "scores")),
            "reorder": (d.reorder_pages, dict(parents=z(2, 3, dt=I64), kv_lens=z(2), tables=z(6, 2), cache=torch.zeros(3, 2, 4, 2, 16, 64)), ("cache",)),
            "copy": (d.copy_pages, dict(copies=z(4, 3), cache=torch.zeros(3, 2, 4, 2, 16, 64)), ("cache",))}


@pytest.mark.parametrize("call,name", [(c, n) for c, (_, _, names) in calls().items() for n in names])
def test_tensors_with_tangents_are_refused_like_those_that_require_gradients(call, name):
    import torch.autograd.forward_ad as fw
    f, args, _ = calls()[call]
    with fw.dual_level():
        dual = fw.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(RuntimeError, match="%s carries a tangent" % name):
            f(**dict(args, **{name: dual}))
        with torch.no_grad(), pytest.raises(RuntimeError, match="%s carries a tangent" % name):       # (no_grad stops the backward mode only)
            f(**dict(args, **{name: dual}))
        with fw._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="HBM"):
            f(**dict(args, **{name: dual}))
        with pytest.raises(RuntimeError, match="HBM"):
            f(**dict(args, **{name: fw.unpack_dual(dual).primal}))
    with pytest.raises(RuntimeError, match="%s requires a gradient" % name):
        f(**dict(args, **{name: args[name].clone().requires_grad_(True)}))
    with torch.no_grad(), pytest.raises(RuntimeError, match="HBM"):
        f(**dict(args, **{name: args[name].clone().requires_grad_(True)}))


def test_tangents_of_function_transforms_are_refused():
    f, args, _ = calls()["select"]
    with pytest.raises(RuntimeError, match="logits carries a tangent"):
        torch.func.jvp(lambda x: f(**dict(args, logits=x)).scores, (args["logits"],), (torch.ones_like(args["logits"]),))


# ---------------------------------------------------------------------------------------------
# schemas: what a call writes is marked, and what it returns is its own
# ---------------------------------------------------------------------------------------------
STATE = {"plan_pages": {"tables", "owned", "free_pages"}, "write_pages": {"key_cache", "value_cache"}, "attend_pages": set(), "select_beams": set(), "reorder_pages": {"cache"},
         "copy_pages": {"cache"}}


@pytest.mark.parametrize("name", STATE)
def test_schemas_mark_what_a_call_writes(name):
    d._lib()
    packet = getattr(torch.ops.mmf_amd_decode, name)
    forms = {"default": STATE[name]}
    if "out" in packet.overloads():
        forms["out"] = STATE[name] | {a.name for a in packet.out._schema.arguments if a.name.startswith("out")}
    assert ("out" in forms) == (name in ("plan_pages", "attend_pages", "select_beams", "reorder_pages"))
    for form, written in forms.items():
        schema = getattr(packet, form)._schema
        assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == written
        assert all(r.alias_info is None for r in schema.returns)
        assert not any(a.name.startswith("out") for a in schema.arguments) or (form == "out" and len(schema.returns) == 0)


@pytest.mark.parametrize("call,out,says", [
    ("select", (torch.zeros(2, 3),), "BeamStep"), ("select", (torch.zeros(2, 3), z(2, 3, dt=I64), z(2, 3, dt=I64), z(2, 3, dt=torch.bool)), "HBM"),
    ("select", (torch.zeros(2, 3), z(2, 3, dt=I64), z(2, 3, dt=I64), z(2, 3, dt=torch.bool), z(2, 3, 4, dt=I64)), "history goes with history"),
    ("select", (torch.zeros(2, 4), z(2, 3, dt=I64), z(2, 3, dt=I64), z(2, 3, dt=torch.bool)), "out.scores"), ("attend", torch.zeros(9, 4, 32, dtype=bf), "out must be"),
    ("attend", torch.zeros(9, 4, 64), "out must be"), ("reorder", z(6, 3), "out must be")])
def test_results_of_another_shape_or_kind_are_refused(call, out, says):
    f, args, _ = calls()[call]
    with pytest.raises(RuntimeError, match=says):
        f(**dict(args, out=out))


def test_a_plan_takes_a_whole_plan_of_results():
    args = dict(q_lens=z(2), kv_lens=z(2), tables=z(6, 4), owned=z(6, 4), free_pages=z(9), free_top=z(1), page_size=16, rows=8, beams=3)
    with pytest.raises(RuntimeError, match="PagePlan"):
        d.plan_pages(**args, out=(z(6), z(2)))
    good = [z(6), z(2), z(2), z(8, dt=I64), z(8), z(6, 3), z(1), z(1)]
    for i, name in enumerate(d.PagePlan._fields[:8]):
        bad = list(good)
        bad[i] = z(11, dt=bad[i].dtype)
        with pytest.raises(RuntimeError, match="out.%s must be" % name):
            d.plan_pages(**args, out=bad)


# ---------------------------------------------------------------------------------------------
# errors between steps
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("entry", ["mmf_decode_take_error", "mmf_paged_attention_take_error"])
def test_errors_of_kernels_that_never_ran_are_not_fetched(entry):
    """Without a GPU a copy from the device fails (-1): a process that has launched none of these kernels makes none."""
    import subprocess
    import sys

    from mmf_amd import _native as nat
    code = "import ctypes; print(ctypes.CDLL(%r).%s())" % (nat.LIB_PATH, entry)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.strip() == "0", (r.stdout, r.stderr)


# ---------------------------------------------------------------------------------------------
# views whose values are not their memory
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("call,name", [(c, n) for c, (_, _, names) in calls().items() for n in names])
def test_negated_views_are_refused(call, name):
    f, args, _ = calls()[call]
    view = torch._neg_view(args[name])
    with pytest.raises(RuntimeError, match="%s is a negated view" % name):
        f(**dict(args, **{name: view}))
    with pytest.raises(RuntimeError, match="HBM"):
        f(**dict(args, **{name: view.resolve_neg()}))
