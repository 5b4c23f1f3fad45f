"""Refusals of the decoding operators (mmf_amd/decoding.py) and of their C entries, and the layouts of their descriptors: no GPU is needed to say no."""
import ctypes as C
import os
import shutil
import subprocess

import pytest
import torch

from mmf_amd import _native as nat
from mmf_amd import decoding as d

I32, I64 = torch.int32, torch.int64


# the descriptors of include/mmf_amd.h, as a caller of the C entries fills them
class PagedPlanDesc(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("q_lens", "kv_lens", "tables", "owned", "free_pages", "free_top", "q_start", "granted", "kv_out", "slots", "positions",
                                          "copies", "top_out", "refused", "ws")] + \
               [(n, C.c_int) for n in ("groups", "beams", "blocks", "page_size", "rows", "shared", "free_capacity")]


class PagedWriteDesc(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p)] + [(n, C.c_int64) for n in ("k_row", "k_head", "v_row", "v_head")] + \
               [("k_cache", C.c_void_p), ("v_cache", C.c_void_p)] + [(n, C.c_int64) for n in ("page_stride", "head_stride", "pos_stride")] + \
               [("slots", C.c_void_p)] + [(n, C.c_int) for n in ("tokens", "pages", "page_size", "kv_heads", "head_dim", "is_f32")]


class PagedAttnDesc(C.Structure):
    _fields_ = [("q", C.c_void_p), ("q_row", C.c_int64), ("q_head", C.c_int64), ("k_cache", C.c_void_p), ("v_cache", C.c_void_p)] + \
               [(n, C.c_int64) for n in ("page_stride", "head_stride", "pos_stride")] + [("tables", C.c_void_p), ("table_row", C.c_int64)] + \
               [(n, C.c_void_p) for n in ("kv_lens", "q_start", "q_lens", "out")] + [("out_row", C.c_int64), ("out_head", C.c_int64), ("ws", C.c_void_p)] + \
               [(n, C.c_int) for n in ("tokens", "requests", "beams", "blocks", "pages", "page_size", "heads", "kv_heads", "head_dim", "max_q", "causal", "is_f32")] + \
               [("scale", C.c_float)]


class BeamSelectDesc(C.Structure):
    _fields_ = [("logits", C.c_void_p), ("ld", C.c_int64)] + \
               [(n, C.c_void_p) for n in ("scores", "finished", "history", "scores_out", "parents", "tokens", "finished_out", "history_out", "ws")] + \
               [(n, C.c_int64) for n in ("vocab", "eos", "length", "step")] + [(n, C.c_int) for n in ("groups", "beams", "is_f32")]


class PagedReorderDesc(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("parents", "kv_lens", "tables", "tables_out", "copies")] + [(n, C.c_int) for n in ("groups", "beams", "blocks", "page_size")]


class PagedCopyDesc(C.Structure):
    _fields_ = [("copies", C.c_void_p), ("cache", C.c_void_p)] + [(n, C.c_int64) for n in ("plane_stride", "page_stride", "head_stride", "pos_stride")] + \
               [(n, C.c_int) for n in ("rows", "planes", "pages", "page_size", "kv_heads", "head_dim", "is_f32")]


def z(*s, dt=I32):
    return torch.zeros(*s, dtype=dt)


def plan_args(**over):
    a = dict(q_lens=z(2), kv_lens=z(2), tables=z(6, 4), owned=z(6, 4), free_pages=z(9), free_top=z(1), page_size=16, rows=8, beams=3)
    return dict(a, **over)


@pytest.mark.parametrize("over,says", [
    (dict(), "HBM"), (dict(page_size=0), "power of two"), (dict(page_size=24), "power of two"), (dict(page_size=2048), "power of two"), (dict(beams=0), "beams"),
    (dict(beams=33), "beams"), (dict(rows=0), "rows"), (dict(q_lens=z(2, dt=I64)), "q_lens"), (dict(kv_lens=z(3)), "kv_lens"), (dict(tables=z(5, 4)), "tables"),
    (dict(tables=z(4, 6).t()), "tables must be contiguous"), (dict(owned=z(6, 5)), "owned"), (dict(free_pages=z(0)), "empty"), (dict(free_top=z(2)), "free_top"), (dict(tables=z(6, 0), owned=z(6, 0)), "empty"),
    (dict(q_lens=z(0), kv_lens=z(0), tables=z(0, 4), owned=z(0, 4)), "groups")])
def test_plan_refuses(over, says):
    with pytest.raises(RuntimeError, match=says):
        d.plan_pages(**plan_args(**over))


def test_plan_refuses_results_of_other_shapes():
    out = d.PagePlan(z(6), z(2), z(2), z(8, dt=I64), z(8), z(6, 3), z(1), z(1), 3)
    with pytest.raises(RuntimeError, match="HBM"):
        d.plan_pages(**plan_args(), out=out)


def pools(dt=torch.bfloat16, pages=4, heads=2, page=16, dim=64):
    return torch.zeros(pages, heads, page, dim, dtype=dt), torch.zeros(pages, heads, page, dim, dtype=dt)


@pytest.mark.parametrize("over,says", [
    (dict(), "HBM"), (dict(k=torch.zeros(5, 2, 64)), "k must be"), (dict(v=torch.zeros(4, 2, 64, dtype=torch.bfloat16)), "v must be"), (dict(k=torch.zeros(5, 3, 64, dtype=torch.bfloat16)), "k must be"),
    (dict(slots=z(5)), "slots"), (dict(key_cache=torch.zeros(4, 2, 24, 64, dtype=torch.bfloat16)), "power of two"), (dict(key_cache=torch.zeros(4, 2, 64, dtype=torch.bfloat16)), "pages"),
    (dict(value_cache=torch.zeros(4, 2, 16, 64)), "value_cache"), (dict(value_cache=torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16)), "one shape"),
    (dict(key_cache=torch.zeros(4, 2, 16, 64, dtype=torch.float16)), "key_cache"), (dict(k=torch.zeros(5, 64, 2, dtype=torch.bfloat16).transpose(1, 2)), "contiguous head_dim"),
    (dict(k=torch.zeros(5, 2, 64, dtype=torch.bfloat16, requires_grad=True)), "gradient")])
def test_write_refuses(over, says):
    kc, vc = pools()
    a = dict(k=torch.zeros(5, 2, 64, dtype=torch.bfloat16), v=torch.zeros(5, 2, 64, dtype=torch.bfloat16), key_cache=kc, value_cache=vc, slots=z(5, dt=I64))
    with pytest.raises(RuntimeError, match=says):
        d.write_pages(**dict(a, **over))


@pytest.mark.parametrize("over,says", [
    (dict(), "HBM"), (dict(max_q=0), "max_q"), (dict(beams=4), "groups of 4"), (dict(q=torch.zeros(9, 3, 64, dtype=torch.bfloat16)), "multiple of 2"), (dict(q=torch.zeros(9, 4, 64)), "q must be"),
    (dict(q=torch.zeros(9, 4, 128, dtype=torch.bfloat16)), "q must be"), (dict(tables=z(6, 3, dt=I64)), "tables"), (dict(tables=z(3, 6).t()), "contiguous rows"), (dict(kv_lens=z(6)), "kv_lens"),
    (dict(q_lens=z(6)), "q_lens"), (dict(q_start=z(3)), "q_start"), (dict(q=torch.zeros(9, 4, 65, dtype=torch.bfloat16)[:, :, 1:]), "16 bytes"),
    (dict(q=torch.zeros(9, 4, 64, dtype=torch.bfloat16, requires_grad=True)), "gradient"), (dict(tables=z(6, 0)), "tables")])
def test_attend_refuses(over, says):
    kc, vc = pools()
    a = dict(q=torch.zeros(9, 4, 64, dtype=torch.bfloat16), key_cache=kc, value_cache=vc, tables=z(6, 3), kv_lens=z(3), q_start=z(6), q_lens=z(3), max_q=2, beams=2)
    with pytest.raises(RuntimeError, match=says):
        d.attend_pages(**dict(a, **over))


def test_attend_refuses_head_dims_and_results_it_has_no_kernel_for():
    kc, vc = pools(dim=32)
    with pytest.raises(RuntimeError, match="64 or 128"):
        d.attend_pages(torch.zeros(3, 2, 32, dtype=torch.bfloat16), kc, vc, z(3, 1), z(3), z(3), z(3), max_q=1)


@pytest.mark.parametrize("over,says", [
    (dict(), "HBM"), (dict(logits=torch.zeros(5, 10)), "logits"), (dict(logits=torch.zeros(6, 10, dtype=torch.float16)), "logits"), (dict(logits=torch.zeros(10, 6).t()), "contiguous rows"),
    (dict(logits=torch.zeros(10).expand(6, 10)), "overlap"), (dict(scores=torch.zeros(2, 3, dtype=torch.float64)), "scores"), (dict(finished=z(2, 3)), "finished"), (dict(eos=10), "eos"),
    (dict(eos=-1), "eos"), (dict(step=5), "step"), (dict(step=-1), "step"), (dict(history=z(2, 3, 5)), "history"), (dict(history=z(2, 4, 5, dt=I64)), "history"),
    (dict(logits=torch.zeros(2 ** 22 + 1).expand(6, -1)), "vocabulary of up to"), (dict(scores=torch.zeros(1, 33), logits=torch.zeros(33, 10)), "beams"), (dict(scores=torch.zeros(0, 3), logits=torch.zeros(0, 10)), "group")])
def test_select_refuses(over, says):
    a = dict(logits=torch.zeros(6, 10), scores=torch.zeros(2, 3), finished=z(2, 3, dt=torch.bool), eos=2, history=z(2, 3, 5, dt=I64), step=4)
    with pytest.raises(RuntimeError, match=says):
        d.select_beams(**dict(a, **over))


@pytest.mark.parametrize("over,says", [
    (dict(), "HBM"), (dict(parents=z(2, 3)), "parents"), (dict(kv_lens=z(3)), "kv_lens"), (dict(tables=z(5, 2)), "tables"), (dict(tables=z(6, 0)), "empty"), (dict(cache=torch.zeros(4, 2, 16)), "cache"),
    (dict(cache=torch.zeros(3, 2, 4, 2, 16, 64)[:, :1]), "run of planes"), (dict(cache=torch.zeros(4, 2, 12, 64)), "power of two"), (dict(cache=torch.zeros(4, 2, 16, 64, dtype=torch.int8)), "cache")])
def test_reorder_refuses(over, says):
    a = dict(parents=z(2, 3, dt=I64), kv_lens=z(2), tables=z(6, 2), cache=torch.zeros(3, 2, 4, 2, 16, 64))
    with pytest.raises(RuntimeError, match=says):
        d.reorder_pages(**dict(a, **over))


def test_copy_and_the_cache_refuse():
    with pytest.raises(RuntimeError, match="copies"):
        d.copy_pages(z(4, 2), torch.zeros(4, 2, 16, 64))
    with pytest.raises(RuntimeError, match="HBM"):
        d.copy_pages(z(4, 3), torch.zeros(4, 2, 16, 64))
    for over, says in ((dict(page_size=7), "power of two"), (dict(head_dim=96), "head_dim"), (dict(dtype=torch.float16), "dtype"), (dict(beams=40), "beams"), (dict(pages=0), "pages")):
        with pytest.raises(RuntimeError, match=says):
            d.PagedCache(1, 2, over.pop("beams", 2), 20, **dict(dict(kv_heads=2, head_dim=64, device="cpu"), **over))


def test_c_entries_refuse_before_they_launch():
    if not os.path.exists(nat.LIB_PATH):
        pytest.skip("library not built")
    L = nat.lib()
    for name, desc in (("mmf_paged_plan", PagedPlanDesc), ("mmf_paged_write", PagedWriteDesc), ("mmf_paged_attention", PagedAttnDesc),
                       ("mmf_beam_select", BeamSelectDesc), ("mmf_paged_reorder", PagedReorderDesc), ("mmf_paged_copy", PagedCopyDesc)):
        assert getattr(L, name)(None, None) != 0 and b"null operand" in L.mmf_amd_last_error(), name
        assert getattr(L, name)(C.byref(desc()), None) != 0 and b"null operand" in L.mmf_amd_last_error(), name

    def filled(desc, **over):
        x = desc()
        for f, t in desc._fields_:
            setattr(x, f, 4096 if t is C.c_void_p else 64 if f in ("head_dim",) else 1)
        for k, v in over.items():
            setattr(x, k, v)
        return x

    for name, x, says in (
            ("mmf_paged_plan", filled(PagedPlanDesc, page_size=3), b"power of two"), ("mmf_paged_plan", filled(PagedPlanDesc, beams=33), b"beams"),
            ("mmf_paged_plan", filled(PagedPlanDesc, rows=0), b"shape"), ("mmf_paged_plan", filled(PagedPlanDesc, blocks=1 << 30, page_size=2), b"2^30"),
            ("mmf_paged_write", filled(PagedWriteDesc, page_size=2000), b"page_size"), ("mmf_paged_write", filled(PagedWriteDesc, pages=0), b"shape"),
            ("mmf_paged_attention", filled(PagedAttnDesc, head_dim=96), b"head_dim"), ("mmf_paged_attention", filled(PagedAttnDesc, heads=3, kv_heads=2), b"multiple"),
            ("mmf_paged_attention", filled(PagedAttnDesc, max_q=0), b"max_q"), ("mmf_paged_attention", filled(PagedAttnDesc, page_size=6), b"power of two"),
            ("mmf_beam_select", filled(BeamSelectDesc, eos=1), b"end token"), ("mmf_beam_select", filled(BeamSelectDesc, eos=0, step=1), b"history"),
            ("mmf_beam_select", filled(BeamSelectDesc, beams=64), b"shape"), ("mmf_paged_reorder", filled(PagedReorderDesc, beams=0), b"shape"),
            ("mmf_paged_copy", filled(PagedCopyDesc, planes=70000), b"shape")):
        assert getattr(L, name)(C.byref(x), None) == 1 and says in L.mmf_amd_last_error(), (name, says, L.mmf_amd_last_error())


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no gcc")
def test_descriptors_have_the_layout_the_c_compiler_gives_them(tmp_path):
    pairs = {"mmf_paged_plan_desc": PagedPlanDesc, "mmf_paged_write_desc": PagedWriteDesc, "mmf_paged_attn_desc": PagedAttnDesc,
             "mmf_beam_select_desc": BeamSelectDesc, "mmf_paged_reorder_desc": PagedReorderDesc, "mmf_paged_copy_desc": PagedCopyDesc}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "mmf_amd.h"', 'int main(void) {']
    for cname, mirror in pairs.items():
        lines += ['printf("%zu", sizeof(' + cname + '));'] + ['printf(" %%zu", offsetof(%s, %s));' % (cname, f[0]) for f in mirror._fields_] + ['printf("\\n");']
    lines += ['printf("%d %d\\n", MMF_BEAMS_MAX, MMF_PAGE_MAX);', "return 0;", "}"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-I", os.path.dirname(nat.HEADER_PATH), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    for line, mirror in zip(out, pairs.values()):
        assert [int(x) for x in line.split()] == [C.sizeof(mirror)] + [getattr(mirror, f[0]).offset for f in mirror._fields_], mirror
    assert out[-1].split() == ["32", "1024"]
