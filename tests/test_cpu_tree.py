"""The host side of the quantised cache and of trees of drafted tokens: descriptor layouts, and the calls that are refused
before anything is launched (no GPU needed: every pointer here is a made-up address that is never read)."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest

from conftest import HIP_LIB, ROOT
from qwen3_tts_amd import hip
from test_cpu_pages import P, Q, append, attn, pages, refused

pytestmark = pytest.mark.skipif(not os.path.exists(HIP_LIB), reason="libqwen_tts_hip.so not built")


def test_descriptor_layouts():
    structs = {"qwen_hip_kv_pages_t": hip.KvPages, "qwen_hip_tree_plan_t": hip.TreePlan, "qwen_hip_tree_t": hip.Tree,
               "qwen_hip_tree_verify_t": hip.TreeVerify, "qwen_hip_tree_commit_t": hip.TreeCommit}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "qwen_tts_hip.h"', 'int main(void){']
    for cname, py in structs.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    lines += ['printf("dt e4m3 %d\\n", QWEN_HIP_DT_E4M3);', "return 0;}"]
    with tempfile.TemporaryDirectory() as td:
        src, exe = os.path.join(td, "probe.c"), os.path.join(td, "probe")
        open(src, "w").write("\n".join(lines))
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), src, "-o", exe], check=True, capture_output=True)
        out = subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split("\n")
    got = {tuple(ln.split()[:2]): int(ln.split()[2]) for ln in out if ln}
    for cname, py in structs.items():
        assert got[(cname, "size")] == C.sizeof(py), cname
        for f, _ in py._fields_:
            assert got[(cname, f)] == getattr(py, f).offset, (cname, f)
    assert got[("dt", "e4m3")] == hip.E4M3


def codes(**kw):
    """A quantised cache of [page][head][place] in four pools."""
    d = dict(k=32 * Q, v=33 * Q, dtype=hip.E4M3, n_pages=10, page_size=16, n_kv_heads=8, head_dim=128, page_stride=16 * 1024, head_stride=16 * 128,
             slot_stride=128, k_scale=34 * Q, v_scale=35 * Q, scale_page_stride=128, scale_head_stride=16, scale_slot_stride=1)
    return hip.KvPages(**{**d, **kw})


def rows8(**kw):
    return append(**{**dict(q=Q, k=3 * Q, v=4 * Q, q_out=6 * Q), **kw})


@pytest.mark.parametrize("kw,word", [
    (dict(k_scale=None), "scale"), (dict(v_scale=None), "scale"), (dict(scale_page_stride=-1), "scale strides"), (dict(scale_slot_stride=-1), "scale strides"),
    (dict(k=32 * Q + 8), "aligned"), (dict(slot_stride=136), "strides"), (dict(page_stride=-16), "strides"), (dict(head_dim=96), "head_dim")])
def test_bad_quantised_caches_are_refused(kw, word):
    L = hip.lib()
    refused(L.qwen_hip_op_page_append(C.byref(codes(**kw)), C.byref(rows8()), None), word)
    for t in (0, 1, 2):
        refused(L.qwen_hip_op_page_attention(C.byref(codes(**kw)), C.byref(attn(dtype=t)), None), word)
    refused(L.qwen_hip_op_tree_commit(C.byref(codes(**kw)), C.byref(commit()), None), word)


@pytest.mark.parametrize("kw,word", [
    (dict(v=32 * Q), "k and v"), (dict(v=32 * Q + 112), "k and v"), (dict(page_stride=1024), "places"),
    (dict(v_scale=34 * Q), "k and v"), (dict(v_scale=34 * Q + 1279), "k and v"), (dict(scale_page_stride=127), "places"), (dict(scale_head_stride=15), "places"),
    (dict(scale_slot_stride=0), "places"), (dict(k_scale=32 * Q), "among"), (dict(k_scale=32 * Q + 9 * 16384 + 16383), "among"),
    (dict(v_scale=33 * Q - 1279), "among"),
    # pages of codes and scales: 16384 + 112 of them, the scales 16 bytes too early
    (dict(page_stride=16384 + 128, scale_page_stride=16384 + 128, k_scale=32 * Q + 16384 - 16, v_scale=35 * Q), "among"),
    (dict(n_pages=1, k_scale=32 * Q + 5), "among")])
def test_append_refuses_a_quantised_cache_whose_places_overlap(kw, word):
    refused(hip.lib().qwen_hip_op_page_append(C.byref(codes(**kw)), C.byref(rows8()), None), word)


def test_caches_and_rows_that_do_not_go_together():
    L = hip.lib()
    refused(L.qwen_hip_op_page_append(C.byref(codes()), C.byref(rows8(dtype=hip.E4M3)), None), "dtype")
    refused(L.qwen_hip_op_page_attention(C.byref(codes()), C.byref(attn(dtype=hip.E4M3)), None), "dtype")
    for t in (0, 1, 2):                                        # refused for the workspace alone
        refused(L.qwen_hip_op_page_attention(C.byref(codes()), C.byref(attn(dtype=t, max_kv=1 << 16, workspace=None)), None), "workspace")


def tree(**kw):
    return hip.Tree(**{**dict(mask=P, pos=P, mask_stride=2, mask_words=2), **kw})


@pytest.mark.parametrize("kw,akw,word", [
    (dict(mask=None), {}, "null"), (dict(pos=None), dict(window=5), "pos"), (dict(mask_words=0), {}, "mask_words"), (dict(mask_words=33, mask_stride=33), {}, "mask_words"),
    (dict(mask_stride=1), {}, "mask_words"), ({}, dict(dtype=2), "cache"), ({}, dict(scale=0.0), "scale"), ({}, dict(q=None), "null"), ({}, dict(out=P), "must not")])
def test_tree_attention_refuses(kw, akw, word):
    refused(hip.lib().qwen_hip_op_tree_attention(C.byref(pages()), C.byref(attn(**akw)), C.byref(tree(**kw)), None), word)


def tree_plan(**kw):
    return hip.TreePlan(**{**dict(parent=P, cu_q=P, kv_len=P, pos=P, mask=P, mask_stride=2, B=3, T=9, mask_words=2), **kw})


@pytest.mark.parametrize("kw,word", [
    (dict(parent=None), "null"), (dict(cu_q=None), "null"), (dict(kv_len=None), "null"), (dict(pos=None), "null"), (dict(mask=None), "null"),
    (dict(B=-1), "B -1"), (dict(B=65536), "B 65536"), (dict(T=-1), "T -1"), (dict(T=(1 << 26) + 1), "T 67108865"), (dict(mask_words=0), "mask_words"),
    (dict(mask_words=33, mask_stride=40), "mask_words"), (dict(mask_stride=1), "mask_words")])
def test_tree_plan_refuses(kw, word):
    refused(hip.lib().qwen_hip_op_tree_plan(C.byref(tree_plan(**kw)), None), word)


def verify(**kw):
    d = {n: P for n in ("p", "q", "tok", "parent", "cu_q", "u", "r", "path", "out_tok", "n_path", "workspace")}
    d.update(p_stride=1000, q_stride=1000, workspace_bytes=1 << 30, dtype=1, B=3, T=9, V=1000)
    return hip.TreeVerify(**{**d, **kw})


@pytest.mark.parametrize("kw,word", [
    *[(({n: None}), "null") for n in ("p", "tok", "parent", "cu_q", "u", "r", "path", "out_tok", "n_path")],
    (dict(dtype=3), "dtype"), (dict(dtype=hip.E4M3), "dtype"), (dict(B=-1), "B -1"), (dict(B=65536), "B 65536"), (dict(T=-1), "T -1"), (dict(V=0), "V 0"),
    (dict(V=(1 << 20) + 1, p_stride=1 << 21, q_stride=1 << 21), "V 1048577"), (dict(p=P + 1), "aligned"), (dict(q=P + 1), "aligned"), (dict(p_stride=999), "strides"), (dict(q_stride=999), "strides"),
    (dict(workspace=None), "workspace"), (dict(workspace_bytes=8), "workspace"), (dict(workspace=P + 8), "aligned"), (dict(max_children=-1), "max_children")])
def test_tree_verify_refuses(kw, word):
    refused(hip.lib().qwen_hip_op_tree_verify(C.byref(verify(**kw)), None), word)


def commit(**kw):
    d = {n: P for n in ("path", "n_path", "cu_q", "kv_len", "table", "kv_len_out", "free_pages", "n_free", "n_free_out", "status")}
    d.update(table_stride=8, table_cols=8, B=3, T=9, n_layers=1)
    return hip.TreeCommit(**{**d, **kw})


@pytest.mark.parametrize("kw,word", [
    *[(({n: None}), "null") for n in ("path", "n_path", "cu_q", "kv_len", "table", "free_pages", "n_free", "n_free_out", "status")],
    (dict(B=-1), "B -1"), (dict(B=2049), "2048"), (dict(T=-1), "T -1"), (dict(n_layers=-1), "layers"), (dict(B=2048, n_layers=1 << 13), "layers"),
    (dict(table_cols=0), "table_cols"), (dict(table_cols=1 << 27, table_stride=1 << 27), "2^30"), (dict(table_stride=7), "table_cols"),
    (dict(n_layers=2), "layers"), (dict(n_layers=2, layer_stride=10 * 16384 - 16), "layers"), (dict(n_layers=2, layer_stride=10 * 16384, scale_layer_stride=1279), "layers"),
    (dict(n_layers=2, layer_stride=64 * Q + 8, scale_layer_stride=2 * Q), "layer_stride")])
def test_tree_commit_refuses(kw, word):
    refused(hip.lib().qwen_hip_op_tree_commit(C.byref(codes()), C.byref(commit(**kw)), None), word)


def test_null_descriptors_are_refused():
    L = hip.lib()
    refused(L.qwen_hip_op_tree_plan(None, None), "null")
    refused(L.qwen_hip_op_tree_attention(None, None, None, None), "null")
    refused(L.qwen_hip_op_tree_attention(C.byref(pages()), C.byref(attn()), None, None), "null")
    refused(L.qwen_hip_op_tree_attention(C.byref(pages()), None, C.byref(tree()), None), "null")
    refused(L.qwen_hip_op_tree_verify(None, None), "null")
    refused(L.qwen_hip_op_tree_verify_workspace(None), "null")
    refused(L.qwen_hip_op_tree_commit(None, C.byref(commit()), None), "null")
    refused(L.qwen_hip_op_tree_commit(C.byref(codes()), None, None), "null")


def test_workspaces_follow_the_descriptor():
    L = hip.lib()
    a, b = (L.qwen_hip_op_tree_verify_workspace(C.byref(verify(V=v))) for v in (1000, 100000))
    assert 0 < a < b and L.qwen_hip_op_tree_verify_workspace(C.byref(verify(B=0))) == 0
    size = lambda kv, **kw: L.qwen_hip_op_page_attention_workspace(C.byref(kv), C.byref(attn(**kw)))  # noqa: E731
    assert size(codes(), max_kv=1 << 16) > 0 and size(codes(), max_kv=16) == 0


def test_empty_calls_do_nothing():
    L = hip.lib()
    assert L.qwen_hip_op_page_append(C.byref(codes()), C.byref(rows8(T=0)), None) == 0
    assert L.qwen_hip_op_page_attention(C.byref(codes()), C.byref(attn(T=0)), None) == 0
    assert L.qwen_hip_op_tree_attention(C.byref(codes()), C.byref(attn(B=0)), C.byref(tree()), None) == 0
    assert L.qwen_hip_op_tree_plan(C.byref(tree_plan(T=0, parent=None)), None) == 0
    assert L.qwen_hip_op_tree_verify(C.byref(verify(B=0)), None) == 0
    assert L.qwen_hip_op_tree_commit(C.byref(codes()), C.byref(commit(B=0)), None) == 0
    assert L.qwen_hip_op_tree_commit(C.byref(codes()), C.byref(commit(n_layers=0, kv_len_out=None)), None) == 0


def apart(**kw):
    """A descriptor's buffers far from each other."""
    return {n: (i + 8) * 64 * Q for i, n in enumerate(kw["names"])}


@pytest.mark.parametrize("a,b", [("pos", "parent"), ("pos", "cu_q"), ("mask", "kv_len"), ("mask", "pos")])
def test_tree_plan_refuses_outputs_that_overlap(a, b):
    d = apart(names=("parent", "cu_q", "kv_len", "pos", "mask"))
    d[a] = d[b]
    refused(hip.lib().qwen_hip_op_tree_plan(C.byref(tree_plan(**d)), None), "overlaps")


@pytest.mark.parametrize("a,b,off", [("out_tok", "tok", 0), ("path", "parent", 32), ("path", "out_tok", -32), ("n_path", "r", 8), ("n_path", "cu_q", 12), ("out_tok", "u", 0),
                                     ("path", "p", 2000 * 9 - 8), ("path", "q", 0), ("workspace", "p", 0), ("n_path", "workspace", 0)])
def test_tree_verify_refuses_outputs_that_overlap(a, b, off):
    d = apart(names=("p", "q", "tok", "parent", "cu_q", "u", "r", "path", "out_tok", "n_path", "workspace"))
    d[a] = d[b] + off
    refused(hip.lib().qwen_hip_op_tree_verify(C.byref(verify(**d)), None), "overlaps")


@pytest.mark.parametrize("a,b,off", [("kv_len_out", "kv_len", 4), ("kv_len_out", "path", 0), ("kv_len_out", "n_path", 0), ("n_free_out", "kv_len", 0), ("n_free_out", "status", 0),
                                     ("free_pages", "table", 0), ("free_pages", "n_free", -8), ("status", "cu_q", 0), ("n_free_out", "free_pages", 36)])
def test_tree_commit_refuses_outputs_that_overlap(a, b, off):
    d = apart(names=("path", "n_path", "cu_q", "kv_len", "table", "kv_len_out", "free_pages", "n_free", "n_free_out", "status"))
    d[a] = d[b] + off
    refused(hip.lib().qwen_hip_op_tree_commit(C.byref(codes()), C.byref(commit(**d)), None), "overlaps")


def test_errors_name_the_call():
    L = hip.lib()
    for f, who in ((lambda a: L.qwen_hip_op_page_attention(C.byref(pages()), C.byref(a), None), "page_attention"),
                   (lambda a: L.qwen_hip_op_tree_attention(C.byref(pages()), C.byref(a), C.byref(tree()), None), "tree_attention")):
        for kw in (dict(scale=0.0), dict(q=None), dict(out_stride=1024), dict(max_kv=1 << 16, workspace=None)):
            refused(f(attn(**kw)), who + ":")


def test_tree_plan_refuses_a_window_under_none():
    refused(hip.lib().qwen_hip_op_tree_plan(C.byref(tree_plan(window=-1)), None), "window")


@pytest.mark.parametrize("kw,layer,scale_layer", [
    (dict(k_scale=32 * Q + 10 * 16384), 10 * 16384, 2 * Q),                                     # layer 1's codes begin where layer 0's scales do
    (dict(v_scale=32 * Q + 2 * 10 * 16384 + 77), 10 * 16384, 10 * 16384),                       # layer 0's scales, layer 2's codes
    (dict(k_scale=32 * Q - 1280 - 10), 10 * 16384, 1290),                                       # layer 1's scales, layer 0's codes
    # [page][layer][codes | scales]: the scales 16 bytes too early
    (dict(page_stride=3 * 17000 // 16 * 16, scale_page_stride=3 * 17000 // 16 * 16, k_scale=32 * Q + 16384 - 16, v=64 * Q, v_scale=66 * Q), 16992, 16992),
    # the same, the scales of the page before over the next page's layer 0
    (dict(page_stride=3 * 16384, scale_page_stride=3 * 16384, k_scale=32 * Q + 3 * 16384 - 100, v=64 * Q, v_scale=66 * Q), 16384, 16384)])
def test_commit_refuses_scales_among_another_layers_codes(kw, layer, scale_layer):
    refused(hip.lib().qwen_hip_op_tree_commit(C.byref(codes(**kw)), C.byref(commit(n_layers=3, layer_stride=layer, scale_layer_stride=scale_layer)), None), "among")


@pytest.mark.parametrize("t", [0, 1])
@pytest.mark.parametrize("what,at,window", [("out", "mask", 0), ("out", "mask", 5), ("out", "pos", 5), ("workspace", "mask", 0), ("workspace", "pos", 5)])
def test_tree_attention_refuses_outputs_that_overlap(t, what, at, window):
    """The last bytes of one, the first of the other."""
    L, heads = hip.lib(), dict(dtype=t, B=1, T=9, n_heads=16, q=96 * Q, out=98 * Q, workspace=128 * Q, workspace_bytes=64 * Q, max_kv=1 << 16, window=window,
                               q_stride=2048, out_stride=2048)
    kv, a, tr = pages(k=8 * Q, v=16 * Q), attn(**heads), tree(mask=100 * Q, pos=101 * Q)
    end = {"mask": 100 * Q + 4 * (8 * 2 + 2), "pos": 101 * Q + 4 * 9}[at]
    setattr(a, what, (end - 1) // 16 * 16)
    refused(L.qwen_hip_op_tree_attention(C.byref(kv), C.byref(a), C.byref(tr), None), what)
    assert "overlap" in hip.last_error()
