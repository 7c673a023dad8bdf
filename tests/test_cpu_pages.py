"""The paged, batched operators' host side: descriptor layouts, and the calls that are refused before
anything is launched (no GPU needed: every pointer here is a made-up address that is never read)."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest

from conftest import HIP_LIB, ROOT
from qwen3_tts_amd import hip

pytestmark = pytest.mark.skipif(not os.path.exists(HIP_LIB), reason="libqwen_tts_hip.so not built")

P = 0x1000          # aligned to 16 bytes, never read


def test_descriptor_layouts():
    structs = {"qwen_hip_kv_pages_t": hip.KvPages, "qwen_hip_page_plan_t": hip.PagePlan, "qwen_hip_page_append_t": hip.PageAppend,
               "qwen_hip_page_attn_t": hip.PageAttn, "qwen_hip_packed_attn_t": hip.PackedAttn, "qwen_hip_logit_rules_t": hip.LogitRules}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "qwen_tts_hip.h"', 'int main(void){']
    for cname, py in structs.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    lines += ['printf("dt f32 %d\\ndt bf16 %d\\ndt f16 %d\\n", QWEN_HIP_DT_F32, QWEN_HIP_DT_BF16, QWEN_HIP_DT_F16);',
              'printf("plan 1 %d\\nplan 2 %d\\nplan 4 %d\\nplan 8 %d\\n", QWEN_HIP_PLAN_NO_PAGES, QWEN_HIP_PLAN_TABLE_FULL, '
              'QWEN_HIP_PLAN_TOO_MANY, QWEN_HIP_PLAN_INVALID);', "return 0;}"]
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
    assert {k: got[("dt", k)] for k in hip.DT} == hip.DT
    for v in (hip.PLAN_NO_PAGES, hip.PLAN_TABLE_FULL, hip.PLAN_TOO_MANY, hip.PLAN_INVALID):
        assert got[("plan", str(v))] == v


def refused(rc, word):
    assert rc == -1
    assert word in hip.last_error(), hip.last_error()


def pages(**kw):
    d = dict(k=P, v=P, dtype=hip.DT["bf16"], n_pages=10, page_size=16, n_kv_heads=8, head_dim=128, page_stride=16 * 1024,
             head_stride=16 * 128, slot_stride=128)
    return hip.KvPages(**{**d, **kw})


def plan(**kw):
    d = {n: P for n in ("new_len", "kv_len", "n_free", "table", "free_pages", "kv_len_out", "n_free_out", "cu_q", "pos", "slot", "status")}
    d.update(table_stride=8, B=4, page_size=16, n_pages=10, table_cols=8, max_tokens=64)
    return hip.PagePlan(**{**d, **kw})


@pytest.mark.parametrize("kw,word", [
    (dict(status=None), "null"), (dict(slot=None), "null"), (dict(B=0), "B 0"), (dict(B=2049), "2048"),
    (dict(page_size=0), "pages"), (dict(n_pages=0), "pages"), (dict(n_pages=1 << 20, page_size=1 << 12), "2^31"),
    (dict(table_cols=0), "table_cols"), (dict(table_cols=1 << 27, table_stride=1 << 27), "2^30"),
    (dict(table_stride=7), "table_stride"), (dict(max_tokens=-1), "max_tokens"), (dict(max_tokens=(1 << 28) + 1), "max_tokens")])
def test_plan_refuses(kw, word):
    refused(hip.lib().qwen_hip_op_page_plan(C.byref(plan(**kw)), None), word)


def test_null_descriptors_are_refused():
    L = hip.lib()
    refused(L.qwen_hip_op_page_plan(None, None), "null")
    refused(L.qwen_hip_op_page_append(None, None, None), "null")
    refused(L.qwen_hip_op_page_append(C.byref(pages()), None, None), "null")
    refused(L.qwen_hip_op_page_attention(None, None, None), "null")
    refused(L.qwen_hip_op_page_attention(C.byref(pages()), None, None), "null")
    refused(L.qwen_hip_op_page_attention_workspace(C.byref(pages()), None), "null")
    refused(L.qwen_hip_op_packed_attention(None, None), "null")
    refused(L.qwen_hip_op_logit_rules(None, None), "null")


BAD_PAGES = [(dict(k=None), "null"), (dict(dtype=0), "dtype"), (dict(dtype=3), "dtype"), (dict(head_dim=96), "head_dim"),
             (dict(n_kv_heads=0), "n_kv_heads"), (dict(n_pages=0), "pages"), (dict(page_size=-1), "pages"),
             (dict(k=P + 8), "aligned"), (dict(slot_stride=124), "strides"), (dict(page_stride=-8), "strides"),
             (dict(slot_stride=0), "overlap"), (dict(head_stride=64), "overlap"), (dict(page_stride=0), "overlap")]


def append(**kw):
    d = dict(q=P, k=P, v=P, q_out=P, q_stride=4096, k_stride=4096, v_stride=4096, q_out_stride=2048, pos=P, slot=P, rope_cos=P, rope_sin=P,
             dtype=0, n_heads=16, T=4, rope_len=100, eps=1e-6)
    return hip.PageAppend(**{**d, **kw})


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=2), "dtype"), (dict(dtype=7), "dtype"), (dict(k=None), "null"), (dict(slot=None), "null"), (dict(q_out=None), "null"),
    (dict(rope_sin=None), "RoPE"), (dict(pos=None), "RoPE"), (dict(rope_len=0), "RoPE"), (dict(T=-1), "T -1"), (dict(T=1 << 24), "T 16777216"),
    (dict(n_heads=0), "n_heads"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(v=P + 4), "aligned"),
    (dict(k_stride=4098), "strides"), (dict(q_out_stride=1024), "strides"), (dict(q_stride=-4), "strides")])
def test_append_refuses(kw, word):
    refused(hip.lib().qwen_hip_op_page_append(C.byref(pages()), C.byref(append(**kw)), None), word)


Q = 1 << 20             # bytes from any other operand


@pytest.mark.parametrize("kw,word", [
    # rows of 2048 q, 1024 k and 1024 v, q written densely into the same memory, and by less than a stride apart
    (dict(q=Q, k=Q + 8192, v=Q + 12288, q_out=Q), "two strides"), (dict(q=Q, k=3 * Q, v=4 * Q, q_out=Q, q_out_stride=4100), "two strides"),
    (dict(q=Q, k=3 * Q, v=4 * Q, q_out=Q + 16, q_out_stride=4096), "overlaps"), (dict(q=Q, k=3 * Q, v=4 * Q, q_out=Q - 16, q_out_stride=4096), "overlaps"),
    (dict(q=Q, k=3 * Q, v=4 * Q, q_out=Q + 16384 + 16, q_out_stride=4096), "overlaps"),
    (dict(q=Q, k=Q + 8192, v=Q + 12288, q_out=Q + 8192, q_out_stride=4096), "overlaps"),
    (dict(q=Q, k=3 * Q, v=4 * Q, q_out=4 * Q), "overlaps"), (dict(q=Q, k=3 * Q, k_stride=0, v=4 * Q, q_out=3 * Q - 3 * 8192 - 8176), "overlaps"),
    (dict(q=Q, k=3 * Q, v=4 * Q, q_out=4 * Q + 3 * 16384 + 4080, q_out_stride=2048), "overlaps"),
    (dict(q=Q, k=3 * Q, v=4 * Q, q_out=Q + 4096, T=1), "overlaps")])
def test_append_refuses_to_write_q_over_rows_that_are_read(kw, word):
    refused(hip.lib().qwen_hip_op_page_append(C.byref(pages(k=32 * Q, v=33 * Q)), C.byref(append(**kw)), None), word)



@pytest.mark.parametrize("kw,word", [
    (dict(v=32 * Q), "k and v"), (dict(v=32 * Q + 240), "k and v"), (dict(v=32 * Q - 9 * 32768 - 7 * 4096 - 15 * 256 - 240), "k and v"),
    # v begins within k's pages, in their gap but for the last 16 bytes
    (dict(page_stride=4 * 16384, v=32 * Q + 3 * 32768 + 16), "k and v"),
    (dict(page_stride=2048), "places"), (dict(page_stride=16384 - 8), "places"), (dict(slot_stride=136), "places"),
    (dict(head_stride=128, slot_stride=1016), "places"), (dict(n_pages=1, page_stride=0, head_stride=128, slot_stride=1016), "places"),
    (dict(n_pages=(1 << 27) - 1, page_stride=1 << 62, head_stride=1 << 62), "places")])
def test_append_refuses_a_cache_whose_rows_overlap(kw, word):
    refused(hip.lib().qwen_hip_op_page_append(C.byref(pages(**{**dict(k=32 * Q, v=40 * Q), **kw})), C.byref(append(q=Q, k=3 * Q, v=4 * Q, q_out=6 * Q)), None), word)



@pytest.mark.parametrize("kw,word", BAD_PAGES)
def test_bad_cache_descriptors_are_refused(kw, word):
    L = hip.lib()
    refused(L.qwen_hip_op_page_append(C.byref(pages(**kw)), C.byref(append()), None), word)
    refused(L.qwen_hip_op_page_attention(C.byref(pages(**kw)), C.byref(attn()), None), word)


def attn(**kw):
    d = dict(q=P, out=2 * P, q_stride=2048, out_stride=2048, cu_q=P, kv_len=P, table=P, table_stride=8, table_cols=8, workspace=P,
             workspace_bytes=1 << 40, dtype=1, n_heads=16, B=4, T=4, max_q=1, max_kv=128, window=0, scale=0.1)
    return hip.PageAttn(**{**d, **kw})


BAD_ROWS = [(dict(dtype=9), "dtype"), (dict(n_heads=12), "heads"), (dict(n_heads=0), "heads"), (dict(n_heads=8 * 65), "heads"),
            (dict(B=-1), "B -1"), (dict(B=65536), "B 65536"), (dict(T=-1), "tokens"), (dict(T=1 << 28), "tokens"),
            (dict(window=-1), "window"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
            (dict(scale=float("inf")), "scale"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(q=P + 8), "aligned"),
            (dict(q_stride=2050), "strides"), (dict(out_stride=1024), "strides"),
            (dict(out=P), "must not"), (dict(T=1 << 22), "rows")]


@pytest.mark.parametrize("kw,word", BAD_ROWS + [
    (dict(dtype=2), "cache"), (dict(kv_len=None), "null"), (dict(table=None), "null"), (dict(table_cols=0), "table_cols"),
    (dict(table_stride=7), "table_cols"), (dict(max_q=-1), "max_q"), (dict(max_kv=-1), "max_kv"),
    (dict(max_kv=1 << 16, workspace=None), "workspace"), (dict(max_kv=1 << 16, workspace_bytes=16), "workspace"),
    (dict(max_kv=1 << 16, workspace=P + 4), "aligned")])
def test_page_attention_refuses(kw, word):
    refused(hip.lib().qwen_hip_op_page_attention(C.byref(pages()), C.byref(attn(**kw)), None), word)


def test_more_tiles_than_a_launch_takes_are_refused():
    refused(hip.lib().qwen_hip_op_page_attention(C.byref(pages(n_kv_heads=65535, page_size=1)),
                                                 C.byref(attn(n_heads=65535, B=65535, T=1, out_stride=65535 * 128)), None), "tiles")


def test_f32_rows_need_a_bf16_cache():
    refused(hip.lib().qwen_hip_op_page_attention(C.byref(pages(dtype=2)), C.byref(attn(dtype=0)), None), "cache")


def test_workspace_follows_the_descriptor():
    L = hip.lib()
    size = lambda **kw: L.qwen_hip_op_page_attention_workspace(C.byref(pages()), C.byref(attn(**kw)))  # noqa: E731
    assert size(max_kv=16) == 0                                  # one range of keys: nothing to join
    long = size(max_kv=1 << 16)
    assert long > 0 and long % (4 * 16 * 130 * 4) == 0           # ranges of T rows of head_dim sums, a maximum, a sum
    refused(size(scale=0.0), "scale")


@pytest.mark.parametrize("kw,word", BAD_ROWS + [(dict(k=None), "null"), (dict(cu=None), "null"), (dict(v=P + 2), "aligned"),
                                                (dict(k_stride=1028), "strides"), (dict(v_stride=-8), "strides"), (dict(head_dim=80), "head_dim")])
def test_packed_attention_refuses(kw, word):
    d = dict(q=P, k=P, v=P, out=2 * P, q_stride=4096, k_stride=4096, v_stride=4096, out_stride=2048, cu=P, dtype=1, n_heads=16, n_kv_heads=8,
             head_dim=128, B=4, T=4, window=0, scale=0.1)
    refused(hip.lib().qwen_hip_op_packed_attention(C.byref(hip.PackedAttn(**{**d, **kw})), None), word)


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=5), "dtype"), (dict(logits=None), "null"), (dict(V=0), "rows"), (dict(B=65536), "rows"), (dict(B=-1), "rows"),
    (dict(out_stride=99), "strides"), (dict(out=P, out_stride=101), "in place"), (dict(hist_off=None), "history"),
    (dict(hist=None), "history"), (dict(hist_cap=-1), "history"), (dict(bias_off=None), "biases"), (dict(bias_val=None), "biases"),
    (dict(bias_cap=-1), "biases"), (dict(mask_stride=3), "mask_stride"), (dict(logits=P + 2), "aligned")])
def test_logit_rules_refuses(kw, word):
    d = dict(logits=P, out=P + 4096, logits_stride=100, out_stride=100, hist=P, hist_off=P, hist_cap=5, rep=P, bias_tok=P, bias_val=P,
             bias_off=P, bias_cap=5, mask=P, mask_stride=4, dtype=0, B=2, V=100)
    refused(hip.lib().qwen_hip_op_logit_rules(C.byref(hip.LogitRules(**{**d, **kw})), None), word)


# rows of 4096 bytes; 4 of them
@pytest.mark.parametrize("kw", [dict(out=Q + 16), dict(out=Q - 16), dict(out=Q + 4 * 4096 - 16), dict(out=Q - 4 * 4096 + 16), dict(q_stride=0, out=Q - 3 * 4096 - 16),
                                dict(q_stride=2056, out=Q + 4096), dict(q_stride=6144, out_stride=6144, out=Q + 2 * 4096 + 16)])
def test_attention_refuses_an_out_that_overlaps(kw):
    L, d = hip.lib(), {**dict(q=Q, T=4), **kw}
    refused(L.qwen_hip_op_page_attention(C.byref(pages(k=32 * Q, v=40 * Q)), C.byref(attn(**d)), None), "out overlaps q")
    for at in ("q", "k", "v"):                                  # k's and v's rows: as wide as q's
        e = dict(q=8 * Q, k=8 * Q, v=8 * Q, q_stride=2048, k_stride=2048, v_stride=2048, out_stride=2048, cu=P, dtype=1, n_heads=16, n_kv_heads=16,
                 head_dim=128, B=4, scale=0.1)
        e.update({at if k == "q" else at + "_stride" if k == "q_stride" else k: v for k, v in d.items()})
        refused(L.qwen_hip_op_packed_attention(C.byref(hip.PackedAttn(**e)), None), "out overlaps")


@pytest.mark.parametrize("kw", [dict(out=Q + 4), dict(out=Q + 396), dict(out=Q - 796 + 4), dict(out=Q + 400, out_stride=101), dict(out=Q + 200, logits_stride=200, out_stride=200)])
def test_logit_rules_refuse_an_out_that_overlaps(kw):
    d = dict(logits=Q, out=Q, logits_stride=100, out_stride=100, dtype=0, B=2, V=100)
    refused(hip.lib().qwen_hip_op_logit_rules(C.byref(hip.LogitRules(**{**d, **kw})), None), "overlaps")



def test_empty_calls_do_nothing():
    L = hip.lib()
    assert L.qwen_hip_op_page_append(C.byref(pages()), C.byref(append(T=0)), None) == 0
    assert L.qwen_hip_op_page_attention(C.byref(pages()), C.byref(attn(T=0)), None) == 0
    assert L.qwen_hip_op_page_attention(C.byref(pages()), C.byref(attn(B=0, q=None, out=None)), None) == 0
    r = hip.LogitRules(logits=P, out=P, logits_stride=4, out_stride=4, dtype=0, B=0, V=4)
    assert L.qwen_hip_op_logit_rules(C.byref(r), None) == 0
