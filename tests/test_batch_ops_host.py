"""CPU checks of the batch-serving operators (paged append, paged attention,
logits): every refusal comes back before any device call, and the ctypes
structures lie in memory as the header's do."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

import arclight_b200 as A

P = 4096          # an aligned address that is never touched: the checks return first
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def cache(**kw):
    d = dict(k=P, v=P, page_table=P, n_pages=10, n_seqs=3, max_pages=4, page_size=16, n_head_kv=2, head_dim=128,
             type=A.ALB_KV_F16)
    d.update(kw)
    return A.PagedKV(**d)


def attend(kv, q=P, rows=3, heads=8, seqs=None, lengths=P, window=0, scale=0.1, ws=P, out=P, lse=None):
    return A.lib().alb_paged_attn(q, rows, heads, None if kv is None else C.byref(kv), seqs, lengths, window, scale,
                                  ws, out, lse, None)


def append(kv, qkv=P, stride=0, T=3, heads=8, qn=P, kn=P, eps=1e-6, rope=P, max_pos=64, pos=P, seqs=None, q=P):
    return A.lib().alb_qk_norm_rope_kv_paged(qkv, stride, T, heads, qn, kn, eps, rope, max_pos, pos, seqs,
                                             None if kv is None else C.byref(kv), q, None)


BAD_CACHES = [
    dict(k=None), dict(v=None), dict(page_table=None), dict(k=P + 2), dict(v=P + 8), dict(head_dim=96),
    dict(head_dim=0), dict(type=2), dict(type=-1), dict(n_pages=0), dict(page_size=0), dict(page_size=-4),
    dict(n_head_kv=0), dict(n_seqs=0), dict(max_pages=0), dict(n_pages=1 << 31), dict(n_pages=1 << 27),
    dict(max_pages=(1 << 26) + 1), dict(page_table=P + 2), dict(table_stride=3), dict(table_stride=-4),
    dict(head_stride=128),                                                    # only one of the three strides
    dict(head_stride=128, cell_stride=128, page_stride=4096),                 # cells on top of one another
    dict(head_stride=128, cell_stride=256, page_stride=4000),                 # pages on top of one another
    dict(head_stride=132, cell_stride=272, page_stride=16 * 272),             # no multiple of 8
    dict(head_stride=-128, cell_stride=256, page_stride=4096),
    dict(head_stride=128, cell_stride=256, page_stride=1 << 62),
]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda d: ",".join(f"{k}={v}" for k, v in d.items()))
def test_a_cache_that_cannot_be_used_is_refused(bad):
    assert attend(cache(**bad)) == A.ALB_ERR_INVALID
    assert append(cache(**bad)) == A.ALB_ERR_INVALID
    assert b"invalid argument" in A.lib().alb_last_error()


def test_attention_refusals():
    ok = cache()
    assert attend(None) == A.ALB_ERR_INVALID
    for bad in (dict(q=None), dict(lengths=None), dict(ws=None), dict(out=None), dict(rows=0), dict(rows=1 << 24),
                dict(heads=0), dict(heads=7), dict(heads=1), dict(window=-1), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(q=P + 4), dict(out=P + 8), dict(ws=P + 4), dict(heads=4096),
                dict(lengths=P + 1), dict(seqs=P + 2), dict(lse=P + 2)):
        assert attend(ok, **bad) == A.ALB_ERR_INVALID, bad
    need = A.lib().alb_paged_attn_workspace_bytes
    assert need(None, 1, 8) == 0
    assert need(C.byref(cache(head_dim=80)), 1, 8) == 0
    assert need(C.byref(ok), 0, 8) == 0
    assert need(C.byref(ok), 3, 7) == 0
    assert need(C.byref(ok), 3, 8) > 0


def test_append_refusals():
    ok = cache()
    assert append(None) == A.ALB_ERR_INVALID
    for bad in (dict(qkv=None), dict(rope=None), dict(pos=None), dict(q=None), dict(T=0), dict(T=1 << 30),
                dict(heads=0), dict(max_pos=0), dict(eps=-1.0), dict(eps=float("nan")), dict(qkv=P + 4),
                dict(rope=P + 8), dict(q=P + 4), dict(qn=P + 4), dict(kn=P + 2), dict(stride=12 * 128 - 4),
                dict(stride=12 * 128 + 2), dict(pos=P + 2), dict(seqs=P + 1)):
        assert append(ok, **bad) == A.ALB_ERR_INVALID, bad


def test_logits_refusals():
    def call(x=P, rows=4, vocab=1000, stride=0, y=1 << 20, ystride=0, nxt=None, **rules):
        r = A.LogitsRules(**rules)
        return A.lib().alb_logits_process(x, rows, vocab, stride, C.byref(r), y, ystride, nxt, None)

    assert A.lib().alb_logits_process(P, 4, 1000, 0, None, 1 << 20, 0, None, None) == A.ALB_ERR_INVALID
    for bad in (dict(x=None), dict(y=None), dict(rows=0), dict(vocab=0), dict(vocab=1 << 31), dict(stride=999),
                dict(ystride=999), dict(x=P + 2), dict(y=P + 4000), dict(y=P, ystride=1001),
                dict(y=P + 4 * 3 * 1000), dict(history=P, repetition=P), dict(history=P, history_stride=1 << 30, presence=P),
                dict(last_n=-1), dict(bias_ids=P, n_bias=4), dict(bias_ids=P, bias_values=P, n_bias=4),
                dict(bias_ids=P, bias_values=P, bias_offsets=P, n_bias=-1), dict(allow=P), dict(allow=P, n_allow=2, allow_stride=31),
                dict(vocab=450001, y=1 << 30), dict(nxt=P + 2), dict(temperature=P + 1), dict(history=P + 2, history_stride=4, frequency=P),
                dict(allow=P + 1, n_allow=2)):
        assert call(**bad) == A.ALB_ERR_INVALID, bad


def test_structures_lie_as_in_the_header(tmp_path):
    cc = shutil.which("gcc")
    if not cc:
        pytest.skip("no gcc")
    lines = []
    for cls, name in ((A.PagedKV, "alb_paged_kv"), (A.LogitsRules, "alb_logits_rules")):
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "lay.c"
    src.write_text('#include <stdio.h>\n#include "alb_cuda.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "lay"
    subprocess.run([cc, "-std=c11", "-Wall", "-Werror", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for cls in (A.PagedKV, A.LogitsRules):
        want.append(C.sizeof(cls))
        want += [getattr(cls, f).offset for f, _ in cls._fields_]
    assert got == want


def test_append_refusals_name_their_reason():
    """With the queries well away from the input, each refusal is its own, and an overlap is one."""
    ok, far = cache(), 1 << 30
    for bad, why in ((dict(qkv=None), b"qkv"), (dict(rope=None), b"rope_table"), (dict(pos=None), b"positions"),
                     (dict(T=0), b"T > 0"), (dict(T=1 << 30), b"T < "), (dict(heads=0), b"n_head > 0"),
                     (dict(max_pos=0), b"max_pos > 0"), (dict(eps=-1.0), b"eps"), (dict(qkv=P + 4), b"& 15"),
                     (dict(kn=P + 2), b"& 15"), (dict(stride=12 * 128 - 4), b"qkv_stride"), (dict(pos=P + 2), b"& 3")):
        assert append(ok, **{**dict(q=far), **bad}) == A.ALB_ERR_INVALID, bad
        message = A.lib().alb_last_error()
        assert why in message and b"q_out ==" not in message and b"qkv == q_out" not in message, (bad, message)
    row = 12 * 128 * 4
    for q, T in ((P, 3), (P + row, 2), (P + 2 * row - 16, 2), (P - 16, 1), (P + 16, 1), (P - 3 * 8 * 128 * 4 + 16, 3)):
        assert append(ok, qkv=P + (1 << 20), q=q + (1 << 20), T=T) == A.ALB_ERR_INVALID, (q, T)
        assert b"qkv == q_out" in A.lib().alb_last_error()


def test_attention_queries_and_outputs_do_not_half_overlap():
    ok, at, size = cache(), 1 << 20, 3 * 8 * 128 * 4
    for out in (at + 16, at - 16, at + size - 16, at - size + 16, at + 128 * 4):
        assert attend(ok, q=at, out=out) == A.ALB_ERR_INVALID, out
        assert b"y0" in A.lib().alb_last_error()
