"""Caches in pages without a GPU: sizes, and what the entry points refuse before any device work."""
import ctypes as C

import pytest

import turboquant_plus_amd as tqa
from turboquant_plus_amd import _lib as L

X, ODD = C.c_void_p(4096), C.c_void_p(4104)


def pages(**kw):
    p = dict(batch=2, n_kv_heads=8, n_pages=16, max_blocks=4, table_stride=4, block_table=4096, cu_new=4096, lens=4096)
    return L.TQPages(**{**p, **kw})


def attn(page_kw=None, **kw):
    p = dict(pages=pages(**(page_kw or {})), n_q_heads=32, causal=1, scale=0.1, dtype=L.TQ_F16, rows=10, q_token=4096, q_head=128)
    return L.TQPagedAttnParams(**{**p, **kw})


BAD_PAGES = [(dict(batch=-1), L.ERR_ARG, "negative"), (dict(n_kv_heads=0), L.ERR_ARG, "negative"), (dict(n_pages=-1), L.ERR_ARG, "negative"),
             (dict(max_blocks=-1), L.ERR_ARG, "negative"), (dict(n_kv_heads=70000), L.ERR_UNSUPPORTED, "65536"),
             (dict(batch=1 << 20, n_kv_heads=4096), L.ERR_UNSUPPORTED, "of all sequences"),
             (dict(max_blocks=1 << 24, table_stride=1 << 24), L.ERR_UNSUPPORTED, "32 bits"), (dict(table_stride=3), L.ERR_ARG, "table_stride"),
             (dict(block_table=None), L.ERR_ARG, "null"), (dict(lens=None), L.ERR_ARG, "null"), (dict(lens=4098), L.ERR_ALIGN, "aligned"),
             (dict(batch=20, cu_new=None), L.ERR_ARG, "10 rows for 20")]


def append(p, k=X, v=X, rows=10, step=1024, dtype=L.TQ_F16, kp=X, vp=X, over=None):
    return L.lib().tq_append_paged(None, None, C.byref(p), k, v, rows, step, 128, step, 128, dtype, kp, vp, over, None)


@pytest.mark.parametrize("kw,code,text", BAD_PAGES)
def test_pages_that_make_no_sense(kw, code, text):
    lib = L.lib()
    assert append(pages(**kw)) == code and text in L.last_error()
    assert lib.tq_load_paged(None, None, C.byref(pages(**kw)), X, X, 10, X, X, None) == code and text in L.last_error()
    assert lib.tq_paged_attention(None, None, C.byref(attn(kw)), X, X, X, X, X, 1 << 40, None) == code and text in L.last_error()
    assert lib.tq_paged_attn_workspace_bytes(C.byref(attn(kw))) == -1


def test_appends_and_loads_that_make_no_sense():
    assert append(pages(), dtype=L.TQ_F64) == L.ERR_ARG
    assert append(pages(), rows=-1) == L.ERR_ARG
    assert append(pages(), k=None) == L.ERR_ARG
    assert append(pages(), kp=None) == L.ERR_ARG
    assert append(pages(), kp=ODD) == L.ERR_ALIGN
    assert append(pages(), k=C.c_void_p(4097)) == L.ERR_ALIGN      # 8-bit rows need their type's alignment
    assert append(pages(), over=C.c_void_p(4098)) == L.ERR_ALIGN
    assert append(pages(batch=0)) == 0 and append(pages(), rows=0) == 0
    load = lambda out, p=X: L.lib().tq_load_paged(None, None, C.byref(pages()), p, X, 10, out, X, None)
    assert load(None) == L.ERR_ARG and load(ODD) == L.ERR_ALIGN and load(X, None) == L.ERR_ARG
    assert L.lib().tq_append_paged(None, None, None, X, X, 10, 1024, 128, 1024, 128, 0, X, X, None, None) == L.ERR_ARG


@pytest.mark.parametrize("kw,text", [(dict(n_q_heads=30), "multiple of the KV head count"), (dict(n_q_heads=0), "multiple"),
                                     (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
                                     (dict(scale=float("inf")), "scale"), (dict(dtype=L.TQ_F32), "dtype"), (dict(max_context=-1), "negative"),
                                     (dict(max_new=-1), "negative"), (dict(rows=-1), "negative")])
def test_attentions_that_make_no_sense(kw, text):
    assert L.lib().tq_paged_attention(None, None, C.byref(attn(**kw)), X, X, X, X, X, 1 << 40, None) == L.ERR_ARG
    assert text in L.last_error()
    assert L.lib().tq_paged_attn_workspace_bytes(C.byref(attn(**kw))) == -1


def test_attention_pointers_and_workspace():
    call = lambda p, q=X, kp=X, out=X, ws=X, n=1 << 40: L.lib().tq_paged_attention(None, None, C.byref(p), q, kp, X, out, ws, n, None)
    assert call(attn(), q=None) == L.ERR_ARG and call(attn(), kp=None) == L.ERR_ARG and call(attn(), ws=None) == L.ERR_ARG
    assert call(attn(), q=ODD) == L.ERR_ALIGN and call(attn(), out=ODD) == L.ERR_ALIGN and call(attn(q_token=4100)) == L.ERR_ALIGN
    assert call(attn(rows=0)) == 0 and call(attn(dict(batch=0))) == 0
    # one row over a long context is split, and its partial results need room: 128 sums, a maximum, a sum of weights each
    p = attn(dict(batch=1, max_blocks=1024, table_stride=1024), rows=1, max_new=1)
    need = L.lib().tq_paged_attn_workspace_bytes(C.byref(p))
    assert need >= 2 * 32 * 130 * 4 and (need - 16) % (32 * 130 * 4) == 0
    assert call(p, n=need - 1) == L.ERR_ARG and "workspace" in L.last_error()
    # many rows are not
    p = attn(dict(batch=8, max_blocks=1024, table_stride=1024), rows=8192)
    assert L.lib().tq_paged_attn_workspace_bytes(C.byref(p)) == 16


def test_sizes_and_arguments_of_the_classes():
    assert tqa.page_bytes(None) == 128 * 136 and [tqa.page_bytes(tqa.TurboCodec(b)) for b in (2, 3, 4)] == [128 * 34, 128 * 50, 128 * 66]
    with pytest.raises(ValueError, match="multiple"):
        tqa.PagedAttention(None, None, 10, 4)
    with pytest.raises(ValueError, match="multiple"):
        tqa.PagedAttention(None, None, 8, 0)
