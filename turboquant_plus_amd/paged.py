"""Caches in pages: packed K and V of many sequences in one pool, appended to and attended to through block tables.

A page is a 128-token block of every KV head of a layer, in the block format of `TurboCodec` (or q8_0-style rows): pools are uint8
[n_pages, n_kv_heads, bytes of a block], one for K and one for V under the same page numbers.  block_table [batch, blocks] (int32)
names the pages of each sequence's 128-token blocks.  Rows of new tokens are token-major [rows, heads, 128], sequence after
sequence; cu_new [batch + 1] (int32) says where each one's begin (None: one row each).  Tables and lengths are device tensors
that are read when a launch runs, so a captured step replays while they change.

The reference has no counterpart: its cache (turboquant/kv_cache.py:41-66) is rebuilt whole.
"""
from __future__ import annotations

import ctypes as C
import math

from . import _lib as L
from .turbo import BLOCK_TOKENS, HEAD_DIM, TurboCodec, _overrun_ptr

OVERRUN_NO_PAGE = 4     # TQ_OVERRUN_NO_PAGE of include/tq.h, beside OVERRUN_NEGATIVE and OVERRUN_NO_ROOM


def page_bytes(codec: TurboCodec | None) -> int:
    """Bytes of one KV head's block in a page (a codec of None: q8_0-style rows)."""
    return BLOCK_TOKENS * (136 if codec is None else 16 * codec.bits + 2)


def new_pages(k_codec: TurboCodec | None, v_codec: TurboCodec | None, n_pages: int, n_kv_heads: int):
    """Zeroed (k_pages, v_pages)."""
    tt, dev = L.torch(), L.require_gpu()
    return tuple(tt.zeros((n_pages, n_kv_heads, page_bytes(c)), dtype=tt.uint8, device=dev) for c in (k_codec, v_codec))


def _handle(codec):
    return None if codec is None else codec.handle.h


def _here(name, x, device):
    if not x.is_cuda or x.get_device() != device:
        raise ValueError(f"{name} must be on the current device")


def _pages(k_codec, v_codec, k_pages, v_pages, block_table, lens, cu_new, device) -> L.TQPages:
    tt = L.torch()
    for name, x, codec in (("k_pages", k_pages, k_codec), ("v_pages", v_pages, v_codec)):
        if x.dtype != tt.uint8 or x.dim() != 3 or x.shape[2] != page_bytes(codec) or not x.is_contiguous():
            raise ValueError(f"{name} must be a contiguous uint8 tensor [pages, KV heads, {page_bytes(codec)}]")
        _here(name, x, device)
    if k_pages.shape[:2] != v_pages.shape[:2]:
        raise ValueError("k_pages and v_pages must have the same pages and KV heads")
    if block_table.dtype != tt.int32 or block_table.dim() != 2 or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError("block_table must be int32 [batch, blocks], a sequence's entries next to each other")
    batch = block_table.shape[0]
    if lens.dtype != tt.int32 or tuple(lens.shape) != (batch,) or not lens.is_contiguous():
        raise ValueError("lengths must be a contiguous int32 tensor [batch]")
    if cu_new is not None:
        if cu_new.dtype != tt.int32 or tuple(cu_new.shape) != (batch + 1,) or not cu_new.is_contiguous():
            raise ValueError("cu_new must be a contiguous int32 tensor [batch + 1]")
        _here("cu_new", cu_new, device)
    _here("block_table", block_table, device)
    _here("lengths", lens, device)
    return L.TQPages(batch, k_pages.shape[1], k_pages.shape[0], block_table.shape[1],
                     block_table.stride(0) if batch > 1 else block_table.shape[1], block_table.data_ptr(),
                     None if cu_new is None else cu_new.data_ptr(), lens.data_ptr())


def _rows(name, x, heads, device):
    """Rows [rows, heads, 128] whose values lie next to each other."""
    if x.dim() != 3 or x.shape[2] != HEAD_DIM or (heads is not None and x.shape[1] != heads):
        raise ValueError(f"{name} must be [rows, {'heads' if heads is None else heads}, {HEAD_DIM}], got {tuple(x.shape)}")
    _here(name, x, device)
    return x if x.stride(2) == 1 else x.contiguous()


def _aligned(x, each):
    """x, or a copy of it whose rows begin at multiples of 16 bytes."""
    step = 16 // each
    return x if x.data_ptr() % 16 == 0 and x.stride(0) % step == 0 and x.stride(1) % step == 0 else x.clone(memory_format=L.torch().contiguous_format)


def append_paged(k_codec: TurboCodec | None, v_codec: TurboCodec | None, k, v, k_pages, v_pages, block_table, starts, cu_new=None, *,
                 overrun=None):
    """The new tokens' k and v [rows, KV heads, 128] (float16, bfloat16 or float32, any strides) into the pages of their
    sequences, from position starts[b] (int32 [batch]) of sequence b on, in one launch (tq_append_paged).  A codec of None stands for
    q8_0-style rows.  The bytes are those of LayerKV.append: earlier tokens stay, the rest of the last block is emptied.
    A page that is written must belong to one sequence.  A sequence without room, or a block without a page, is left out;
    `overrun` (a zeroed int32 device tensor with one element) then collects OVERRUN_* bits, see overrun_bits()."""
    tt, device = L.torch(), L._current_device()
    pages = _pages(k_codec, v_codec, k_pages, v_pages, block_table, starts, cu_new, device)
    k, v = _rows("k", k, pages.n_kv_heads, device), _rows("v", v, pages.n_kv_heads, device)
    if k.dtype != v.dtype or k.shape[0] != v.shape[0]:
        raise ValueError("k and v must have the same rows and dtype")
    code = L.TQ_BF16 if k.dtype == tt.bfloat16 else L.dtype_code(k)
    if code == L.TQ_F64:
        raise TypeError("unsupported dtype torch.float64")
    each = k.element_size()
    k, v = _aligned(k, each), _aligned(v, each)
    L.check(L.lib().tq_append_paged(_handle(k_codec), _handle(v_codec), C.byref(pages), k.data_ptr(), v.data_ptr(), k.shape[0], k.stride(0),
                                    k.stride(1), v.stride(0), v.stride(1), code, k_pages.data_ptr(), v_pages.data_ptr(),
                                    _overrun_ptr(overrun), L.stream_ptr()))
    return k_pages, v_pages


def load_paged(k_codec: TurboCodec | None, v_codec: TurboCodec | None, k_pages, v_pages, block_table, starts, cu_new=None,
               rows: int | None = None, *, out=None):
    """Positions starts[b] .. of every sequence, as many as cu_new gives it, back as fp16 values in the original domain: K and V
    [rows, KV heads, 128] in one launch (tq_load_paged).  rows: of the outputs (needed with cu_new); `out`: a pair of such
    tensors to write to instead.  Rows behind the last sequence, and rows without a page, are left as they were."""
    tt, device = L.torch(), L._current_device()
    pages = _pages(k_codec, v_codec, k_pages, v_pages, block_table, starts, cu_new, device)
    if out is not None:
        rows = out[0].shape[0]
    elif rows is None:
        if cu_new is not None:
            raise ValueError("load_paged needs the number of rows (rows, or out)")
        rows = pages.batch
    shape = (rows, pages.n_kv_heads, HEAD_DIM)
    if out is None:
        out = tuple(tt.empty(shape, dtype=tt.float16, device=k_pages.device) for _ in range(2))
    for x in out:
        if x.dtype != tt.float16 or tuple(x.shape) != shape or not x.is_contiguous():
            raise ValueError(f"outputs must be contiguous fp16 tensors {shape}")
        _here("out", x, device)
    L.check(L.lib().tq_load_paged(_handle(k_codec), _handle(v_codec), C.byref(pages), k_pages.data_ptr(), v_pages.data_ptr(), rows,
                                  out[0].data_ptr(), out[1].data_ptr(), L.stream_ptr()))
    return out


class PagedAttention:
    """softmax(scale q k^T) v of new tokens over a paged cache (tq_paged_attention): single tokens, a few drafted ones, chunks
    and whole prompts of a ragged batch, and (causal=False) queries over another sequence's states.

    Holds a workspace that grows to the largest call's need (a smaller one stays with the object, for calls that were captured with
    it): calls of one object must not overlap in time, replayed ones among them.
    A codec of None stands for q8_0-style rows on that side.
    """

    def __init__(self, k_codec: TurboCodec | None, v_codec: TurboCodec | None, n_q_heads: int, n_kv_heads: int, *, scale: float | None = None,
                 causal: bool = True):
        if n_kv_heads < 1 or n_q_heads < 1 or n_q_heads % n_kv_heads:
            raise ValueError(f"{n_q_heads} query heads are not a multiple of {n_kv_heads} KV heads")
        self.k_codec, self.v_codec = k_codec, v_codec
        self.n_q_heads, self.n_kv_heads, self.causal = n_q_heads, n_kv_heads, bool(causal)
        self.scale = 1.0 / math.sqrt(HEAD_DIM) if scale is None else float(scale)
        self.workspace, self._outgrown = None, []

    def __call__(self, q, k_pages, v_pages, block_table, lens, cu_new=None, *, max_context: int | None = None, max_new: int | None = None,
                 out=None):
        """q [rows, query heads, 128], float16 or bfloat16, original domain -> out of the same shape and dtype, contiguous.
        lens (int32 [batch]): tokens that each sequence's pages hold, the new ones among them; row t of a sequence's n sees the
        positions before lens[b] - n + t + 1 (all lens[b] of them with causal=False), and a row that sees nothing is 0.
        Rows behind the last sequence are left as they were (`out`: a contiguous tensor to write to).
        max_context, max_new: no sequence holds more tokens, or has more new ones.  They size the launch: without them the table's
        width and the number of rows do, and a call on short sequences takes longer.  Of a sequence that exceeds them the
        tokens behind max_context are not seen and the rows from max_new on are left as they were."""
        tt, device = L.torch(), L._current_device()
        pages = _pages(self.k_codec, self.v_codec, k_pages, v_pages, block_table, lens, cu_new, device)
        if pages.n_kv_heads != self.n_kv_heads:
            raise ValueError(f"pages of {pages.n_kv_heads} KV heads, expected {self.n_kv_heads}")
        q = _rows("q", q, self.n_q_heads, device)
        if q.dtype not in (tt.float16, tt.bfloat16):
            raise TypeError(f"queries must be float16 or bfloat16, not {q.dtype}")
        q = _aligned(q, 2)
        if out is None:
            out = tt.empty(q.shape, dtype=q.dtype, device=q.device)
        elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
            raise ValueError("out must be a contiguous tensor of q's shape and dtype")
        else:
            _here("out", out, device)
        p = L.TQPagedAttnParams(pages, self.n_q_heads, self.causal, self.scale, L.TQ_BF16 if q.dtype == tt.bfloat16 else L.TQ_F16, q.shape[0],
                                q.stride(0), q.stride(1), 0 if max_context is None else max_context, 0 if max_new is None else max_new)
        need = L.lib().tq_paged_attn_workspace_bytes(C.byref(p))
        if need < 0:
            L.check(L.ERR_ARG)
        if self.workspace is None or self.workspace.numel() < need or self.workspace.get_device() != device:
            if self.workspace is not None:
                self._outgrown.append(self.workspace)     # a captured call may still write to it
            self.workspace = tt.empty(need, dtype=tt.uint8, device=q.device)
        L.check(L.lib().tq_paged_attention(_handle(self.k_codec), _handle(self.v_codec), C.byref(p), q.data_ptr(), k_pages.data_ptr(),
                                           v_pages.data_ptr(), out.data_ptr(), self.workspace.data_ptr(), self.workspace.numel(),
                                           L.stream_ptr()))
        return out
