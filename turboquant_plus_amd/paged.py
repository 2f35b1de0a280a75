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


def _refuse_place(device, **tensors):
    for name, x in tensors.items():
        if x is not None and x.get_device() != device:     # -1: host memory
            raise ValueError(f"{name} must be on the current device")


# The checks below are most of what a call on a few tokens takes on the host (14 us a call at first, 4 of them the launch), so each asks
# a tensor once and no name is made before something is wrong.

def _pages(k_codec, v_codec, k_pages, v_pages, block_table, lens, cu_new, device) -> L.TQPages:
    tt = L.torch()
    k_shape, v_shape = k_pages.shape, v_pages.shape
    for name, x, shape, codec in (("k_pages", k_pages, k_shape, k_codec), ("v_pages", v_pages, v_shape, v_codec)):
        if x.dtype is not tt.uint8 or len(shape) != 3 or shape[2] != page_bytes(codec) or not x.is_contiguous():
            raise ValueError(f"{name} must be a contiguous uint8 tensor [pages, KV heads, {page_bytes(codec)}]")
    if k_shape[:2] != v_shape[:2]:
        raise ValueError("k_pages and v_pages must have the same pages and KV heads")
    if block_table.dtype is not tt.int32 or block_table.dim() != 2:
        raise ValueError("block_table must be int32 [batch, blocks], a sequence's entries next to each other")
    (batch, blocks), (row, entry) = block_table.shape, block_table.stride()
    if blocks > 1 and entry != 1:
        raise ValueError("block_table must be int32 [batch, blocks], a sequence's entries next to each other")
    if lens.dtype is not tt.int32 or lens.shape != (batch,) or not lens.is_contiguous():
        raise ValueError("lengths must be a contiguous int32 tensor [batch]")
    cu = None
    if cu_new is not None:
        if cu_new.dtype is not tt.int32 or cu_new.shape != (batch + 1,) or not cu_new.is_contiguous():
            raise ValueError("cu_new must be a contiguous int32 tensor [batch + 1]")
        cu = cu_new.data_ptr()
    if (k_pages.get_device() != device or v_pages.get_device() != device or block_table.get_device() != device or lens.get_device() != device
            or (cu is not None and cu_new.get_device() != device)):
        _refuse_place(device, k_pages=k_pages, v_pages=v_pages, cu_new=cu_new, block_table=block_table, lengths=lens)
    return L.TQPages(batch, k_shape[1], k_shape[0], blocks, row if batch > 1 else blocks, block_table.data_ptr(), cu, lens.data_ptr())


def _rows(name, x, heads, device, step):
    """(x, its strides): rows [rows, heads, 128] whose values lie next to each other, and which begin at multiples of 16 bytes (`step`
    values); a copy where they do not."""
    shape = x.shape
    if len(shape) != 3 or shape[2] != HEAD_DIM or shape[1] != heads:
        raise ValueError(f"{name} must be [rows, {heads}, {HEAD_DIM}], got {tuple(shape)}")
    if x.get_device() != device:
        _refuse_place(device, **{name: x})
    strides = x.stride()
    if strides[2] != 1 or strides[0] % step or strides[1] % step or x.data_ptr() % 16:
        x = x.clone(memory_format=L.torch().contiguous_format)
        strides = x.stride()
    return x, strides


_APPENDED = {}      # torch dtype -> its code


def append_paged(k_codec: TurboCodec | None, v_codec: TurboCodec | None, k, v, k_pages, v_pages, block_table, starts, cu_new=None, *,
                 overrun=None):
    """The new tokens' k and v [rows, KV heads, 128] (float16, bfloat16 or float32, any strides) into the pages of their
    sequences, from position starts[b] (int32 [batch]) of sequence b on, in one launch (tq_append_paged).  A codec of None stands for
    q8_0-style rows.  The bytes are those of LayerKV.append: earlier tokens stay, the rest of the last block is emptied.
    A page that is written must belong to one sequence.  A sequence without room, or a block without a page, is left out;
    `overrun` (a zeroed int32 device tensor with one element) then collects OVERRUN_* bits, see overrun_bits()."""
    tt, device = L.torch(), L._current_device()
    pages = _pages(k_codec, v_codec, k_pages, v_pages, block_table, starts, cu_new, device)
    dtype, heads = k.dtype, k_pages.shape[1]
    code = _APPENDED.get(dtype)
    if code is None:
        _APPENDED.update({tt.float16: L.TQ_F16, tt.bfloat16: L.TQ_BF16, tt.float32: L.TQ_F32})
        code = _APPENDED.get(dtype)
        if code is None:
            raise TypeError(f"unsupported dtype {dtype}")
    step = 4 if code == L.TQ_F32 else 8
    k, ks = _rows("k", k, heads, device, step)
    v, vs = _rows("v", v, heads, device, step)
    rows = k.shape[0]
    if rows != v.shape[0] or v.dtype is not dtype:
        raise ValueError("k and v must have the same rows and dtype")
    L.check(L.lib().tq_append_paged(_handle(k_codec), _handle(v_codec), C.byref(pages), k.data_ptr(), v.data_ptr(), rows, ks[0], ks[1], vs[0], vs[1],
                                    code, k_pages.data_ptr(), v_pages.data_ptr(), None if overrun is None else _overrun_ptr(overrun),
                                    L.stream_ptr()))
    return k_pages, v_pages


def load_paged(k_codec: TurboCodec | None, v_codec: TurboCodec | None, k_pages, v_pages, block_table, starts, cu_new=None,
               rows: int | None = None, *, out=None):
    """Positions starts[b] .. of every sequence, as many as cu_new gives it, back as fp16 values in the original domain: K and V
    [rows, KV heads, 128] in one launch (tq_load_paged).  rows: of the outputs (needed with cu_new); `out`: a pair of such
    tensors to write to instead.  Rows behind the last sequence, and rows without a page, are left as they were."""
    tt, device = L.torch(), L._current_device()
    pages = _pages(k_codec, v_codec, k_pages, v_pages, block_table, starts, cu_new, device)
    if out is None:
        if rows is None:
            if cu_new is not None:
                raise ValueError("load_paged needs the number of rows (rows, or out)")
            rows = pages.batch
        shape = (rows, pages.n_kv_heads, HEAD_DIM)
        out = k_pages.new_empty(shape, dtype=tt.float16), k_pages.new_empty(shape, dtype=tt.float16)
    else:
        rows = out[0].shape[0]
        shape = (rows, pages.n_kv_heads, HEAD_DIM)
        for x in out:
            if x.dtype != tt.float16 or x.shape != shape or not x.is_contiguous():
                raise ValueError(f"outputs must be contiguous fp16 tensors {shape}")
            if x.get_device() != device:
                _refuse_place(device, out=x)
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
        self.workspace, self._spaces = None, {}      # the last call's; every device's, ever larger

    def __call__(self, q, k_pages, v_pages, block_table, lens, cu_new=None, *, max_context: int | None = None, max_new: int | None = None,
                 out=None):
        """q [rows, query heads, 128], float16 or bfloat16, original domain -> out of the same shape and dtype, contiguous.
        lens (int32 [batch]): tokens that each sequence's pages hold, the new ones among them; row t of a sequence's n sees the
        positions before lens[b] - n + t + 1 (all lens[b] of them with causal=False), and a row that sees nothing is 0.
        Rows behind the last sequence are left as they were (`out`: a contiguous tensor to write to, apart from q's memory).
        max_context, max_new: no sequence holds more tokens, or has more new ones.  They size the launch: without them the table's
        width and the number of rows do, and a call on short sequences takes longer.  Of a sequence that exceeds them the
        tokens behind max_context are not seen and the rows from max_new on are left as they were."""
        tt, device = L.torch(), L._current_device()
        pages = _pages(self.k_codec, self.v_codec, k_pages, v_pages, block_table, lens, cu_new, device)
        if pages.n_kv_heads != self.n_kv_heads:
            raise ValueError(f"pages of {pages.n_kv_heads} KV heads, expected {self.n_kv_heads}")
        dtype = q.dtype
        if dtype is not tt.float16 and dtype is not tt.bfloat16:
            raise TypeError(f"queries must be float16 or bfloat16, not {dtype}")
        q, (q_token, q_head, _) = _rows("q", q, self.n_q_heads, device, 8)
        if out is None:
            out = q.new_empty(q.shape)
        elif out.shape != q.shape or out.dtype is not dtype or not out.is_contiguous():
            raise ValueError("out must be a contiguous tensor of q's shape and dtype")
        elif out.get_device() != device:
            _refuse_place(device, out=out)
        p = L.TQPagedAttnParams(pages, self.n_q_heads, self.causal, self.scale, L.TQ_BF16 if dtype is tt.bfloat16 else L.TQ_F16, q.shape[0],
                                q_token, q_head, 0 if max_context is None else max_context, 0 if max_new is None else max_new)
        lib, at = L.lib(), C.byref(p)
        need = lib.tq_paged_attn_workspace_bytes(at)
        if need < 0:
            L.check(L.ERR_ARG)
        spaces = self._spaces.get(device)
        if spaces is None or spaces[-1].numel() < need:     # smaller ones stay: a captured call may still write to them
            spaces = self._spaces.setdefault(device, [])
            spaces.append(tt.empty(need, dtype=tt.uint8, device=q.device))
        self.workspace = space = spaces[-1]
        L.check(lib.tq_paged_attention(_handle(self.k_codec), _handle(self.v_codec), at, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                                       out.data_ptr(), space.data_ptr(), space.numel(), L.stream_ptr()))
        return out
