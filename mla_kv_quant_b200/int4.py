"""The 4-bit latent cache: storing rows, attention over them, and attention over selected pages.

One layer holds ``codes`` uint8 ``[slots, D/2]`` (element ``2i`` in the low half of byte ``i``), ``params`` f32
``[slots, D/128, 2]`` (scale, zero; an element stands for ``(code - zero) * scale``) and ``rope`` bf16 ``[slots, Dr]``,
64 slots to a page.  For the page selection a box is kept beside each page: ``center`` int8 and ``radius`` uint8
``[pages, D + Dr]`` in units of ``2^exps[page, part]`` (int32 ``[pages, 2]``: the latent's and the rotary part's).
The C entry points are ``rolaq_int4_*`` in ``include/rolaq_b200.h``, with the exact rules.

The codec is the reference's uniform min/max codec (``mla_quant/oscar.py:91-101``) with 16 levels; rows are written in
the frame they are given in (rotate them first, ``ops.rotate_rows``, where the cache is to be rotated).

    pool = int4.Int4LatentPool(size=64 * 4096, layer_num=27, boxes=True)
    pool.write(layer, c_kv, k_pe, slots)                    # every new row
    pool.update_boxes(layer, pages, counts)                 # the pages they went to
    ws = pool.workspace(batch, heads=16, max_pages=256, budget=32)
    pool.decode(layer, q, page_table, seq_lens, sm_scale, out, lse, ws)
    pool.sparse_decode(layer, q, page_table, seq_lens, sm_scale, 32, out, lse, ws)

Nothing here allocates device memory except the constructors; calls run on the current stream of the
tensors' device.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib

PAGE = 64
GROUP_SIZE = 128

_BF16, _F32, _I32, _I64, _U8, _I8 = torch.bfloat16, torch.float32, torch.int32, torch.int64, torch.uint8, torch.int8


class Int4View:
    """The tensors of one layer's 4-bit cache, checked once.  ``boxes`` is (center, radius, exps) or None."""

    def __init__(self, codes: torch.Tensor, params: torch.Tensor, rope: torch.Tensor, boxes=None):
        if codes.dtype != _U8 or codes.dim() != 2:
            raise TypeError("codes must be uint8 [slots, D/2]")
        slots, d = codes.shape[0], codes.shape[1] * 2
        if params.dtype != _F32 or tuple(params.shape) != (slots, d // GROUP_SIZE, 2):
            raise TypeError("params must be float32 [slots, D/128, 2]")
        if rope.dtype != _BF16 or rope.dim() != 2 or rope.shape[0] != slots:
            raise TypeError("rope must be bfloat16 [slots, Dr]")
        if slots % PAGE or slots == 0:
            raise ValueError(f"slots must be a positive multiple of {PAGE}")
        if d not in (256, 512) or rope.shape[1] not in (32, 64):
            raise ValueError("D must be 256 or 512 and Dr 32 or 64")
        w = d + rope.shape[1]
        tensors = [codes, params, rope]
        if boxes is not None:
            center, radius, exps = boxes
            if center.dtype != _I8 or radius.dtype != _U8 or exps.dtype != _I32:
                raise TypeError("boxes must be (int8 center, uint8 radius, int32 exps)")
            if tuple(center.shape) != (slots // PAGE, w) or center.shape != radius.shape or tuple(exps.shape) != (slots // PAGE, 2):
                raise ValueError("boxes must be center and radius [slots/64, D + Dr], exps [slots/64, 2]")
            tensors += [center, radius, exps]
        for t in tensors:
            if not t.is_contiguous():
                raise ValueError("cache tensors must be contiguous")
            if t.device != codes.device:
                raise ValueError("cache tensors must be on one device")
        _lib.require_device(codes)
        self.codes, self.params, self.rope, self.boxes = codes, params, rope, boxes
        self.latent_dim, self.rope_dim, self.num_slots = d, rope.shape[1], slots
        self.device, self.index = codes.device, codes.get_device()
        ptrs = [t.data_ptr() for t in tensors] + [None] * (6 - len(tensors))
        self._c = _lib.Int4Cache(*ptrs, slots, d, rope.shape[1])
        self._ref = ctypes.addressof(self._c)


class Workspace:
    """Device scratch of ``decode`` / ``select_pages`` / ``sparse_decode`` calls of up to this size, and the selection's
    page table ``sel_table`` int32 ``[batch, budget]`` and lengths ``sel_lens`` (a smaller ``sparse_decode`` leaves its
    choice in ``sel_table[:B, :budget]`` and ``sel_lens[:B]``).  One per stream."""

    def __init__(self, view: Int4View, batch: int, q_len: int, heads: int, max_pages: int, budget: int = 0):
        n = _lib.load().rolaq_int4_workspace_bytes(batch, q_len, heads, view.latent_dim, max_pages)
        if n < 0:
            raise ValueError("batch must be in [0, 65535], q_len in [1, 64], heads in [1, 128], max_pages >= 0")
        self.scratch = torch.zeros(n, dtype=_U8, device=view.device)
        self.nbytes = n
        self._ptr = self.scratch.data_ptr()
        self.sel_table = torch.full((batch, max(budget, 1)), -1, dtype=_I32, device=view.device)
        self.sel_lens = torch.zeros(batch, dtype=_I32, device=view.device)


_raw_stream = torch._C._cuda_getCurrentRawStream  # torch.cuda.current_stream(d).cuda_stream without its object
_current_device = torch.cuda.current_device


def _stream(index: int, *tensors) -> int:
    """The current stream of device ``index``, on which all of ``tensors`` and which the current device have to be."""
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError(f"tensors on cuda:{index} and {t.device}: one device is needed")
    if index != _current_device():
        raise ValueError(f"the cache is on cuda:{index}, the current device is cuda:{_current_device()}")
    return _raw_stream(index)


def _need(t: torch.Tensor, name: str, dtype, ndim: int) -> None:
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must be {ndim}-D, got shape {tuple(t.shape)}")


def _rows(t: torch.Tensor, name: str, n: int, width: int) -> None:
    if t.shape != (n, width):
        raise ValueError(f"{name} must be [{n}, {width}], got {tuple(t.shape)}")
    if t.stride(1) != 1:
        raise ValueError(f"{name} rows must be contiguous")


def _slots(t: torch.Tensor) -> int:
    if t.dtype != _I64 and t.dtype != _I32:
        raise TypeError("slots must be int32 or int64")
    if t.dim() != 1 or not t.is_contiguous():
        raise ValueError("slots must be 1-D and contiguous")
    return int(t.dtype == _I64)


def _err(t: torch.Tensor | None):
    if t is None:
        return None
    if t.dtype != _I32 or t.numel() < 1:
        raise TypeError("err must be an int32 tensor with at least one element")
    return t.data_ptr()


def write(view: Int4View, c: torch.Tensor, k_pe: torch.Tensor, slots: torch.Tensor,
          err: torch.Tensor | None = None) -> None:
    """Quantise the rows ``c`` (bf16 or f32 ``[n, D]``) into ``slots`` and copy ``k_pe`` (bf16 ``[n, Dr]``) beside them.
    A slot that several rows share holds parts of any of them: only one that nothing reads (padding) may be shared."""
    is64 = _slots(slots)
    n = slots.shape[0]
    if c.dtype != _BF16 and c.dtype != _F32:
        raise TypeError(f"c must be bfloat16 or float32, got {c.dtype}")
    if k_pe.dtype != _BF16:
        raise TypeError(f"k_pe must be bfloat16, got {k_pe.dtype}")
    _rows(c, "c", n, view.latent_dim)
    _rows(k_pe, "k_pe", n, view.rope_dim)
    _lib.call("rolaq_int4_write", c.data_ptr(), c.dtype == _F32, c.stride(0), k_pe.data_ptr(), k_pe.stride(0),
              slots.data_ptr(), is64, n, view._ref, _err(err), _stream(view.index, c, k_pe, slots, err))


def read(view: Int4View, slots: torch.Tensor, out: torch.Tensor, out_pe: torch.Tensor | None = None,
         err: torch.Tensor | None = None) -> None:
    """The values of ``slots`` into ``out`` (bf16 or f32 ``[n, D]``), their rotary parts into ``out_pe`` (bf16 ``[n, Dr]``)."""
    is64 = _slots(slots)
    n = slots.shape[0]
    if out.dtype != _BF16 and out.dtype != _F32:
        raise TypeError(f"out must be bfloat16 or float32, got {out.dtype}")
    _rows(out, "out", n, view.latent_dim)
    if out_pe is not None:
        if out_pe.dtype != _BF16:
            raise TypeError(f"out_pe must be bfloat16, got {out_pe.dtype}")
        _rows(out_pe, "out_pe", n, view.rope_dim)
    _lib.call("rolaq_int4_read", view._ref, slots.data_ptr(), is64, n, out.data_ptr(), out.dtype == _F32, out.stride(0),
              None if out_pe is None else out_pe.data_ptr(), 0 if out_pe is None else out_pe.stride(0), _err(err),
              _stream(view.index, out, out_pe, slots, err))


def _pages(t: torch.Tensor, name: str, n: int | None = None) -> int:
    _need(t, name, _I32, 1)
    if not t.is_contiguous() or (n is not None and t.shape[0] != n):
        raise ValueError(f"{name} must be contiguous, one entry per page")
    return t.shape[0]


def update_boxes(view: Int4View, pages: torch.Tensor, counts: torch.Tensor, err: torch.Tensor | None = None) -> None:
    """The boxes of the first ``counts[i]`` tokens of ``pages[i]`` (both int32), from what the cache holds."""
    n = _pages(pages, "pages")
    _pages(counts, "counts", n)
    _lib.call("rolaq_int4_update_boxes", view._ref, pages.data_ptr(), counts.data_ptr(), n, _err(err),
              _stream(view.index, pages, counts, err))


def read_boxes(view: Int4View, pages: torch.Tensor, lo: torch.Tensor, hi: torch.Tensor,
               err: torch.Tensor | None = None) -> None:
    """The bounds that the boxes of ``pages`` stand for: ``lo``, ``hi`` f32 ``[n, D + Dr]``."""
    n = _pages(pages, "pages")
    w = view.latent_dim + view.rope_dim
    for name, t in (("lo", lo), ("hi", hi)):
        _need(t, name, _F32, 2)
        _rows(t, name, n, w)
    if lo.stride(0) != hi.stride(0):
        raise ValueError("lo and hi must share the row stride")
    _lib.call("rolaq_int4_read_boxes", view._ref, pages.data_ptr(), n, lo.data_ptr(), hi.data_ptr(), lo.stride(0),
              _err(err), _stream(view.index, pages, lo, hi, err))


def _requests(shape, q, view, page_table, seq_lens) -> tuple[int, int]:
    """Checks what the attention and the selection share; the page table's row stride and width."""
    b = shape[0]
    if q.dtype != _BF16 or shape[-1] != view.latent_dim + view.rope_dim or q.stride(-1) != 1:
        raise ValueError("q must be bfloat16 [B, T, H, D + Dr] or [B, H, D + Dr] with contiguous rows")
    if page_table.dtype != _I32 or seq_lens.dtype != _I32:
        raise TypeError("page_table and seq_lens must be int32")
    table = page_table.shape
    if len(table) != 2 or table[0] != b or (table[1] > 1 and page_table.stride(1) != 1):
        raise ValueError("page_table must be [B, max_pages] with contiguous rows")
    if seq_lens.shape != (b,) or not seq_lens.is_contiguous():
        raise ValueError("seq_lens must be contiguous [B]")
    return page_table.stride(0) if b > 1 else table[1], table[1]  # one row has no stride


def decode(q: torch.Tensor, view: Int4View, page_table: torch.Tensor, seq_lens: torch.Tensor, sm_scale: float,
           out: torch.Tensor, lse: torch.Tensor | None, ws: Workspace, err: torch.Tensor | None = None) -> None:
    """Attention of ``q`` (bf16 ``[B, H, D + Dr]``, or ``[B, T, H, D + Dr]`` for the last T tokens of each request,
    causal among themselves) over the requests' tokens: ``out`` bf16 ``[B, (T,) H, D]``, ``lse`` f32 ``[B, (T,) H]``
    (natural log, or None).  Rows that see no token get 0 and -inf."""
    shape = q.shape
    if len(shape) == 4:
        b, t, h, _ = shape
        q_sb, q_st, q_sh, _ = q.stride()
    elif len(shape) == 3:
        b, h, _ = shape
        q_sb, q_sh, _ = q.stride()
        t, q_st = 1, 0
    else:
        raise ValueError("q must be [B, H, D + Dr] or [B, T, H, D + Dr]")
    pt_stride, max_pages = _requests(shape, q, view, page_table, seq_lens)
    if out.dtype != _BF16 or out.shape != (*shape[:-1], view.latent_dim) or out.stride(-1) != 1:
        raise ValueError("out must be bfloat16, q's shape with D columns, with contiguous rows")
    o_stride = out.stride()
    if lse is not None and (lse.dtype != _F32 or lse.shape != shape[:-1] or not lse.is_contiguous()):
        raise ValueError("lse must be contiguous float32 of q's shape without the last axis")
    _lib.call("rolaq_int4_decode", q.data_ptr(), q_sb, q_st, q_sh, b, t, h, view._ref, page_table.data_ptr(), pt_stride,
              max_pages, seq_lens.data_ptr(), sm_scale, ws._ptr, ws.nbytes, out.data_ptr(), o_stride[0],
              o_stride[1] if t > 1 or len(shape) == 4 else 0, o_stride[-2], None if lse is None else lse.data_ptr(),
              None if err is None else _err(err),
              _stream(view.index, q, page_table, seq_lens, out, lse, ws.scratch, err))


def select_pages(q: torch.Tensor, view: Int4View, page_table: torch.Tensor, seq_lens: torch.Tensor, budget: int,
                 sel_table: torch.Tensor, sel_lens: torch.Tensor, ws: Workspace, keep_first: int = 1,
                 keep_last: int = 2, err: torch.Tensor | None = None) -> None:
    """The ``budget`` pages that each single-token query ``q`` (``[B, H, D + Dr]`` or ``[B, 1, H, D + Dr]``) attends to,
    as a page table (``sel_table``, rows at any stride): the first ``keep_first``, the last ``keep_last``, and those whose
    boxes score highest."""
    if view.boxes is None:
        raise ValueError("the cache has no page boxes")
    if q.dim() not in (3, 4) or q.dim() == 4 and q.shape[1] != 1:
        raise ValueError("pages are selected for one query token per request: q must be [B, H, D + Dr] or [B, 1, H, D + Dr]")
    shape = q.shape
    b, h = shape[0], shape[-2]
    pt_stride, max_pages = _requests(shape, q, view, page_table, seq_lens)
    if sel_table.dtype != _I32 or sel_table.shape != (b, budget) or (budget > 1 and sel_table.stride(1) != 1):
        raise ValueError("sel_table must be int32 [B, budget] with contiguous rows")
    if sel_lens.dtype != _I32 or sel_lens.shape != (b,) or not sel_lens.is_contiguous():
        raise ValueError("sel_lens must be contiguous int32 [B]")
    _lib.call("rolaq_int4_select_pages", q.data_ptr(), q.stride(0), q.stride(-2), b, h, view._ref,
              page_table.data_ptr(), pt_stride, max_pages, seq_lens.data_ptr(), budget, keep_first,
              keep_last, ws._ptr, ws.nbytes, sel_table.data_ptr(), sel_table.stride(0) if b > 1 else budget,
              sel_lens.data_ptr(), _err(err),
              _stream(view.index, q, page_table, seq_lens, sel_table, sel_lens, ws.scratch, err))


def sparse_decode(q: torch.Tensor, view: Int4View, page_table: torch.Tensor, seq_lens: torch.Tensor, sm_scale: float,
                  budget: int, out: torch.Tensor, lse: torch.Tensor | None, ws: Workspace, keep_first: int = 1,
                  keep_last: int = 2, err: torch.Tensor | None = None) -> None:
    """``select_pages`` into the workspace's ``sel_table`` / ``sel_lens`` (their first rows and columns, where the workspace
    was made for more), then ``decode`` over what it chose."""
    b, table, lens = q.shape[0], ws.sel_table, ws.sel_lens
    if table.shape != (b, budget):
        if b > table.shape[0] or budget > table.shape[1]:
            raise ValueError(f"the workspace was made for batch and budget {tuple(table.shape)}, not {(b, budget)}")
        table, lens = table[:b, :budget], lens[:b]
    select_pages(q, view, page_table, seq_lens, budget, table, lens, ws, keep_first, keep_last, err)
    decode(q, view, table, lens, sm_scale, out, lse, ws, err)


class Int4LatentPool:
    """The 4-bit cache of all layers, with the accounting of ``PackedLatentPool`` (rolaq_sglang.patch:166-188)."""

    def __init__(self, size: int, layer_num: int, kv_lora_rank: int = 512, qk_rope_head_dim: int = 64,
                 device: str | torch.device = "cuda", boxes: bool = False, start_layer: int = 0):
        if size % PAGE or size <= 0:
            raise ValueError(f"pool size must be a positive multiple of {PAGE} slots")
        d, dr, pages = kv_lora_rank, qk_rope_head_dim, size // PAGE
        self.size, self.layer_num, self.start_layer = size, layer_num, start_layer
        self.kv_lora_rank, self.qk_rope_head_dim = d, dr
        self._boxes = boxes
        self.views = []
        for _ in range(layer_num):
            box = None
            if boxes:
                box = (torch.zeros(pages, d + dr, dtype=_I8, device=device), torch.zeros(pages, d + dr, dtype=_U8, device=device),
                       torch.zeros(pages, 2, dtype=_I32, device=device))
            self.views.append(Int4View(torch.zeros(size, d // 2, dtype=_U8, device=device),
                                       torch.zeros(size, d // GROUP_SIZE, 2, dtype=_F32, device=device),
                                       torch.zeros(size, dr, dtype=_BF16, device=device), box))

    def layer_view(self, layer_id: int) -> Int4View:
        return self.views[layer_id - self.start_layer]

    def workspace(self, batch: int, heads: int, max_pages: int, q_len: int = 1, budget: int = 0) -> Workspace:
        return Workspace(self.views[0], batch, q_len, heads, max_pages, budget)

    def write(self, layer_id: int, c: torch.Tensor, k_pe: torch.Tensor, slots: torch.Tensor, err=None) -> None:
        write(self.layer_view(layer_id), c, k_pe, slots, err)

    def read(self, layer_id: int, slots: torch.Tensor, out: torch.Tensor, out_pe=None, err=None) -> None:
        read(self.layer_view(layer_id), slots, out, out_pe, err)

    def update_boxes(self, layer_id: int, pages: torch.Tensor, counts: torch.Tensor, err=None) -> None:
        update_boxes(self.layer_view(layer_id), pages, counts, err)

    def decode(self, layer_id: int, q, page_table, seq_lens, sm_scale, out, lse, ws, err=None) -> None:
        decode(q, self.layer_view(layer_id), page_table, seq_lens, sm_scale, out, lse, ws, err)

    def sparse_decode(self, layer_id: int, q, page_table, seq_lens, sm_scale, budget, out, lse, ws, keep_first=1,
                      keep_last=2, err=None) -> None:
        sparse_decode(q, self.layer_view(layer_id), page_table, seq_lens, sm_scale, budget, out, lse, ws, keep_first,
                      keep_last, err)

    def cell_size_bytes(self) -> int:
        """Bytes per token slot over all layers, the boxes' share included."""
        d, dr = self.kv_lora_rank, self.qk_rope_head_dim
        per_page = PAGE * (d // 2 + d // GROUP_SIZE * 8 + dr * 2) + (2 * (d + dr) + 8 if self._boxes else 0)
        return -(-per_page * self.layer_num // PAGE)

    def get_kv_size_bytes(self) -> int:
        d, dr, pages = self.kv_lora_rank, self.qk_rope_head_dim, self.size // PAGE
        per_layer = self.size * (d // 2 + d // GROUP_SIZE * 8 + dr * 2) + (pages * (2 * (d + dr) + 8) if self._boxes else 0)
        return per_layer * self.layer_num
