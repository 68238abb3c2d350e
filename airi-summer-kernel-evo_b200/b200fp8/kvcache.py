"""Paged key / value cache at 4.5 bits an element, and the attention that reads it.

Pages of 16, 32 or 64 tokens; e2m1 codes with one e4m3 scale for 16 consecutive elements of a
head and an f32 scale for all keys and for all values (include/b200fp8.h has the layout).
Every list that changes while a model runs (table, lengths, use counts) lives on the device,
no call waits for the GPU, and all calls can be captured in CUDA graphs (copy_pages with the
pages that it was given then).

A step of a serving loop:

    cache.extend(counts, rows=rows)             # pages for the new tokens
    q, k = ops.rotary(q, k, positions, plan, ...)
    cache.write(k, v, layer=l, rows=rows)
    ctx = cache.attention(q, heads=h, layer=l, rows=rows)

What a call on the device finds wrong (a row out of range, too few pages) it leaves undone and
records in the device status word (:func:`b200fp8.device_status`: 5 bad lists, 6 no pages).
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from ._lib import check
from .ops import _DT, _raw_stream, _sig

_IN_KINDS = (torch.bfloat16, torch.float8_e4m3fn, torch.float16, torch.float32, torch.uint8)
_READ_KINDS = (torch.bfloat16, torch.float16, torch.float32)
_QUERY_KINDS = (torch.bfloat16, torch.float8_e4m3fn, torch.float16, torch.uint8)
_GATE_KINDS = (torch.float8_e4m3fn, torch.bfloat16, torch.uint8)
_PAGE_SIZES = (16, 32, 64)
_HEAD_DIMS = (64, 128, 256)


class Fp4Cache:
    """``layers`` x ``pages`` pages of ``page_size`` tokens of ``kv_heads`` heads, and a table of
    ``max_seqs`` sequences of at most ``max_pages`` pages each."""

    def __init__(self, *, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int,
                 max_seqs: int, max_pages: int, k_scale: float = 1.0, v_scale: float = 1.0,
                 device="cuda"):
        if page_size not in _PAGE_SIZES or head_dim not in _HEAD_DIMS:
            raise ValueError("page_size must be 16, 32 or 64 and head_dim 64, 128 or 256")
        block = page_size * head_dim * 9 // 8
        i32 = dict(dtype=torch.int32, device=device)
        self._init(torch.zeros((layers, pages, kv_heads, block), dtype=torch.uint8, device=device),
                   torch.full((max_seqs, max_pages), -1, **i32), torch.zeros(max_seqs, **i32),
                   torch.zeros(pages, **i32), page_size, head_dim, k_scale, v_scale)

    @classmethod
    def from_buffers(cls, storage: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
                     refs: torch.Tensor, *, page_size: int, head_dim: int, k_scale: float = 1.0,
                     v_scale: float = 1.0) -> "Fp4Cache":
        """A cache over the caller's buffers: ``storage`` uint8 [layers, pages, kv_heads,
        page_size * head_dim * 9 / 8], ``table`` int32 [seqs, pages of a sequence], ``lens``
        int32 [seqs], ``refs`` int32 [pages] (the number of table rows that use a page)."""
        self = cls.__new__(cls)
        self._init(storage, table, lens, refs, page_size, head_dim, k_scale, v_scale)
        return self

    def _init(self, storage, table, lens, refs, page_size, head_dim, k_scale, v_scale):
        if page_size not in _PAGE_SIZES or head_dim not in _HEAD_DIMS:
            raise ValueError("page_size must be 16, 32 or 64 and head_dim 64, 128 or 256")
        block = page_size * head_dim * 9 // 8
        if (storage.dtype != torch.uint8 or storage.dim() != 4 or storage.shape[3] != block
                or storage.stride(3) != 1 or storage.stride(2) != block):
            raise ValueError(f"storage must be uint8 [layers, pages, kv_heads, {block}], its pages "
                             "in one piece")
        for t, dim in ((table, 2), (lens, 1), (refs, 1)):
            if t.dtype != torch.int32 or t.dim() != dim or t.stride(-1) != 1:
                raise TypeError("table, lens and refs must be int32 of 2, 1 and 1 dimensions, "
                                "rows in one piece")
        if lens.shape[0] != table.shape[0] or refs.shape[0] != storage.shape[1]:
            raise ValueError("lens goes by the table's rows, refs by the storage's pages")
        if not storage.is_cuda or any(t.device != storage.device for t in (table, lens, refs)):
            raise ValueError("b200fp8 ops take CUDA tensors only (no CPU fallback), of one device")
        self.storage, self.table, self.lens, self.refs = storage, table, lens, refs
        self.layers, self.pages, self.kv_heads = storage.shape[:3]
        self.page_size, self.head_dim = page_size, head_dim
        self.k_scale, self.v_scale = float(k_scale), float(v_scale)
        self.device = storage.device
        self._index = storage.get_device()
        self._cols, self._seqs = self.kv_heads * head_dim, table.shape[0]
        lib = _lib.lib()
        self._write, self._read, self._attention = (lib.b2f_kv4_write, lib.b2f_kv4_read,
                                                    lib.b2f_kv4_attention)
        self._workspace = lib.b2f_kv4_attention_workspace_bytes
        c = _lib.Kv4Cache()
        c.storage, c.page_stride = storage.data_ptr(), storage.stride(1)
        c.pages, c.kv_heads = self.pages, self.kv_heads
        c.head_dim, c.page_size = head_dim, page_size
        c.k_scale, c.v_scale = self.k_scale, self.v_scale
        c.table, c.table_rows, c.table_cols = table.data_ptr(), *table.shape
        c.table_ld, c.lens = table.stride(0), lens.data_ptr()
        self._cache = c
        p = _lib.Kv4Pool()
        p.storage, p.layer_stride, p.page_stride = (storage.data_ptr(), storage.stride(0),
                                                    storage.stride(1))
        p.layers, p.pages, p.page_size = self.layers, self.pages, page_size
        p.page_bytes = self.kv_heads * block
        p.table, p.table_rows, p.table_cols = table.data_ptr(), *table.shape
        p.table_ld, p.lens, p.refs = table.stride(0), lens.data_ptr(), refs.data_ptr()
        self._pool = p
        # Argument blocks of calls that passed the checks, by shapes, strides, types and options
        # (never by addresses or values): a serving loop makes the same few calls over and over.
        self._known = {}

    # ------------------------------------------------------------------ helpers

    def _run(self, fn, *args) -> None:
        """Calls ``fn(*args, stream)`` with this cache's device current, on its current stream."""
        if torch.cuda.current_device() == self._index:
            code = fn(*args, _raw_stream(self._index))
        else:
            with torch.cuda.device(self._index):
                code = fn(*args, _raw_stream(self._index))
        if code:
            check(code)

    def _here(self, t: torch.Tensor, name: str) -> None:
        if t.get_device() != self._index:
            if not t.is_cuda:
                raise ValueError("b200fp8 ops take CUDA tensors only (no CPU fallback)")
            raise ValueError(f"{name} is on {t.device}, the cache is on {self.device}")

    def _list(self, t: torch.Tensor, name: str) -> int:
        """Length of an int32 list on this cache's device."""
        self._here(t, name)
        if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
            raise TypeError(f"{name} must be a contiguous int32 vector")
        return t.shape[0]

    def _batch(self, a, layer: int, tokens: int, rows, starts) -> None:
        """Fills in the cache and the batch of an argument block."""
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} of {self.layers}")
        a.cache = self._cache
        if layer:
            a.cache.storage = self._cache.storage + layer * self._pool.layer_stride
        b = a.batch
        if rows is not None:
            seqs = self._list(rows, "rows")
            b.rows = rows.data_ptr()
        elif starts is not None:
            seqs = starts.shape[0] - 1
        else:
            seqs = self._seqs
        if starts is not None:
            if self._list(starts, "starts") != seqs + 1:
                raise ValueError("starts must have one entry more than there are sequences")
            b.starts = starts.data_ptr()
        elif seqs == 0 or tokens % seqs:
            raise ValueError("without starts, every sequence has the same number of new tokens")
        b.seqs, b.tokens = seqs, tokens

    def _remember(self, key, a) -> bytes:
        if len(self._known) >= 1024:
            self._known.clear()
        known = self._known[key] = bytes(a)
        return known

    def _matrix(self, t: torch.Tensor, name: str, tokens: int, cols: int, kinds) -> int:
        """Row pitch of a row-major [tokens, cols] tensor on this cache's device."""
        self._here(t, name)
        if t.shape != (tokens, cols) or (cols > 1 and t.stride(1) != 1):
            raise ValueError(f"{name} must be a row-major [{tokens}, {cols}] tensor")
        if t.dtype not in kinds:
            raise TypeError(f"{name} must be one of {[str(d) for d in kinds]}")
        return t.stride(0)

    # ------------------------------------------------------------------ tokens

    def write(self, k: torch.Tensor, v: torch.Tensor, *, layer: int = 0,
              rows: Optional[torch.Tensor] = None, starts: Optional[torch.Tensor] = None,
              k_in_scale: float = 1.0, v_in_scale: float = 1.0) -> None:
        """Quantises the new tokens' keys and values ([tokens, kv_heads * head_dim], both f32,
        bf16, f16 or e4m3; value = stored * in_scale) into their places: token i of the n of a
        sequence at position length - n + i.  ``starts`` int32 [seqs + 1] cuts the packed
        tokens into sequences (None: equal parts), ``rows`` int32 [seqs] names their table
        rows (None: in order; distinct).  A page that rows share is written for all of them: after
        a fork only tokens that were added since are a row's own."""
        key = (0, k.shape, k.stride(), k.dtype, k.get_device(), v.shape, v.stride(), v.dtype,
               v.get_device(), layer, _sig(rows), _sig(starts), k_in_scale, v_in_scale)
        known = self._known.get(key)
        if known is None:
            tokens = k.shape[0]
            a = _lib.Kv4WriteArgs()
            a.k_ld = self._matrix(k, "k", tokens, self._cols, _IN_KINDS)
            a.v_ld = self._matrix(v, "v", tokens, self._cols, _IN_KINDS)
            if k.dtype != v.dtype:
                raise TypeError("k and v must have one type")
            if tokens == 0:
                return
            self._batch(a, layer, tokens, rows, starts)
            a.k_in_scale, a.v_in_scale, a.dtype = k_in_scale, v_in_scale, _DT[k.dtype]
            known = self._remember(key, a)
        a = _lib.Kv4WriteArgs.from_buffer_copy(known)
        if rows is not None:
            a.batch.rows = rows.data_ptr()
        if starts is not None:
            a.batch.starts = starts.data_ptr()
        a.k, a.v = k.data_ptr(), v.data_ptr()
        self._run(self._write, a)

    def read(self, tokens: int, *, layer: int = 0, rows: Optional[torch.Tensor] = None,
             starts: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16,
             k: Optional[torch.Tensor] = None, v: Optional[torch.Tensor] = None
             ) -> Tuple[torch.Tensor, torch.Tensor]:
        """The values that the cache holds for the last tokens of the sequences, placed as in
        :meth:`write`: (k, v), [tokens, kv_heads * head_dim] each, f32, bf16 or f16.  Rows of
        given ``k`` / ``v`` that belong to no sequence are left as they are."""
        if k is None:
            k = self.lens.new_empty((tokens, self._cols), dtype=dtype)
        if v is None:
            v = torch.empty_like(k)
        key = (1, tokens, k.shape, k.stride(), k.dtype, k.get_device(), v.shape, v.stride(), v.dtype,
               v.get_device(), layer, _sig(rows), _sig(starts))
        known = self._known.get(key)
        if known is None:
            a = _lib.Kv4ReadArgs()
            a.k_ld = self._matrix(k, "k", tokens, self._cols, _READ_KINDS)
            a.v_ld = self._matrix(v, "v", tokens, self._cols, _READ_KINDS)
            if k.dtype != v.dtype:
                raise TypeError("k and v must have one type")
            if tokens == 0:
                return k, v
            self._batch(a, layer, tokens, rows, starts)
            a.dtype = _DT[k.dtype]
            known = self._remember(key, a)
        a = _lib.Kv4ReadArgs.from_buffer_copy(known)
        if rows is not None:
            a.batch.rows = rows.data_ptr()
        if starts is not None:
            a.batch.starts = starts.data_ptr()
        a.k, a.v = k.data_ptr(), v.data_ptr()
        self._run(self._read, a)
        return k, v

    def attention(self, q: torch.Tensor, *, heads: int, layer: int = 0,
                  rows: Optional[torch.Tensor] = None, starts: Optional[torch.Tensor] = None,
                  causal: bool = True, q_scale: float = 1.0, sm_scale: float = 0.0,
                  gate: Optional[torch.Tensor] = None, gate_scale: float = 1.0,
                  gate_head_stride: Optional[int] = None, out: Optional[torch.Tensor] = None,
                  out_dtype: torch.dtype = torch.bfloat16, ctx_scale: float = 1.0,
                  return_lse: bool = False, lse: Optional[torch.Tensor] = None):
        """Attention of the new tokens ([tokens, heads * head_dim]; bf16, f16, or e4m3 with
        value = stored * q_scale) over the cached keys of their sequences, the new ones among
        them (see b2f_kv4_attention).  ``out`` bf16, f16 or e4m3 (stored = value / ctx_scale).
        With ``return_lse`` returns (out, lse f32 [tokens, heads])."""
        tokens, cols = q.shape[0], heads * self.head_dim
        key = (2, q.shape, q.stride(), q.dtype, q.get_device(), heads, layer, _sig(rows),
               _sig(starts), causal, q_scale, sm_scale, _sig(gate), gate_scale, gate_head_stride,
               _sig(out), out_dtype, ctx_scale, _sig(lse), return_lse)
        if out is None:
            out = q.new_empty((tokens, cols), dtype=out_dtype)
        if return_lse and lse is None:
            lse = q.new_empty((tokens, heads), dtype=torch.float32)
        known = self._known.get(key)
        if known is None:
            a = _lib.Kv4AttnArgs()
            a.q_ld = self._matrix(q, "q", tokens, cols, _QUERY_KINDS)
            a.out_ld = self._matrix(out, "out", tokens, cols, _QUERY_KINDS)
            if lse is not None:
                self._here(lse, "lse")
                if (lse.dtype != torch.float32 or lse.shape != (tokens, heads)
                        or not lse.is_contiguous()):
                    raise ValueError("lse must be contiguous float32 [tokens, heads]")
            if gate is not None:
                self._here(gate, "gate")
                stride = self.head_dim if gate_head_stride is None else gate_head_stride
                if (gate.dim() != 2 or gate.shape[0] != tokens or gate.stride(1) != 1
                        or gate.dtype not in _GATE_KINDS
                        or gate.shape[1] < (heads - 1) * stride + self.head_dim):
                    raise ValueError("gate must be row-major e4m3 or bf16, with a row for every "
                                     "token and a column for every element of every head")
                a.gate_dtype, a.gate_ld = _DT[gate.dtype], gate.stride(0)
                a.gate_head_stride, a.gate_scale = stride, gate_scale
            if tokens == 0:
                return (out, lse) if return_lse else out
            self._batch(a, layer, tokens, rows, starts)
            a.heads, a.causal, a.q_dtype, a.out_dtype = heads, causal, _DT[q.dtype], _DT[out.dtype]
            a.q_scale, a.sm_scale, a.ctx_scale = q_scale, sm_scale, ctx_scale
            with torch.cuda.device(self._index):
                a.workspace_bytes = -(-self._workspace(a) // 16) * 16
            known = self._remember(key, a)
        a = _lib.Kv4AttnArgs.from_buffer_copy(known)
        if rows is not None:
            a.batch.rows = rows.data_ptr()
        if starts is not None:
            a.batch.starts = starts.data_ptr()
        if gate is not None:
            a.gate = gate.data_ptr()
        if lse is not None:
            a.lse = lse.data_ptr()
        # A workspace of this call's own, from the caching allocator of the current stream: calls
        # on other streams, and in graphs, never share it.
        work = self.storage.new_empty(a.workspace_bytes)
        a.q, a.out, a.workspace = q.data_ptr(), out.data_ptr(), work.data_ptr()
        self._run(self._attention, a)
        return (out, lse) if return_lse else out

    # ------------------------------------------------------------------ pages

    def extend(self, counts: torch.Tensor, rows: Optional[torch.Tensor] = None) -> None:
        """Lengthens rows (None: rows 0 .. n - 1) by ``counts`` tokens (int32 [n], n <= 1024) and
        gives them the pages for it, or does nothing when the pages do not suffice."""
        n = self._list(counts, "counts")
        if rows is not None and self._list(rows, "rows") != n:
            raise ValueError("rows and counts must have one length")
        if n:
            self._run(_lib.lib().b2f_kv4_extend, self._pool,
                      None if rows is None else rows.data_ptr(), counts.data_ptr(), n)

    def fork(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Makes the empty rows ``dst`` copies of rows ``src`` (int32 [n], n <= 1024; src may
        repeat): full pages are shared, a last page that is not full is copied."""
        n = self._list(src, "src")
        if self._list(dst, "dst") != n:
            raise ValueError("src and dst must have one length")
        if n:
            work = self.lens.new_empty(n + 1)
            self._run(_lib.lib().b2f_kv4_fork, self._pool, src.data_ptr(), dst.data_ptr(), n,
                      work.data_ptr(), 4 * (n + 1))

    def free(self, rows: Optional[torch.Tensor] = None) -> None:
        """Empties ``rows`` (int32 [n]; None: all); pages that no other row uses become free."""
        free = _lib.lib().b2f_kv4_free
        if rows is None:
            rows = torch.arange(self._seqs, dtype=torch.int32, device=self.device)
        n = self._list(rows, "rows")
        for at in range(0, n, 1024):
            self._run(free, self._pool, rows.data_ptr() + 4 * at, min(1024, n - at))

    def compact(self) -> None:
        """Moves the pages in use to the front of the pool; the table follows."""
        lib = _lib.lib()
        ints = int(lib.b2f_kv4_compact_workspace_bytes(self.pages)) // 4
        work = self.lens.new_empty(ints)
        self._run(lib.b2f_kv4_compact, self._pool, work.data_ptr(), 4 * ints)

    def copy_pages(self, src: Sequence[int], dst: Sequence[int]) -> None:
        """Copies pages ``src[i]`` to ``dst[i]`` in all layers (host lists); table and counts
        stay as they are."""
        n = len(src)
        if len(dst) != n:
            raise ValueError("src and dst must have one length")
        if n:
            ints = ctypes.c_int * n
            # a number that no C int holds names no page either; ctypes would cut it off to one
            src, dst = ([p if 0 <= p < self.pages else -1 for p in x] for x in (src, dst))
            self._run(_lib.lib().b2f_kv4_copy_pages, self._pool, ints(*src), ints(*dst), n)

    def free_pages(self) -> int:
        """Pages that no row uses (waits for the device)."""
        return int((self.refs == 0).sum().item())
