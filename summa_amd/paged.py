"""Paged KV cache: append and attention over pages in 16 or 8 bits.

The cache of ``AttnCache`` (summa-llm/src/model/attention.rs:20-40) in pages that any
sequence may hold, so rollouts of unequal length take what they use. Calls mirror
``sm_paged_append`` / ``sm_paged_attention`` (include/summa_amd.h, which states the
layouts and what each call leaves alone). A batch is described by device tensors:

- ``block_table`` int32 [S, columns]: entry j of a row is the page of the sequence's
  tokens ``j * page_tokens ..``;
- ``pos0`` int32 [S]: the tokens that each sequence holds before the call;
- ``row_start`` int32 [S + 1]: the sequences' rows in the row tensors, with ``max_rows``
  no less than any sequence has; without it every sequence has ``rows / S``.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import SM_BF16, SM_F8E4M3, SM_F16, SM_F32, call
from .ops import _head_rows, _rope_angles, _rope_layout, _stream_on

BLOCK = 16  # tokens of a cache block and of a scale
_CACHE = {torch.bfloat16: SM_BF16, torch.float16: SM_F16, torch.float8_e4m3fn: SM_F8E4M3}
_ROWS = {torch.float32: SM_F32, torch.bfloat16: SM_BF16, torch.float16: SM_F16}


def v_shape(pages: int, kv_heads: int, page_tokens: int, head_dim: int, dtype) -> tuple:
    """Shape of the values' storage: token 4 g + j and dim 16 (c T + t) + r of a 16-token
    block at [c, g, r, t, j], with T 4 (8-bit) or 2 (16-bit)."""
    T = 4 if dtype.itemsize == 1 else 2
    return (pages, kv_heads, page_tokens // BLOCK, head_dim // (16 * T), 4, 16, T, 4)


class PagedKVCache:
    """``pages`` pages of ``page_tokens`` tokens of ``kv_heads`` heads, in bfloat16, float16
    or float8_e4m3fn (8 bits with a power-of-two scale per 16 tokens and head)."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int, page_tokens: int = 64,
                 dtype: torch.dtype = torch.float8_e4m3fn, device="cuda"):
        if dtype not in _CACHE:
            raise TypeError("cache dtype must be bfloat16, float16 or float8_e4m3fn")
        if head_dim not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        if pages <= 0 or kv_heads <= 0 or page_tokens <= 0 or page_tokens % BLOCK:
            raise ValueError("need pages and kv_heads > 0, page_tokens a multiple of 16")
        shape = (pages, kv_heads, page_tokens, head_dim)
        k = torch.zeros(shape, dtype=torch.uint8 if dtype.itemsize == 1 else dtype, device=device)
        v = torch.zeros(v_shape(*shape, dtype), dtype=k.dtype, device=device)
        ks = vs = None
        if dtype.itemsize == 1:
            ks, vs = (torch.zeros(pages, kv_heads, page_tokens // BLOCK, dtype=torch.uint8,
                                  device=device) for _ in range(2))
        self._set(k.view(dtype), v.view(dtype), ks, vs)

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_scales: torch.Tensor | None = None,
                     v_scales: torch.Tensor | None = None) -> "PagedKVCache":
        """A cache over storage that the caller made: ``k`` [pages, kv_heads, page_tokens,
        head_dim], ``v`` of ``v_shape``, scales [pages, kv_heads, page_tokens / 16] uint8."""
        self = cls.__new__(cls)
        self._set(k, v, k_scales, v_scales)
        return self

    def _set(self, k, v, ks, vs) -> None:
        if k.dtype not in _CACHE or v.dtype != k.dtype:
            raise TypeError("cache dtype must be bfloat16, float16 or float8_e4m3fn")
        if k.dim() != 4 or tuple(v.shape) != v_shape(*k.shape, k.dtype):
            raise ValueError("k must be [pages, kv_heads, page_tokens, head_dim], v of v_shape")
        scales = (k.shape[0], k.shape[1], k.shape[2] // BLOCK)
        tensors = [(k, "k"), (v, "v")]
        if k.dtype.itemsize == 1:
            for t, name in ((ks, "k_scales"), (vs, "v_scales")):
                if t is None or t.dtype != torch.uint8 or tuple(t.shape) != scales:
                    raise ValueError(f"{name} must be uint8 [pages, kv_heads, page_tokens / 16]")
                tensors.append((t, name))
        else:
            ks = vs = None
        for t, name in tensors:
            if not t.is_cuda or t.device != k.device:
                raise ValueError(f"{name} must be a device tensor, all on one device")
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
        self._tensors = k, v, ks, vs  # (the descriptor below holds their addresses)
        self.pages, self.kv_heads, self.page_tokens, self.head_dim = k.shape
        self.dtype, self.device, self.index = k.dtype, k.device, k.get_device()
        self._c = _lib.PagedCache(k.data_ptr(), v.data_ptr(), ks.data_ptr() if ks is not None else 0,
                                  vs.data_ptr() if vs is not None else 0, self.pages,
                                  self.kv_heads, self.page_tokens, self.head_dim,
                                  _CACHE[k.dtype])
        self._at = C.addressof(self._c)

    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    k_scales = property(lambda self: self._tensors[2])
    v_scales = property(lambda self: self._tensors[3])

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self._tensors if t is not None)


def _rows(cache, t: torch.Tensor, name: str):
    """(rows, heads, row stride) of checked [rows, heads, head_dim] rows."""
    rows, heads, hd, ld = _head_rows(t, name)
    if hd != cache.head_dim:
        raise ValueError(f"{name} must be [rows, heads, {cache.head_dim}]")
    if t.get_device() != cache.index:
        raise ValueError(f"{name} must be on the cache's device")
    return rows, heads, ld


def _out(cache, out, rows, heads, dtype) -> torch.Tensor:
    hd = cache.head_dim
    if out is None:
        return torch.empty_strided((rows, heads, hd), (heads * hd, hd, 1), dtype=dtype,
                                   device=cache.device)
    if out.shape != (rows, heads, hd) or out.dtype is not dtype or not out.is_contiguous() or \
            out.get_device() != cache.index:
        raise ValueError(f"out must be contiguous [{rows}, {heads}, {hd}] {dtype} on the cache's "
                         "device")
    return out


def _batch(cache, rows, block_table, pos0, row_start, max_rows):
    """(stream, sequences, columns, row_start pointer, max_rows) of a checked batch."""
    index = cache.index
    stream = _stream_on(index)
    shape = block_table.shape
    if len(shape) != 2 or not block_table.is_contiguous():
        raise ValueError("block_table must be contiguous [sequences, columns]")
    S, cols = shape
    if pos0.shape != (S,) or not pos0.is_contiguous():
        raise ValueError("pos0 must be contiguous [sequences]")
    if block_table.dtype is not torch.int32 or pos0.dtype is not torch.int32:
        raise TypeError("block_table and pos0 must be int32")
    if block_table.get_device() != index or pos0.get_device() != index:
        raise ValueError("block_table and pos0 must be on the cache's device")
    if row_start is None:
        if S and rows % S:
            raise ValueError("without row_start every sequence has rows / sequences rows")
        return stream, S, cols, None, rows // S if S else 0
    if row_start.dtype is not torch.int32 or row_start.shape != (S + 1,) or \
            not row_start.is_contiguous() or row_start.get_device() != index:
        raise ValueError("row_start must be int32 [sequences + 1] on the cache's device")
    if max_rows is None:
        raise ValueError("row_start needs max_rows")
    return stream, S, cols, row_start.data_ptr(), min(int(max_rows), rows)


def paged_append(cache: PagedKVCache, k: torch.Tensor, v: torch.Tensor,
                 block_table: torch.Tensor, pos0: torch.Tensor,
                 row_start: torch.Tensor | None = None, *, q: torch.Tensor | None = None,
                 rope_table: torch.Tensor | None = None, layout: str = "interleaved",
                 q_dtype: torch.dtype | None = None, max_rows: int | None = None,
                 out: torch.Tensor | None = None):
    """Keys and values [rows, kv_heads, head_dim] (float32, bfloat16 or float16; rows may be
    strided, as those of fused qkv) into the pages at their positions, keys rotated by
    ``rope_table`` (``ops.rope_table``; None: no rotation). With ``q`` [rows, H, head_dim]
    also returns the rotated queries in ``q_dtype`` (bfloat16 or float16; default the
    cache's 16-bit type, or that of ``q``, or float16), in ``out`` where given; rows of no
    sequence are not written. (project_qkv + slice_assign,
    summa-llm/src/model/attention.rs:142-177, 331-356.)"""
    rows, heads, ldk = _rows(cache, k, "k")
    v_rows, v_heads, ldv = _rows(cache, v, "v")
    if heads != cache.kv_heads or v_heads != heads or v_rows != rows:
        raise ValueError(f"k and v must be [rows, {cache.kv_heads}, {cache.head_dim}]")
    dt = _ROWS.get(k.dtype)
    if dt is None or v.dtype is not k.dtype or (q is not None and q.dtype is not k.dtype):
        raise TypeError("q, k and v must be float32, bfloat16 or float16, of one dtype")
    stream, S, cols, starts, most = _batch(cache, rows, block_table, pos0, row_start, max_rows)
    H = ldq = 0
    qd, at_q, at_out = SM_F16, None, None
    if q is not None:
        q_rows, H, ldq = _rows(cache, q, "q")
        if q_rows != rows:
            raise ValueError("q must have the rows of k")
        if out is not None:
            if q_dtype not in (None, out.dtype):
                raise TypeError("out must have q_dtype")
            q_dtype = out.dtype
        elif q_dtype is None:
            q_dtype = cache.dtype if cache.dtype.itemsize == 2 else \
                q.dtype if q.dtype.itemsize == 2 else torch.float16
        if q_dtype is not torch.bfloat16 and q_dtype is not torch.float16:
            raise TypeError("q_dtype must be bfloat16 or float16")
        qd = _ROWS[q_dtype]
        out = _out(cache, out, rows, H, q_dtype)
        at_q, at_out = q.data_ptr(), out.data_ptr()
    elif out is not None:
        raise ValueError("out is for the queries: q is needed")
    table, table_rows, rot = _rope_angles(rope_table, cache.index)
    call("sm_paged_append", cache._at, block_table.data_ptr(), cols, pos0.data_ptr(), starts, S,
         rows, most, at_q, ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, dt, H, table, table_rows,
         rot, _rope_layout(layout), at_out, qd, stream)
    return out


def paged_attention(cache: PagedKVCache, q: torch.Tensor, block_table: torch.Tensor,
                    pos0: torch.Tensor, row_start: torch.Tensor | None = None, *,
                    max_rows: int | None = None, max_tokens: int | None = None,
                    want_lse: bool = False, out: torch.Tensor | None = None):
    """Attention of q [rows, H, head_dim] (bfloat16 or float16; a 16-bit cache's own type)
    over the pages, row i of a sequence seeing keys 0 .. pos0 + i; returns out [rows, H,
    head_dim] (``out`` where given; rows of no sequence are not written) and, with
    ``want_lse``, lse [rows, H] f32. ``max_tokens``: the longest sequence, new rows
    included (default: what the block table can hold); it decides how the keys are
    split, not which are read. With more than 16 rows a KV head (``max_rows * H / kv_heads``)
    softmax weights are rounded once to 16 bits, bf16 for a bf16 cache and f16 else; with up to
    16 the error is the output's rounding alone. (forward_cached / sdpa,
    summa-llm/src/model/attention.rs:216-265, 318-371.)"""
    rows, H, ldq = _rows(cache, q, "q")
    dt = _ROWS.get(q.dtype)
    if dt is None or dt == SM_F32:
        raise TypeError("q must be bfloat16 or float16")
    stream, S, cols, starts, most = _batch(cache, rows, block_table, pos0, row_start, max_rows)
    if max_tokens is None:
        max_tokens = min(cols * cache.page_tokens, 0x7fffffff)
    nbytes, ws = 0, None
    if max_tokens > 512:  # (none for fewer)
        nbytes = _lib.lib().sm_paged_attention_workspace_bytes(S, rows, most, H, cache.kv_heads,
                                                               cache.head_dim, max_tokens)
        if nbytes < 0:
            raise _lib.SummaError(-1, _lib.lib().sm_last_error().decode())
        if nbytes:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=cache.device)
    out = _out(cache, out, rows, H, q.dtype)
    lse = torch.empty((rows, H), dtype=torch.float32, device=cache.device) if want_lse else None
    call("sm_paged_attention", cache._at, block_table.data_ptr(), cols, pos0.data_ptr(), starts,
         S, rows, most, max_tokens, q.data_ptr(), dt, ldq, H, out.data_ptr(),
         None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(), nbytes,
         stream)
    return (out, lse) if want_lse else out
