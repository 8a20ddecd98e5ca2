"""The pages of a paged KV cache: who holds which.

``refs`` int32 [pages] counts the block-table entries that hold each page, 0 a free one; it
is all the state there is, one for the caches of all layers (which hold a sequence's tokens
in the same pages). Pages are given lowest free one first. Rollouts of a group share their
prompt's full pages (GrpoGenerationBatchRequest, summa-train/src/posttrain.rs:1206-1216):

    refs = page_refs(pages)
    page_reserve(refs, prompts, lengths, page_tokens)          # then prefill
    table, src, dst = page_fork(refs, prompts, lengths, source, page_tokens)
    paged.paged_copy(caches, src, dst)
    page_reserve(refs, table, lengths_so_far + room, page_tokens)   # as the rollouts grow
    page_free(refs, table, page_tokens)                        # at their end

Calls on one ``refs`` must be ordered, as on one stream; none synchronises.
"""
from __future__ import annotations

import torch

from ._lib import call
from .ops import _stream_on


def page_refs(pages: int, device="cuda") -> torch.Tensor:
    """The counts of a pool of free pages."""
    if pages <= 0:
        raise ValueError("need pages > 0")
    return torch.zeros(pages, dtype=torch.int32, device=device)


def _check(refs: torch.Tensor, *others) -> int:
    """The stream; every tensor contiguous int32 of the named dimensions, on refs' device."""
    index = refs.get_device()
    stream = _stream_on(index)
    for t, name, dims in ((refs, "refs", 1), *others):
        if t is None:
            continue
        if t.dtype is not torch.int32 or t.dim() != dims or not t.is_contiguous() or \
                t.get_device() != index:
            raise ValueError(f"{name} must be contiguous int32 of {dims} dimension"
                             f"{'s' if dims > 1 else ''} on the device of refs")
    return stream


def _p(t):
    return None if t is None else t.data_ptr()


def _missing(missing):
    if missing is not None and missing.shape != (1,):
        raise ValueError("missing must be int32 [1]")
    return missing, "missing", 1


def _rows(t: torch.Tensor, name: str, table: torch.Tensor) -> None:
    if t.shape[0] != table.shape[0]:
        raise ValueError(f"{name} must have one value a row of block_table")


def page_reserve(refs: torch.Tensor, block_table: torch.Tensor, tokens: torch.Tensor,
                 page_tokens: int, missing: torch.Tensor | None = None) -> None:
    """Pages for ``tokens[s]`` tokens of each row of ``block_table`` [S, columns], from its first
    entry that names none on. ``missing`` int32 [1] gets how many were not there (their entries
    stay -1)."""
    stream = _check(refs, (block_table, "block_table", 2), (tokens, "tokens", 1),
                    _missing(missing))
    _rows(tokens, "tokens", block_table)
    call("sm_page_reserve", refs.data_ptr(), refs.shape[0], block_table.data_ptr(),
         *block_table.shape, tokens.data_ptr(), int(page_tokens), _p(missing), stream)


def page_fork(refs: torch.Tensor, block_table: torch.Tensor, tokens: torch.Tensor,
              source: torch.Tensor, page_tokens: int, *, out: torch.Tensor | None = None,
              missing: torch.Tensor | None = None):
    """(table [children, columns], src, dst [children]): child c shares the full pages that hold
    the ``tokens[source[c]]`` tokens of row ``source[c]`` of ``block_table``, and has a page of
    its own for an unfinished last one, to be copied with ``paged.paged_copy(caches, src, dst)``
    (both -1: none). What the prompt's row does not hold, the child's does not either, and
    ``missing`` counts it. ``out``: the table to write (what it held before is not freed)."""
    stream = _check(refs, (block_table, "block_table", 2), (tokens, "tokens", 1),
                    (source, "source", 1), (out, "out", 2), _missing(missing))
    _rows(tokens, "tokens", block_table)
    (P, cols), C = block_table.shape, source.shape[0]
    if out is None:
        out = refs.new_empty((C, cols))
    elif out.shape != (C, cols):
        raise ValueError("out must have a row a child and the columns of block_table")
    src, dst = torch.empty_like(source), torch.empty_like(source)
    call("sm_page_fork", refs.data_ptr(), refs.shape[0], block_table.data_ptr(), P, cols,
         tokens.data_ptr(), source.data_ptr(), C, int(page_tokens), out.data_ptr(),
         src.data_ptr(), dst.data_ptr(), _p(missing), stream)
    return out, src, dst


def page_free(refs: torch.Tensor, block_table: torch.Tensor, page_tokens: int,
              tokens: torch.Tensor | None = None) -> None:
    """Entries of ``block_table`` behind those of the first ``tokens[s]`` tokens (default: all)
    leave their pages and become -1."""
    stream = _check(refs, (block_table, "block_table", 2), (tokens, "tokens", 1))
    if tokens is not None:
        _rows(tokens, "tokens", block_table)
    call("sm_page_free", refs.data_ptr(), refs.shape[0], block_table.data_ptr(),
         *block_table.shape, _p(tokens), int(page_tokens), stream)


def page_compact(refs: torch.Tensor, out: torch.Tensor | None = None):
    """(refs, page_map [pages], src, dst [pages / 2]) with the L live pages in front: where each
    page is then (-1: free), and the pages to be moved with ``paged.paged_copy(caches, src,
    dst)`` (-1 behind the last). Tables follow with ``page_remap``. ``out`` (``refs`` itself
    may be given) gets the new counts; without it ``refs`` stays as it is."""
    stream = _check(refs, (out, "out", 1))
    pages = refs.shape[0]
    if out is None:
        out = torch.empty_like(refs)
    elif out.shape != refs.shape:
        raise ValueError("out must have the shape of refs")
    page_map = torch.empty_like(refs)
    src, dst = refs.new_empty(pages // 2), refs.new_empty(pages // 2)
    call("sm_page_compact", refs.data_ptr(), pages, out.data_ptr(), page_map.data_ptr(),
         src.data_ptr(), dst.data_ptr(), stream)
    return out, page_map, src, dst


def page_remap(block_table: torch.Tensor, page_map: torch.Tensor,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """``block_table`` [S, columns] with every page where ``page_map`` puts it; ``out`` may be
    ``block_table``."""
    stream = _check(page_map, (block_table, "block_table", 2), (out, "out", 2))
    if out is None:
        out = torch.empty_like(block_table)
    elif out.shape != block_table.shape:
        raise ValueError("out must have the shape of block_table")
    call("sm_page_remap", block_table.data_ptr(), block_table.numel(), page_map.data_ptr(),
         page_map.shape[0], out.data_ptr(), stream)
    return out
