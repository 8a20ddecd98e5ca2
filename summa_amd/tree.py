"""Trees of drafted tokens: who sees whom, and which path the sampled tokens confirm.

``TextGenerator::generate`` (summa-llm/src/generate.rs:68-124) forwards one token a step.
With drafted continuations a step forwards a tree of them: row 0 of a sequence is the last
token chosen (not yet in the cache), row i continues row ``parents[i]`` < i. A step is

    mask, positions = tree_masks(parents, pos0)
    for each layer:
        q, k rotated at ``positions`` (ops.rope), k and v appended (paged.paged_append)
        paged.paged_tree_attention(cache, q, mask, block_table, pos0)
    sampled, logprobs = sampling.sample_rows(logits, uniforms, ...)
    path, count, emitted = tree_accept(parents, tokens, sampled)
    paged.paged_keep(caches, path, count, block_table, pos0)
    pos0 += count

Rows are given as [sequences, n], or as [rows] with ``row_start`` int32 [sequences + 1] and
``max_rows``, no less than any sequence has; at most 1024 a sequence.
"""
from __future__ import annotations

import torch

from ._lib import call
from .ops import _stream_on


def _tree(t: torch.Tensor, name: str, row_start, max_rows):
    """(stream, sequences, rows, max_rows, row_start pointer) of checked rows."""
    index = t.get_device()
    stream = _stream_on(index)
    if t.dtype is not torch.int32 or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32")
    if row_start is None:
        if t.dim() != 2:
            raise ValueError(f"without row_start, {name} must be [sequences, rows]")
        return stream, t.shape[0], t.numel(), t.shape[1], None
    if t.dim() != 1:
        raise ValueError(f"with row_start, {name} must be [rows]")
    if row_start.dtype is not torch.int32 or row_start.dim() != 1 or row_start.shape[0] < 1 or \
            not row_start.is_contiguous() or row_start.get_device() != index:
        raise ValueError(f"row_start must be int32 [sequences + 1] on {name}'s device")
    if max_rows is None:
        raise ValueError("row_start needs max_rows")
    rows = t.shape[0]
    return stream, row_start.shape[0] - 1, rows, min(int(max_rows), rows), row_start.data_ptr()


def tree_masks(parents: torch.Tensor, pos0: torch.Tensor, row_start: torch.Tensor | None = None,
               *, max_rows: int | None = None):
    """(mask int32 [rows, words], positions int32 [rows]) of every row: the rows that it sees, its
    ancestors and itself, a bit each, and ``pos0`` plus its depth. Rows of no sequence are not
    written."""
    stream, S, rows, most, starts = _tree(parents, "parents", row_start, max_rows)
    if pos0.dtype is not torch.int32 or pos0.shape != (S,) or not pos0.is_contiguous() or \
            pos0.get_device() != parents.get_device():
        raise ValueError("pos0 must be contiguous int32 [sequences] on the device of parents")
    words = max(1, (most + 31) // 32)
    mask, positions = parents.new_empty((rows, words)), parents.new_empty(rows)
    call("sm_tree_masks", parents.data_ptr(), pos0.data_ptr(), starts, S, rows, most,
         mask.data_ptr(), words, positions.data_ptr(), stream)
    return mask, positions


def tree_accept(parents: torch.Tensor, tokens: torch.Tensor, sampled: torch.Tensor,
                row_start: torch.Tensor | None = None, *, max_rows: int | None = None):
    """(path int32 [sequences, max_rows], count int32 [sequences], emitted int32 [sequences,
    max_rows]): from row 0 on, the rows of which each is the first that continues the one before
    and whose drafted token (``tokens``) is the one ``sampled`` behind that, and the sampled tokens
    along them; -1 behind ``count``. ``emitted[s, count - 1]`` is the next tree's row 0."""
    stream, S, rows, most, starts = _tree(parents, "parents", row_start, max_rows)
    for t, name in ((tokens, "tokens"), (sampled, "sampled")):
        if t.dtype is not torch.int32 or t.shape != parents.shape or not t.is_contiguous() or \
                t.get_device() != parents.get_device():
            raise ValueError(f"{name} must be contiguous int32 of parents' shape, on its device")
    path = torch.empty_like(parents) if starts is None else parents.new_empty((S, most))
    emitted, count = torch.empty_like(path), parents.new_empty(S)
    call("sm_tree_accept", parents.data_ptr(), tokens.data_ptr(), sampled.data_ptr(), starts, S,
         rows, most, path.data_ptr(), count.data_ptr(), emitted.data_ptr(), stream)
    return path, count, emitted
