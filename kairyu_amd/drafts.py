"""Drafted tokens that branch, verified over the paged 8-bit cache.

A step of speculative decoding, for a batch whose sequences' new rows are drafted
tokens (counterpart of the speculative decoding in the reference's
kairyu/engine/core, next to this package's projections and attention):

* a sequence's first new row is its pending token, whose text is settled; the others
  name the row that they continue, ``parents [R]``;
* :func:`draft_tree` turns parents into positions and masks of ancestors, once a step;
* every layer runs :func:`kairyu_amd.attention.rotate_append` with the tree's positions
  and :func:`kairyu_amd.attention.tree_attention`, or both behind a pack's projection,
  ``QuantLinearPack.attend(..., tree=tree)``;
* :func:`accept_drafts` walks along the tokens that the model agrees with;
* :func:`keep_tokens` moves their keys and values, in every layer's cache, into the
  slots behind the context, and gives the new lengths.

All read lengths, tables and trees on the device only, so a whole step can be captured
into a graph.  On CPU tensors the same is computed by elementary torch operations.
"""

from __future__ import annotations

import torch

from kairyu_amd.attention import E4M3, MOST_NODES, DraftTree, PagedKvCache
from kairyu_amd.kernels import kv_cache_hip as hip
from kairyu_amd.pages import KvCaches, caches_of, check_ints, check_table

__all__ = ["DraftTree", "accept_drafts", "draft_tree", "keep_tokens"]


def _check_most(most: int) -> None:
    if not 1 <= most <= MOST_NODES:
        raise ValueError(f"most must be 1 to {MOST_NODES} new rows of a sequence, got {most}")


def draft_tree(parents: torch.Tensor, cu_rows: torch.Tensor, lengths: torch.Tensor, most: int, *,
               window: int = 0) -> DraftTree:
    """Positions and masks of drafted tokens from their parents.

    ``parents [R]`` int32 is each row's parent, counted from its sequence's first new row
    and before the row itself; -1 (and whatever is no such row) marks a root, which
    follows the context.  ``cu_rows`` and ``lengths`` are the batch's, the new rows
    included; ``most`` is at least any sequence's new rows.

    A row's position is the context's length plus its depth; its mask holds itself and its
    ancestors, with ``window`` only those at most ``window - 1`` above it.  Padding, rows at
    or past ``most`` of their sequence, and rows before the first token (of sequences
    with more rows than tokens) have position -1 and an empty mask."""

    _check_most(most)
    if not 0 <= window <= 1 << 30:
        raise ValueError(f"window must be 0 or a positive number of tokens, got {window}")
    check_ints(parents.device, parents=parents, cu_rows=cu_rows, lengths=lengths)
    if cu_rows.shape[0] != lengths.shape[0] + 1:
        raise ValueError(f"cu_rows {tuple(cu_rows.shape)} does not match {lengths.shape[0]} lengths")
    if not parents.is_cuda:
        return _draft_tree_plain(parents, cu_rows, lengths, most, window)
    return DraftTree(*hip.draft_tree(parents, cu_rows, lengths, most, window))


def accept_drafts(tokens: torch.Tensor, targets: torch.Tensor, parents: torch.Tensor, cu_rows: torch.Tensor,
                  most: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The drafted tokens that the model agrees with, by the greedy rule.

    ``tokens [R]`` are the rows' own, ``targets [R]`` what the model says comes after each
    (int32 or int64 alike).  The walk starts at a sequence's first new row and goes on to
    the lowest child whose token is the target of the row that it is at, until there is none.

    Returns ``kept [S, most]`` int32 (the rows walked along, counted from the sequence's
    first, -1 behind them), ``counts [S]`` int32 and ``following [S]``, the target of the
    last of them, which is the next step's pending token (-1 for a sequence without rows).
    Rows at or past ``most`` of a sequence are not looked at."""

    _check_most(most)
    if tokens.dim() != 1 or tokens.dtype not in (torch.int32, torch.int64) or not tokens.is_contiguous():
        raise ValueError(f"tokens must be contiguous int32 or int64 of one dimension, got {tokens.dtype} {tuple(tokens.shape)}")
    if targets.shape != tokens.shape or targets.dtype is not tokens.dtype or not targets.is_contiguous():
        raise ValueError(f"targets must be like tokens, got {targets.dtype} {tuple(targets.shape)}")
    if targets.device != tokens.device:
        raise RuntimeError(f"targets must be on {tokens.device}; found {targets.device}")
    check_ints(tokens.device, parents=parents, cu_rows=cu_rows)
    if parents.shape != tokens.shape or not cu_rows.shape[0]:
        raise ValueError(f"parents {tuple(parents.shape)} and cu_rows {tuple(cu_rows.shape)} do not match {tokens.shape[0]} rows")
    if not tokens.is_cuda:
        return _accept_plain(tokens, targets, parents, cu_rows, most)
    return hip.accept_drafts(tokens, targets, parents, cu_rows, most)


def keep_tokens(caches: PagedKvCache | KvCaches, block_table: torch.Tensor, cu_rows: torch.Tensor, lengths: torch.Tensor,
                kept: torch.Tensor, counts: torch.Tensor) -> torch.Tensor:
    """Make the kept new tokens of each sequence its only new ones: the ``i``-th of them,
    new row ``kept[s, i]``, moves to slot ``i`` behind the context in every cache.
    Returns the new lengths ``[S]``.

    ``kept [S, most]`` and ``counts [S]`` are int32, as :func:`accept_drafts` gives them.
    The kept tokens of a sequence end before the first that is not a new row of the
    sequence (of at most 1024), not above the one before it, or in a slot (its own or the
    one that it moves to) without a page; a sequence with more rows than tokens keeps none.

    A page into which tokens move has the largest scale that the page of any token that it
    then holds had, and its codes are rounded to that once; slots behind the kept tokens stay
    as they are.  A page is appended to by one sequence, as in an append."""

    caches = caches_of(caches)
    device = caches.device
    seqs = check_table(block_table, device)[0]
    check_ints(device, cu_rows=cu_rows, lengths=lengths, counts=counts)
    if lengths.shape[0] != seqs or cu_rows.shape[0] != seqs + 1 or counts.shape[0] != seqs:
        raise ValueError(f"cu_rows {tuple(cu_rows.shape)}, lengths {tuple(lengths.shape)} and counts {tuple(counts.shape)} "
                         f"do not match {seqs} sequences")
    if len(kept.shape) != 2 or kept.shape[0] != seqs or kept.dtype is not torch.int32 or not kept.is_contiguous():
        raise ValueError(f"kept must be contiguous int32 [{seqs}, most], got {kept.dtype} {tuple(kept.shape)}")
    if kept.shape[1] > MOST_NODES:
        raise ValueError(f"kept must name at most {MOST_NODES} tokens of a sequence, got {kept.shape[1]}")
    if kept.device != device:
        raise RuntimeError(f"kept must be on {device}; found {kept.device}")
    if not block_table.is_cuda:
        return _keep_plain(caches, block_table, cu_rows, lengths, kept, counts)
    return hip.keep_tokens(caches, block_table, cu_rows, lengths, kept, counts)


# ------------------------------------------------------------- plain forms
def _spans(rows: int, cu_rows: torch.Tensor):
    """(first row, rows) of each sequence, held within the tensors."""

    cu = [min(max(int(c), 0), rows) for c in cu_rows]
    return [(lo, max(hi - lo, 0)) for lo, hi in zip(cu, cu[1:])]


def _draft_tree_plain(parents, cu_rows, lengths, most, window):
    rows = parents.shape[0]
    mask = torch.zeros((rows, -(-most // 32)), dtype=torch.int32)
    positions = torch.full((rows,), -1, dtype=torch.int32)
    for (row, n), length in zip(_spans(rows, cu_rows), lengths.tolist()):
        first, above = max(length, 0) - n, []
        for i, p in enumerate(parents[row: row + min(n, most)].tolist()):
            above.append((above[p] if 0 <= p < i else []) + [i])
            position = first + len(above[i]) - 1
            if first + i < 0 or position < 0:
                continue
            positions[row + i] = position
            for j in above[i][-window:]:
                word = int(mask[row + i, j // 32]) & 0xFFFFFFFF | 1 << j % 32
                mask[row + i, j // 32] = word - (word >> 31 << 32)
    return DraftTree(mask, positions)


def _accept_plain(tokens, targets, parents, cu_rows, most):
    spans = _spans(tokens.shape[0], cu_rows)
    kept = torch.full((len(spans), most), -1, dtype=torch.int32)
    counts = torch.zeros(len(spans), dtype=torch.int32)
    following = torch.full((len(spans),), -1, dtype=tokens.dtype)
    for s, (row, n) in enumerate(spans):
        at = 0
        while at < min(n, most):
            kept[s, int(counts[s])] = at
            counts[s] += 1
            following[s] = targets[row + at]
            right = [i for i in range(at + 1, min(n, most)) if parents[row + i] == at and tokens[row + i] == targets[row + at]]
            at = right[0] if right else n
    return kept, counts, following


def _keep_plain(caches, table, cu_rows, lengths, kept, counts):
    pages, _, page, _ = caches.shape
    out = torch.zeros_like(lengths)
    for s, (row, n) in enumerate(_spans(1 << 24, cu_rows)):
        first = max(int(lengths[s]), 0) - n

        def place(node):
            slot = (first + node) // page
            p = int(table[s, slot]) if slot < table.shape[1] else -1
            return (p, (first + node) % page) if 0 <= p < pages else None

        moves, last = [], -1
        for i, node in enumerate(kept[s, : max(int(counts[s]), 0)].tolist()):
            if first < 0 or not last < node < min(n, MOST_NODES) or place(node) is None or place(i) is None:
                break
            moves.append((place(i), place(node)))
            last = node
        out[s] = max(first, 0) + len(moves)
        if not moves:
            continue
        to, of = (torch.tensor(x) for x in zip(*moves))
        for cache in caches.layers:
            for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
                old, raw = scales.clone(), codes.view(torch.uint8)
                value = codes[of[:, 0], :, of[:, 1]].to(torch.float32)
                for p in to[:, 0].unique().tolist():
                    here = of[to[:, 0] == p, 0].unique()
                    before = first % page if p == int(table[s, first // page]) else 0
                    new = old[torch.cat((here, torch.tensor([p]))) if before else here].amax(0)
                    scales[p] = new
                    if before:
                        codes[p, :, :before] = (codes[p, :, :before].to(torch.float32) * (old[p] / new)[:, None, None]).to(E4M3)
                value = (value * (old[of[:, 0]] / scales[to[:, 0]])[..., None]).to(E4M3)
                raw[to[:, 0], :, to[:, 1]] = value.view(torch.uint8)
    return out
