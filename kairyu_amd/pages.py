"""Pages of the paged 8-bit cache that sequences share: copies, forks and returns.

The append (``kairyu_amd/attention.py``) writes a page for one sequence only.
Sequences that begin alike (samples of one prompt, beams, a cached prefix) share the
full pages of what they have in common and go on in pages of their own.  Who holds
what is kept on the device, in block tables (-1: no page) and ``holders [pages]``, the
number of table entries that name each page: a page that none does is free.  (The
reference's scheduler and radix cache, kairyu/engine/core, keep such counts on the host.)

* :func:`fork_sequences` lets rows go on as other rows: forks, reorders beams, ends
  sequences, and gives every row the pages that its next tokens are stored in.
* :func:`copy_pages` copies whole pages, for owners that keep their own books.

A page is the same in every layer, so all layers' caches are handed over at once,
:class:`KvCaches`.  Nothing is read by the host, so the calls can be captured into a
graph.  On CPU tensors the same is computed by elementary torch operations.
"""

from __future__ import annotations

import ctypes
from collections.abc import Sequence
from functools import lru_cache

import torch

from kairyu_amd.attention import E4M3, PagedKvCache, _check_cache, _rows_apart
from kairyu_amd.kernels import kv_cache_hip as hip

__all__ = ["KvCaches", "copy_pages", "fork_sequences"]


class KvCaches:
    """The caches of a model's layers, alike in shape and device, made once and kept by
    the program: pages, tables and lengths are the same for all of them.

    Launches go by the addresses that the tensors have when it is made, and it keeps that memory
    alive.  Where a tensor is given other memory afterwards (``.data =``, ``set_``, a move to another
    device) a new one has to be made, and the memory itself must not be resized under it."""

    __slots__ = ("layers", "shape", "device", "pointers", "memory")

    def __init__(self, layers: Sequence[PagedKvCache]) -> None:
        self.layers = tuple(layers)
        if not self.layers:
            raise ValueError("KvCaches needs at least one layer's cache")
        self.shape, self.device = _check_cache(self.layers[0]), self.layers[0].k.device
        for cache in self.layers:
            if cache is not self.layers[0] and _check_cache(cache) != self.shape:
                raise ValueError(f"caches must be alike: {tuple(cache.k.shape)} beside {tuple(self.shape)}")
            for t in cache:
                if t.device != self.device:
                    raise RuntimeError(f"caches must be on {self.device}; found {t.device}")
        at = [t.data_ptr() for cache in self.layers for t in cache]
        if self.shape[0] and len(set(at)) != len(at):
            raise ValueError("the layers' caches must be different tensors")
        self.pointers = _addresses(len(at))(*at)
        self.memory = [t.untyped_storage() for cache in self.layers for t in cache]


@lru_cache(maxsize=None)
def _addresses(n: int):
    return ctypes.c_uint64 * n


def caches_of(caches: PagedKvCache | KvCaches) -> KvCaches:
    return caches if isinstance(caches, KvCaches) else KvCaches((caches,))


def check_ints(device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if len(t.shape) != 1 or t.dtype is not torch.int32 or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous int32 of one dimension, got {t.dtype} {tuple(t.shape)}")
        if t.device != device:
            raise RuntimeError(f"{name} must be on {device}; found {t.device}")


def check_table(table: torch.Tensor, device: torch.device) -> torch.Size:
    shape = table.shape
    if len(shape) != 2 or table.dtype is not torch.int32 or not (table.is_contiguous() or _rows_apart(table)):
        raise ValueError("block_table must be int32 [S, W] with contiguous rows that do not overlap")
    if table.device != device:
        raise RuntimeError(f"block_table must be on {device}; found {table.device}")
    return shape


def copy_pages(caches: PagedKvCache | KvCaches, sources: torch.Tensor, targets: torch.Tensor) -> None:
    """Copy page ``sources[i]`` to page ``targets[i]`` (int32, device) in every cache,
    codes and scales.  Pairs that name no page, or one page twice, do nothing.  No page may
    be the target of two pairs, nor the target of one and the source of another."""

    caches = caches_of(caches)
    check_ints(caches.device, sources=sources, targets=targets)
    if sources.shape != targets.shape:
        raise ValueError(f"{sources.shape[0]} sources and {targets.shape[0]} targets")
    if not sources.is_cuda:
        _copy_plain(caches, sources, targets)
        return
    hip.copy_pages(caches, sources, targets)


def fork_sequences(caches: PagedKvCache | KvCaches, holders: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
                   parents: torch.Tensor, room: int = 1) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Row ``j`` of the new batch goes on as row ``parents[j]`` of the old one: ``(table
    [R, W], lengths [R], missing [1])``, all int32.

    ``holders [pages]`` counts the entries of ``block_table [S, W]`` that name each page
    (and whatever else shall keep a page from being given away); it is brought up to date
    in place, so that the old table is not to be used again.  ``parents [R]`` int32 may name a row any number of
    times; rows that none names are given back, as is a new row whose parent is no row (it is
    empty).  ``parents = arange(S)`` gives a batch its next pages.

    A new row shares the pages that its parent's tokens fill.  Those that the next ``room``
    tokens go to are its own: the parent's page where nobody else holds it and no earlier row
    has the same parent, otherwise the lowest pages that were free before the call, in the
    order of rows and slots; the tokens of a half-filled page are copied in every cache
    (its other slots stay as they are).  Pages behind those are given back.  With ``room`` 0
    a half-filled page is shared, and given back where its row goes on with ``room`` later.

    ``missing`` is the number of pages that there were too few; such entries are -1, and
    the row's tokens there are lost."""

    caches = caches_of(caches)
    pages = caches.shape[0]
    table_shape = check_table(block_table, caches.device)
    check_ints(caches.device, holders=holders, lengths=lengths, parents=parents)
    if holders.shape[0] != pages:
        raise ValueError(f"holders must count {pages} pages, got {holders.shape[0]}")
    if lengths.shape[0] != table_shape[0]:
        raise ValueError(f"block_table {tuple(table_shape)} does not match {lengths.shape[0]} lengths")
    if not 0 <= room <= 1 << 24:
        raise ValueError(f"room must be 0 to 2^24 tokens, got {room}")
    if not block_table.is_cuda:
        return _fork_plain(caches, holders, block_table, lengths, parents, room)
    return hip.fork_sequences(caches, holders, block_table, lengths, parents, room)


# ------------------------------------------------------------- plain forms
def _copy_plain(caches, sources, targets):
    pages = caches.shape[0]
    pairs = [(a, b) for a, b in zip(sources.tolist(), targets.tolist()) if 0 <= a < pages and 0 <= b < pages and a != b]
    for cache in caches.layers:
        for t in cache:
            raw = t.view(torch.uint8) if t.dtype is E4M3 else t
            for a, b in pairs:
                raw[b] = raw[a]


def _fork_plain(caches, holders, table, lengths, parents, room):
    pages, _, page, _ = caches.shape
    (seqs, width), rows = table.shape, parents.shape[0]
    old = table.tolist()
    free = [p for p, n in enumerate(holders.tolist()) if n == 0]
    held = holders.clone()
    new = torch.full((rows, width), -1, dtype=torch.int32)
    out = torch.zeros(rows, dtype=torch.int32)
    wanted, heard, copies = 0, set(), []

    def real(p):
        return 0 <= p < pages

    for j, s in enumerate(parents.tolist()):
        if not 0 <= s < seqs:
            continue
        eldest = s not in heard
        heard.add(s)
        length = max(int(lengths[s]), 0)
        out[j] = length
        begin = length // page
        for slot in range(width):
            p = old[s][slot]
            if slot < begin or (room == 0 and slot * page < length):
                new[j, slot] = p if real(p) else -1
            elif slot * page < length + room:
                if eldest and real(p) and int(holders[p]) == 1:
                    new[j, slot] = p
                    continue
                new[j, slot] = free[wanted] if wanted < len(free) else -1
                if slot == begin and length % page and real(p) and wanted < len(free):
                    copies.append((p, free[wanted], length % page))
                wanted += 1
    for entries, step in ((table, -1), (new, 1)):
        named = entries[(entries >= 0) & (entries < pages)].long()
        held.index_add_(0, named, torch.full_like(named, step, dtype=torch.int32))
    for cache in caches.layers:
        for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
            for a, b, tokens in copies:
                codes.view(torch.uint8)[b, :, :tokens] = codes.view(torch.uint8)[a, :, :tokens]
                scales[b] = scales[a]
    holders.copy_(held)
    return new, out, torch.tensor([max(wanted - len(free), 0)], dtype=torch.int32)
