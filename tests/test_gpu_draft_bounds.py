"""Calls of drafts at the ends of their ranges: the largest batches, where indices of threads pass
31 bits, and heads that do not divide the workgroups."""

from __future__ import annotations

import pytest
import torch

import draft_helpers as dh
import kv_helpers as kv
from gpu_helpers import banner
from kairyu_amd.attention import DraftTree, tree_attention
from kairyu_amd.drafts import draft_tree
from oracle import drafts as odr

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs", [1 << 21, (1 << 21) + 3])
def test_trees_of_two_million_sequences(cuda, seqs):
    """1024 threads a sequence, 2^31 and more in all: the workgroups past 2^21 have padding, or
    none, and sequences of their own to look at."""
    banner(f"draft trees of {seqs} sequences")
    at, new, total = [5, (1 << 21) - 2, seqs - 1], [40, 7, 33], [60, 7, 1000]
    counts = torch.zeros(seqs, dtype=torch.int32)
    counts[at] = dh.ints(*new)
    lengths = torch.zeros(seqs, dtype=torch.int32)
    lengths[at] = dh.ints(*total)
    for lead, pad in ((0, 0), (3, 90)):  # (padding before the first sequence too)
        cu = torch.nn.functional.pad(counts.cumsum(0), (1, 0)).to(torch.int32) + lead
        par = torch.cat((torch.full((lead,), -1, dtype=torch.int32), dh.parents(new, 6, pad=pad)))
        got = draft_tree(par.to(cuda), cu.to(cuda), lengths.to(cuda), 1024)
        torch.cuda.synchronize()
        few = torch.tensor([0, *new]).cumsum(0) + lead  # (sequences without rows leave nothing)
        seen, positions = odr.tree(par, few, dh.ints(*total), 1024)
        assert got.positions.tolist() == positions and torch.equal(got.mask.cpu(), odr.pack(seen, 32))


@pytest.mark.parametrize("heads", [(20, 10, 256), (12, 6, 256), (7, 7, 256)], ids=str)
@pytest.mark.parametrize("window", [0, 64, 1024])
def test_attention_where_kv_heads_do_not_divide_the_workgroups(cuda, heads, window):
    """A window takes tiles of 16 columns, more of them than the wider ones without it."""
    banner(f"tree attention {heads} window {window}")
    (hq, hk, dim), new, total, page = heads, [20, 12], [1500, 300], 64
    table, cu, lengths, rows, pages = kv.batch(new, total, page, seed=1)
    pool = kv.cache(pages, hk, page, dim, seed=2)
    kv.stain(pool, table, lengths)
    tree, seen = dh.oracle_tree(dh.parents(new, 3), cu, lengths, max(new), window)
    q = (torch.randn(rows, hq, dim, generator=kv.gen(4)) * 2).to(torch.bfloat16)
    table = torch.nn.functional.pad(table, (0, 65536 // page - table.shape[1]), value=-1)
    out = tree_attention(q.to(cuda), kv.to(pool, cuda), table.to(cuda), cu.to(cuda), lengths.to(cuda),
                         DraftTree(*(t.to(cuda) for t in tree)), window=window)
    torch.cuda.synchronize()
    dh.check_attention(out, q, pool, table, cu, lengths, seen, tree.positions, window=window)
