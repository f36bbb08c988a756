"""Drafts in the largest batches, where indices of threads pass 31 bits."""

from __future__ import annotations

import pytest
import torch

import draft_helpers as dh
from gpu_helpers import banner
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
