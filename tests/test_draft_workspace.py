"""The scratch of tree attention: what its size entry says is enough for every call."""

from __future__ import annotations

import itertools

import pytest
import torch

from kairyu_amd import _native


@pytest.mark.skipif(torch.cuda.is_available(), reason="calls that nothing refuses end at the missing device")
@pytest.mark.parametrize("kv_heads", [1, 2, 3, 5, 6, 7, 8, 10, 12, 13, 24, 40, 64, 300])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_the_size_covers_every_window(dim, kv_heads):
    size = _native.library().kq_kv_tree_attention_workspace_size
    groups, batches = (1, 2, 8), ((1, 1), (9, 1), (32, 2), (70, 3), (400, 24), (4000, 150))
    for group, (rows, seqs), page, tokens in itertools.product(groups, batches, (16, 64), (1024, 8192, 65536, 1 << 20)):
        heads, width = kv_heads * group, tokens // page
        if heads > 1024:
            continue
        need = size(rows, heads, kv_heads, dim, page, width, seqs)
        for window in (0, 1, 64, 300, 1024, 1500, 4000, 1 << 30):
            with pytest.raises(RuntimeError, match="launch failed"):
                _native.call("kq_kv_tree_attention", 16, heads * dim, dim, 1, rows, heads, kv_heads, dim, 16, 16, 16, 16, 64, page,
                             16, width, width, 16, 16, seqs, 16, 1, 16, 1.0, window, 16, 16 if need else None, need, None)
